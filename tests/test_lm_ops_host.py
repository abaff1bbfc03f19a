"""What the language-model operators refuse, and their geometry, without a GPU:
the backend's methods on tensors with made-up addresses, and the C entry points
called directly (they check arguments before they need a device).  Also the
float64 formulas the GPU tests compare with, against differences."""
import ctypes
import os
import re
import shutil
import subprocess

import numpy as np
import pytest

import lm_reference as ref
import neon_amd.backends  # noqa: F401
from neon_amd.backends import HIPTensor, NervanaHIP, bfloat16
from neon_amd.backends.hip import lmops
from neon_amd.backends.hip import runtime as hiprt


ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class NoDevice(object):
    """stands for the runtime: every call of the library is written down"""

    def __init__(self):
        self.calls, self.lib, self.stream = [], self, None

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0
        return call


@pytest.fixture()
def be():
    b = object.__new__(NervanaHIP)
    b.rt = NoDevice()
    b._lm_ws, b._temp_pool, b._rec_temps = None, {}, None
    b._lm_forms, b._pending, b._deferred = {}, [], []
    b._flush = lambda: None
    return b


_next = [1 << 32]


def T(be, shape, dtype=np.float32, strides=None, at=None):
    if at is None:
        at = _next[0]
        _next[0] += 1 << 28
    return HIPTensor(be, shape, dtype=dtype, gpudata=at, strides=strides)


def ln_args(be, axis=0, f=6, n=4, dtype=np.float32):
    big, per_f, per_n = ((f, n), (f, 1), (1, n)) if axis == 0 else ((n, f), (1, f), (n, 1))
    return dict(x=T(be, big, dtype), xmean=T(be, per_n), xvar=T(be, per_n), gamma=T(be, per_f), beta=T(be, per_f),
                y=T(be, big, dtype), eps=1e-5, axis=axis)


def ln_grad_args(be, **kw):
    a = ln_args(be, **kw)
    return dict(delta_out=T(be, a["x"].shape, a["x"].dtype), grad_gamma=T(be, a["gamma"].shape), grad_beta=T(be, a["gamma"].shape),
                delta_in=a["y"], x=a["x"], xmean=a["xmean"], xvar=a["xvar"], gamma=a["gamma"], eps=1e-5, axis=a["axis"])


def distill_args(be, axis=0, v=9, n=4, k=3):
    o = (lambda r: (r, n)) if axis == 0 else (lambda r: (n, r))
    return dict(y=T(be, o(v)), ids=T(be, o(k), np.int32), t=T(be, o(k)), loss=T(be, o(1)), stats=T(be, o(4)), axis=axis)


def test_calls_reach_the_library_with_the_layout_of_memory(be):
    for axis in (0, 1):
        be.rt.calls = []
        a = ln_args(be, axis)
        be.compound_fprop_ln(**a)
        name, args = be.rt.calls[-1]
        assert name == "nh_ln_fprop" and args[7:13] == (0, axis, 6, 4, 6 if axis else 4, 6 if axis else 4)
        # the transposed view of the other layout's memory
        a["x"], a["y"] = (T(be, t.shape[::-1]).T for t in (a["x"], a["y"]))
        be.compound_fprop_ln(**a)
        args = be.rt.calls[-1][1]
        assert args[7:13] == (0, 1 - axis, 6, 4, 4 if axis else 6, 4 if axis else 6)
    assert lmops._leading(T(be, (4, 6), strides=(12, 2)), 1, lmops.ROWS) is None
    assert lmops._leading(T(be, (4, 6), strides=(9, 1)), 1, lmops.ROWS) == 9
    assert lmops._leading(T(be, (4, 6), strides=(5, 1)), 1, lmops.ROWS) is None          # lines that overlap
    assert lmops._leading(T(be, (4, 6), strides=(-6, 1)), 1, lmops.ROWS) is None
    assert lmops._leading(T(be, (1, 6), strides=(1, 1)), 1, lmops.ROWS) == 6


def test_layer_norm_refusals(be):
    def refused(error, **change):
        for grad in (False, True):
            a = ln_grad_args(be) if grad else ln_args(be)
            if not set(change) <= set(a):
                continue
            with pytest.raises(error):
                (be.compound_bprop_ln if grad else be.compound_fprop_ln)(**dict(a, **change))
    refused(ValueError, axis=2)
    refused(TypeError, x=np.zeros((6, 4), np.float32))
    refused(TypeError, x=T(be, (6, 4), np.int32))
    refused(ValueError, x=T(be, (6, 5)))
    refused(ValueError, x=T(be, (6, 4, 1)))
    refused(TypeError, y=T(be, (6, 4), np.float16))
    refused(TypeError, delta_in=T(be, (6, 4), bfloat16))
    refused(ValueError, gamma=T(be, (1, 6)))
    refused(TypeError, gamma=T(be, (6, 1), np.float16))
    refused(ValueError, xmean=T(be, (4, 1)))
    refused(ValueError, grad_beta=T(be, (6, 2)))
    for out, grad in (("y", False), ("delta_out", True)):
        a = ln_grad_args(be) if grad else ln_args(be)
        a[out].rounding = 8
        with pytest.raises(NotImplementedError):
            (be.compound_bprop_ln if grad else be.compound_fprop_ln)(**a)
    # memory: shifted by one element, a stored statistic inside x, two outputs in one place
    a = ln_args(be)
    with pytest.raises(ValueError):
        be.compound_fprop_ln(**dict(a, y=T(be, (6, 4), at=a["x"].gpudata + 4)))
    with pytest.raises(ValueError):
        be.compound_fprop_ln(**dict(a, xmean=T(be, (1, 4), at=a["x"].gpudata)))
    with pytest.raises(ValueError):
        be.compound_fprop_ln(**dict(a, xvar=a["xmean"]))
    with pytest.raises(ValueError):
        be.compound_fprop_ln(**dict(a, y=T(be, (6, 4), strides=(1, 6), at=a["x"].gpudata)))
    with pytest.raises(ValueError):
        be.compound_fprop_ln(**dict(a, xmean=T(be, (1, 4), strides=(0, 0))))
    g = ln_grad_args(be)
    with pytest.raises(ValueError):
        be.compound_bprop_ln(**dict(g, grad_gamma=g["gamma"]))
    assert not be.rt.calls
    be.compound_bprop_ln(**dict(g, delta_out=g["delta_in"]))
    be.compound_fprop_ln(**dict(a, y=a["x"]))
    with pytest.raises(ValueError):
        be.compound_fprop_ln(T(be, (0, 4)), T(be, (1, 4)), T(be, (1, 4)), T(be, (0, 1)), T(be, (0, 1)), T(be, (0, 4)), 1e-5)


def test_views_that_interleave_are_told_from_views_that_overlap(be):
    """against the sets of addresses, over random pairs of views"""
    rs = np.random.RandomState(0)
    told = 0
    for _ in range(4000):
        ld = rs.randint(1, 12)
        views = []
        for _k in range(2):
            shape = tuple(int(v) for v in rs.randint(1, 5, 2))
            strides = (int(ld * rs.randint(1, 3)), int(rs.randint(1, 4)))
            if rs.rand() < 0.3:
                strides = strides[::-1]
            views.append(T(be, shape, strides=strides, at=4096 + 4 * int(rs.randint(0, 30))))
        if rs.rand() < 0.6:
            views[1] = T(be, views[1].shape, strides=views[0].strides, at=views[1].gpudata)
        at = [set((np.add.outer(np.arange(v.shape[0]) * v.strides[0], np.arange(v.shape[1]) * v.strides[1]) * 4
                   + v.gpudata).ravel().tolist()) for v in views]
        if lmops._interleaved(*views):
            told += 1
            assert not at[0] & at[1]
    assert told > 300
    # the statistics of a layer as two columns of one matrix
    stats = T(be, (4, 2))
    assert lmops._interleaved(stats[:, 0:1], stats[:, 1:2]) and not lmops._interleaved(stats[:, 0:1], stats[0:2, 0:1])


def test_embedding_refusals(be):
    def args(**change):
        return dict(dict(inputs=T(be, (1, 4), np.int32), W=T(be, (10, 6)), outputs=T(be, (6, 4))), **change)

    def grads(**change):
        return dict(dict(inputs=T(be, (1, 4), np.int32), error=T(be, (6, 4)), dW=T(be, (10, 6))), **change)
    for bad, error in ((dict(inputs=T(be, (1, 4))), TypeError), (dict(inputs=T(be, (1, 5), np.int32)), ValueError),
                       (dict(axis=1), ValueError), (dict(W=T(be, (10, 6), np.float16)), TypeError),
                       (dict(W=T(be, (10, 6), np.int32)), TypeError), (dict(outputs=T(be, (4, 6))), ValueError),
                       (dict(W=T(be, (0, 6))), ValueError), (dict(axis=-1), ValueError),
                       (dict(inputs=T(be, (1, 4), np.int32, strides=(4, -1))), NotImplementedError)):
        with pytest.raises(error):
            be.compound_fprop_lut(**args(**bad))
    a = args()
    with pytest.raises(ValueError):
        be.compound_fprop_lut(**dict(a, outputs=T(be, (6, 4), at=a["W"].gpudata + 96)))
    for bad, error in ((dict(error=T(be, (4, 6))), ValueError), (dict(error=T(be, (6, 4), np.float16)), TypeError),
                       (dict(dW=T(be, (10, 5))), ValueError), (dict(dW=T(be, (10, 6), np.uint8)), TypeError)):
        with pytest.raises(error):
            be.compound_update_lut(**grads(**bad))
    g = grads()
    with pytest.raises(ValueError):
        be.compound_update_lut(**dict(g, dW=T(be, (10, 6), at=g["error"].gpudata)))
    assert not be.rt.calls
    be.compound_update_lut(**grads())
    assert be.rt.calls[-1][0] == "nh_embed_update"


def test_distillation_refusals(be):
    for bad, error in ((dict(temperature=0.0), ValueError), (dict(temperature=-1), ValueError),
                       (dict(temperature=float("nan")), ValueError), (dict(temperature=float("inf")), ValueError),
                       (dict(temperature=1e20), ValueError), (dict(temperature=1e-20), ValueError),
                       (dict(ids=T(be, (3, 4))), TypeError), (dict(ids=T(be, (3, 5), np.int32)), ValueError),
                       (dict(t=T(be, (2, 4))), ValueError), (dict(t=T(be, (3, 4), np.int32)), TypeError),
                       (dict(loss=T(be, (4, 1))), ValueError), (dict(stats=T(be, (1, 4))), ValueError),
                       (dict(stats=T(be, (4, 4), np.float16)), TypeError), (dict(y=T(be, (0, 4))), ValueError)):
        with pytest.raises(error):
            be.compound_fprop_distill(**dict(distill_args(be), **bad))
    a = distill_args(be)
    with pytest.raises(ValueError):
        be.compound_fprop_distill(**dict(a, loss=T(be, (1, 4), at=a["stats"].gpudata)))
    a.pop("loss")
    for bad, error in ((dict(delta=a["y"]), ValueError), (dict(delta=T(be, (9, 5))), ValueError),
                       (dict(delta=T(be, (9, 4), np.float16)), TypeError), (dict(weight=T(be, (4, 1))), ValueError),
                       (dict(weight=T(be, (1, 4), np.float16)), TypeError)):
        with pytest.raises(error):
            be.compound_bprop_distill(**dict(dict(a, delta=T(be, (9, 4))), **bad))
    assert not be.rt.calls


def test_a_call_of_a_form_seen_before_is_checked_where_it_can_differ(be):
    """the second call of equal shapes takes the short way: same library call,
    but overlap, rounding and changed layouts are still found"""
    for axis in (0, 1):
        be.rt.calls = []
        a, b = ln_args(be, axis), ln_args(be, axis)
        be.compound_fprop_ln(**a)
        be.compound_fprop_ln(**b)
        first, second = [c[1] for c in be.rt.calls if c[0] == "nh_ln_fprop"]
        assert first[6:13] == second[6:13] and second[0] == b["y"].gpudata and second[3] == b["x"].gpudata
        for bad in (dict(y=T(be, b["x"].shape, at=b["x"].gpudata + 4)), dict(xmean=T(be, b["xmean"].shape, at=b["x"].gpudata)),
                    dict(xvar=b["xmean"]), dict(gamma=b["y"])):
            with pytest.raises(ValueError):
                be.compound_fprop_ln(**dict(b, **bad))
        be.compound_fprop_ln(**dict(b, y=b["x"]))
        be.compound_fprop_ln(**dict(b, beta=b["gamma"]))                  # inputs may share memory
        b["y"].rounding = 10
        with pytest.raises(NotImplementedError):
            be.compound_fprop_ln(**b)
        b["y"].rounding = 0
        turned = dict(b, x=T(be, b["x"].shape[::-1]).T, y=T(be, b["x"].shape[::-1]).T)
        be.compound_fprop_ln(**turned)
        assert be.rt.calls[-1][1][8] == 1 - axis
        with pytest.raises(TypeError):
            be.compound_fprop_ln(**dict(b, x=T(be, b["x"].shape, np.float16)))
        with pytest.raises(ValueError):
            be.compound_fprop_ln(**dict(b, axis=1 - axis))
    # a reversed view lies below its first element
    d = distill_args(be)
    d["ids"] = T(be, (3, 4), np.int32, strides=(-4, 1), at=d["ids"].gpudata + 32)
    be.compound_fprop_distill(**d)
    be.rt.calls = []
    be.compound_fprop_distill(**d)
    assert [c[0] for c in be.rt.calls] == ["nh_distill_fprop"]
    with pytest.raises(ValueError):
        be.compound_fprop_distill(**dict(d, loss=T(be, (1, 4), at=d["ids"].gpudata - 32)))
    d = distill_args(be)
    for _ in range(2):
        be.compound_fprop_distill(**d)
        with pytest.raises(ValueError):
            be.compound_fprop_distill(**dict(d, temperature=0))


def test_the_workspace_grows_and_is_kept(be):
    events = []
    be.rt = NoDevice()
    be.rt.malloc = lambda n: events.append(("malloc", n)) or 4096 + len(events)
    be.rt.free = lambda p: events.append(("free", p))
    be.synchronize = lambda: events.append(("wait",))
    first = be._lm_workspace(10)
    assert first[1] >= 10 and be._lm_workspace(first[1]) == first and be._lm_workspace(0) == (0, 0)
    second = be._lm_workspace(first[1] + 1)
    assert [e[0] for e in events] == ["malloc", "wait", "free", "malloc"] and second[1] > first[1]


# ---- the C entry points -------------------------------------------------------------------------
def codes(lib, name, good, bads):
    fn = getattr(lib, name)
    for bad in bads:
        a = list(good)
        for i, v in bad.items():
            a[i] = v
        assert fn(*a) == hiprt.NH_EINVAL, (name, bad)
        assert lib.nh_last_error().startswith(name.encode())
    return fn(*good)


def test_entry_points_check_arguments_before_they_need_a_device():
    lib = hiprt.load_library()
    P, BIG = 4096, 1 << 40
    ok = []
    #       y mean var x gamma beta eps  dtype axis F   N  ldx ldy ws bytes stream
    good = [P, P, P, P, P, P, 1e-5, 0, 0, 5000, 64, 64, 64, P, BIG, None]
    ok.append(codes(lib, "nh_ln_fprop", good, [
        {0: None}, {1: None}, {2: None}, {3: None}, {4: None}, {5: None}, {7: 3}, {7: -1}, {8: 2}, {9: 0}, {9: 1 << 31},
        {10: 1 << 41}, {11: 63}, {12: 63}, {13: None}, {13: P + 8}, {14: lib.nh_ln_workspace_bytes(0, 0, 0, 5000, 64) - 1}]))
    #       dx dg db dy x mean var gamma eps dtype axis F N ldx lddy lddx ws bytes stream
    good = [P, P, P, P, P, P, P, P, 1e-5, 2, 1, 100, 64, 100, 100, 100, P, BIG, None]
    ok.append(codes(lib, "nh_ln_bprop", good, [
        {0: None}, {1: None}, {2: None}, {3: None}, {4: None}, {5: None}, {6: None}, {7: None}, {9: 9}, {10: 5}, {11: 0},
        {13: 99}, {14: 99}, {15: 99}, {16: None}, {16: P + 4}, {17: lib.nh_ln_workspace_bytes(1, 2, 1, 100, 64) - 1}]))
    #       out W ids scale dtype axis N E V ldw ldout pad stream
    good = [P, P, P, 1.0, 1, 0, 50, 20, 30, 20, 50, -1, None]
    ok.append(codes(lib, "nh_embed_fprop", good, [
        {0: None}, {1: None}, {2: None}, {4: 7}, {5: 2}, {6: 1 << 31}, {7: 0}, {7: 1 << 27}, {8: 0}, {8: 1 << 31}, {9: 19},
        {10: 49}]))
    #       dW err ids scale beta dtype axis N E V lddw lderr pad ws bytes stream
    good = [P, P, P, 1.0, 0.0, 1, 1, 50, 20, 30, 20, 20, -1, P, BIG, None]
    ok.append(codes(lib, "nh_embed_update", good, [
        {0: None}, {1: None}, {2: None}, {5: 7}, {6: 2}, {7: 1 << 31}, {8: 0}, {9: 0}, {10: 19}, {11: 19}, {13: None}, {13: P + 8},
        {14: lib.nh_embed_update_workspace_bytes(1, 1, 50, 20, 30) - 1}]))
    s = hiprt.int64s(5, 1, 5, 1, 1, 5, 1)
    #       loss stats z ids t T dtype tdtype axis V N K ldz strides ws bytes stream
    good = [P, P, P, P, P, 1.0, 0, 2, 0, 90, 5, 3, 5, s, P, BIG, None]
    ok.append(codes(lib, "nh_distill_fprop", good, [
        {0: None}, {1: None}, {2: None}, {3: None}, {4: None}, {5: 0.0}, {5: -1.0}, {5: float("nan")},
        {5: float("inf")}, {5: 1e-40}, {5: 1e-20}, {5: 1e20}, {6: 3}, {7: 3}, {8: 2}, {9: 0}, {9: 1 << 31}, {10: 1 << 41}, {11: 1025}, {12: 4},
        {13: None}, {14: None}, {14: P + 8}, {15: lib.nh_distill_workspace_bytes(0, 0, 90, 5) - 1}]))
    #       dz z ids t stats w wall T dtype tdtype axis V N K ldz lddz strides ws bytes stream
    good = [P, P, P, P, P, None, 1.0, 1.0, 0, 2, 0, 90, 5, 3, 5, 5, s, None]
    ok.append(codes(lib, "nh_distill_bprop", good, [
        {0: None}, {1: None}, {2: None}, {3: None}, {4: None}, {7: 0.0}, {8: 3}, {9: 3}, {10: 2}, {11: 0},
        {13: 1025}, {14: 4}, {15: 4}, {16: None}]))
    count = ctypes.c_int(0)
    if lib.nh_device_count(ctypes.byref(count)) or not count.value:
        assert ok == [hiprt.NH_ENOTINIT] * 6


test_entry_points_check_arguments_before_they_need_a_device = pytest.mark.skipif(
    hiprt.device_count() > 0, reason="a device is there: the good calls above would run on made-up addresses")(
        test_entry_points_check_arguments_before_they_need_a_device)


# ---- registers ------------------------------------------------------------------------------------
@pytest.mark.skipif(shutil.which("hipcc") is None, reason="hipcc not on PATH")
@pytest.mark.parametrize("source", ["layernorm", "embedding", "distill"])
def test_kernels_keep_to_their_registers(source):
    """tensors held in registers that spilled would still give the right values,
    two or three times slower; a few registers' worth of scratch is let pass"""
    cmd = ["hipcc", "-O3", "-std=c++17", "--offload-arch=gfx950", "-ffp-contract=off", "-Xclang", "-target-feature", "-Xclang",
           "-packed-fp32-ops", "-I" + os.path.join(ROOT, "include"), "-I" + os.path.join(ROOT, "neon_amd", "csrc"), "-c",
           os.path.join(ROOT, "neon_amd", "csrc", source + ".hip"), "-o", os.devnull, "--offload-device-only",
           "-Rpass-analysis=kernel-resource-usage"]
    out = subprocess.run(cmd, capture_output=True, text=True)
    assert out.returncode == 0, out.stderr[-2000:]
    names = re.findall(r"Function Name: (\S+)", out.stderr)
    scratch = [int(v) for v in re.findall(r"ScratchSize \[bytes/lane\]: (\d+)", out.stderr)]
    assert len(names) == len(scratch) >= 10
    assert not [(n, s) for n, s in zip(names, scratch) if s > 16]


# ---- the formulas themselves ---------------------------------------------------------------------
def _slope(f, args, at, u, h=1e-5):
    moved = [[a + (s * h * u if i == at else 0.0) for i, a in enumerate(args)] for s in (1, -1)]
    return (f(*moved[0]) - f(*moved[1])) / (2 * h)


def test_formulas_against_differences():
    rs = np.random.RandomState(0)
    n, f = 5, 9
    x, w = rs.standard_normal((n, f)), rs.standard_normal((n, f))
    gamma, beta = rs.standard_normal((1, f)), rs.standard_normal((1, f))
    _, mean, var = ref.ln(x, gamma, beta, 1e-3)
    grads = ref.ln_grad(w, x, mean, var, gamma, 1e-3)
    for at, g in enumerate(grads):
        u = rs.standard_normal(g.shape)
        s = _slope(lambda *a: (ref.ln(*a, 1e-3)[0] * w).sum(), (x, gamma, beta), at, u)
        assert abs(s - (g * u).sum()) < 1e-7
    z, t, weight = rs.standard_normal((n, 30)), rs.standard_normal((n, 4)), rs.rand(n, 1)
    ids = rs.randint(-1, 30, (n, 4))
    ids[1], ids[2, :2] = -1, 3
    _, stats = ref.distill(z, ids, t, 1.7)
    g, u = ref.distill_grad(z, ids, t, stats, weight, 1.7), rs.standard_normal(z.shape)
    assert abs(_slope(lambda a: (ref.distill(a, ids, t, 1.7)[0] * weight).sum(), (z,), 0, u) - (g * u).sum()) < 1e-7
    W, err, words = rs.standard_normal((7, 3)), rs.standard_normal((n, 3)), np.array([1, 5, 1, 9, -1])
    g, u = ref.table_grad(W * 0, err, words, 2.0, 0.0, 5), rs.standard_normal(W.shape)
    assert abs(_slope(lambda a: (ref.lookup(a, words, 2.0, 5) * err).sum(), (W,), 0, u) - (g * u).sum()) < 1e-8
