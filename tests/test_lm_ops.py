"""Layer normalisation, embedding lookup / table gradient and distillation on
the GPU against float64 formulas (``lm_reference``), at the sizes, layouts, types
and masks where such kernels go wrong.  Inputs are rounded to the storage type
first, so a bound counts the kernels' own roundings only."""
import ctypes

import numpy as np
import pytest

import lm_reference as ref
from neon_amd.backends import bfloat16
from neon_amd.backends.hip import bf16 as host_bf16
from neon_amd.backends.hip import runtime as hiprt

pytestmark = pytest.mark.gpu

F32, F16 = "float32", "float16"
BF16 = "bfloat16"
DTYPES = [F32, F16, BF16]
EPS = 1e-5


def np_dtype(name):
    return bfloat16 if name == BF16 else np.dtype(name)


def quantise(a, name):
    """the values a tensor of that type holds for ``a``, as float64"""
    if name == BF16:
        return host_bf16.quantise(np.asarray(a, np.float32)).astype(np.float64)
    return np.asarray(a).astype(np.float32).astype(name).astype(np.float64)


def place(be, a, axis, how, name):
    """(positions, values) host values -> a device matrix for ``axis`` whose
    memory is laid out as ``how`` says; None: uninitialised"""
    n, f = a.shape if isinstance(a, np.ndarray) else a
    shape = (f, n) if axis == 0 else (n, f)
    dt = np_dtype(name)
    if how == "plain":
        t = be.empty(shape, dtype=dt)
    elif how == "turned":
        t = be.empty(shape[::-1], dtype=dt).T
    elif how == "window":             # lines further apart than they are long, odd starts
        t = be.empty((shape[0] + 2, shape[1] + 5), dtype=dt)[1:1 + shape[0], 3:3 + shape[1]]
    elif how == "sparse":             # strides along both axes
        t = be.empty((2 * shape[0], 2 * shape[1]), dtype=dt)[::2, ::2]
    if isinstance(a, np.ndarray):
        v = be.array(np.ascontiguousarray(a.T if axis == 0 else a).astype(np.float32), dtype=dt)
        t[:] = v
    elif shape[0] and shape[1]:
        t[:] = 77.0
    return t


def vec(be, a, axis, name=F32):
    """(1, values) or (positions, 1) host values -> device matrix"""
    a = np.asarray(a, np.float64)
    return be.array(np.ascontiguousarray(a.T if axis == 0 else a).astype(np.float32), dtype=np_dtype(name))


def host(t, axis):
    g = np.asarray(t.get(), np.float64)
    return g.T if axis == 0 else g


# ---- layer normalisation -------------------------------------------------------------------
def ln_inputs(n, f, name, seed=0, shift=0.5):
    rs = np.random.RandomState(seed + 7 * n + f)
    x = quantise(rs.standard_normal((n, f)) * 2 + shift, name)
    dy = quantise(rs.standard_normal((n, f)) * 0.3, name)
    gamma = (rs.rand(1, f) + 0.5).astype(np.float32).astype(np.float64)
    beta = (rs.standard_normal((1, f)) * 0.1).astype(np.float32).astype(np.float64)
    return x, dy, gamma, beta


def run_ln(be, x, dy, gamma, beta, axis, how, name, eps=EPS):
    n, f = x.shape
    tx, ty = place(be, x, axis, how, name), place(be, (n, f), axis, how, name)
    one_f, one_n = ((f, 1), (1, n)) if axis == 0 else ((1, f), (n, 1))
    g, b = vec(be, gamma, axis), vec(be, beta, axis)
    mean, var = be.empty(one_n), be.empty(one_n)
    be.compound_fprop_ln(tx, mean, var, g, b, ty, eps, axis=axis)
    td, tdx = place(be, dy, axis, how, name), place(be, (n, f), axis, how, name)
    dg, db = be.empty(one_f), be.empty(one_f)
    be.compound_bprop_ln(tdx, dg, db, td, tx, mean, var, g, eps, axis=axis)
    return [host(t, axis) for t in (ty, mean, var, tdx, dg, db)]


def check_ln(got, x, dy, gamma, beta, name, eps=EPS):
    y, mean, var, dx, dg, db = got
    want = ref.ln(x, gamma, beta, eps)
    e_y, e_mean, e_var = ref.ln_bounds(x, gamma, beta, eps)
    ref.within(mean, want[1], e_mean, "mean")
    ref.within(var, want[2], e_var, "var")
    ref.within(y, want[0], ref.stored(want[0], name, e_y), "y")
    # backward from the statistics that were saved
    grads = ref.ln_grad(dy, x, mean, var, gamma, eps)
    e_dx, e_dg, e_db = ref.ln_grad_bounds(dy, x, mean, var, gamma, eps)
    ref.within(dx, grads[0], ref.stored(grads[0], name, e_dx), "dx")
    ref.within(dg, grads[1], e_dg, "dgamma")
    ref.within(db, grads[2], e_db, "dbeta")


LN_SIZES = [(1, 1), (1, 5), (7, 1), (3, 2), (64, 5), (5, 64), (33, 127), (130, 256), (65, 257), (64, 513), (128, 1000),
            (40, 1025), (77, 1537), (9, 2049), (600, 48), (3, 4097), (6, 5000), (2, 8191), (3, 16385), (2, 33000)]


@pytest.mark.parametrize("name", DTYPES)
@pytest.mark.parametrize("n,f", LN_SIZES)
def test_layer_norm(hip, n, f, name):
    x, dy, gamma, beta = ln_inputs(n, f, name)
    for axis in (0, 1):
        for how in ("plain", "turned"):
            check_ln(run_ln(hip, x, dy, gamma, beta, axis, how, name), x, dy, gamma, beta, name)


@pytest.mark.parametrize("name", DTYPES)
@pytest.mark.parametrize("how", ["window", "sparse"])
@pytest.mark.parametrize("n,f", [(1, 3), (37, 19), (130, 300), (5, 1100), (70, 2049)])
def test_layer_norm_on_views(hip, n, f, how, name):
    x, dy, gamma, beta = ln_inputs(n, f, name)
    for axis in (0, 1):
        check_ln(run_ln(hip, x, dy, gamma, beta, axis, how, name), x, dy, gamma, beta, name)


@pytest.mark.parametrize("name", DTYPES)
def test_layer_norm_of_very_long_positions(hip, name):
    for n, f in ((3, 70001), (2, 131072)):
        x, dy, gamma, beta = ln_inputs(n, f, name)
        for axis in (0, 1):
            check_ln(run_ln(hip, x, dy, gamma, beta, axis, "plain", name), x, dy, gamma, beta, name)


@pytest.mark.parametrize("n,f", [(40000, 24), (3000, 700), (2600, 4100)])
def test_layer_norm_of_many_positions(hip, n, f):
    """more positions than workgroups, in both layouts"""
    x, dy, gamma, beta = ln_inputs(n, f, F16)
    for axis in (0, 1):
        check_ln(run_ln(hip, x, dy, gamma, beta, axis, "plain", F16), x, dy, gamma, beta, F16)


def test_layer_norm_keeps_small_deviations_of_large_means(hip):
    x, dy, gamma, beta = ln_inputs(50, 700, F32, shift=3000.0)
    for axis in (0, 1):
        check_ln(run_ln(hip, x, dy, gamma, beta, axis, "plain", F32), x, dy, gamma, beta, F32)


def test_layer_norm_of_equal_features(hip):
    """a variance of exactly zero: y is beta, gradients stay finite"""
    x, dy, gamma, beta = ln_inputs(6, 96, F32)
    x[:] = np.arange(6)[:, None] * 0.25
    for axis in (0, 1):
        got = run_ln(hip, x, dy, gamma, beta, axis, "plain", F32)
        assert np.array_equal(got[0], np.broadcast_to(beta, x.shape))
        assert not got[2].any()
        check_ln(got, x, dy, gamma, beta, F32)


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("f", [70, 1500, 20000])
def test_layer_norm_keeps_a_bad_position_to_itself(hip, bad, f):
    x, dy, gamma, beta = ln_inputs(5, f, F32)
    clean = [run_ln(hip, x, dy, gamma, beta, axis, "plain", F32) for axis in (0, 1)]
    x[2, f // 2] = bad
    for axis in (0, 1):
        got = run_ln(hip, x, dy, gamma, beta, axis, "plain", F32)
        others = [0, 1, 3, 4]
        for k in (0, 1, 2, 3):
            assert np.array_equal(got[k][others], clean[axis][k][others])
        assert np.isnan(got[0][2]).all() and np.isnan(got[3][2]).all() and np.isnan(got[4]).all()
        assert np.array_equal(got[5], clean[axis][5])


@pytest.mark.parametrize("n,f", [(20, 90), (70, 1300), (3, 17000)])
def test_layer_norm_in_place(hip, n, f):
    be = hip
    x, dy, gamma, beta = ln_inputs(n, f, F16)
    for axis in (0, 1):
        want = run_ln(be, x, dy, gamma, beta, axis, "plain", F16)
        g, b = vec(be, gamma, axis), vec(be, beta, axis)
        mean, var = vec(be, want[1], axis), vec(be, want[2], axis)
        dg, db = be.empty(g.shape), be.empty(g.shape)
        tx, td = place(be, x, axis, "plain", F16), place(be, dy, axis, "plain", F16)
        be.compound_bprop_ln(td, dg, db, td, tx, mean, var, g, EPS, axis=axis)
        for t, w in ((td, want[3]), (dg, want[4]), (db, want[5])):
            assert np.array_equal(host(t, axis), w)
        td = place(be, dy, axis, "plain", F16)
        be.compound_bprop_ln(tx, dg, db, td, tx, mean, var, g, EPS, axis=axis)
        for t, w in ((tx, want[3]), (dg, want[4]), (db, want[5])):
            assert np.array_equal(host(t, axis), w)
        tx = place(be, x, axis, "plain", F16)
        be.compound_fprop_ln(tx, mean, var, g, b, tx, EPS, axis=axis)
        assert np.array_equal(host(tx, axis), want[0])


def test_layer_norm_without_positions(hip):
    for axis in (0, 1):
        e = hip.empty((8, 0) if axis == 0 else (0, 8))
        s = hip.empty((1, 0) if axis == 0 else (0, 1))
        g = vec(hip, np.ones((1, 8)), axis)
        hip.compound_fprop_ln(e, s, s, g, g, e, EPS, axis=axis)
        dg, db = vec(hip, np.ones((1, 8)), axis), vec(hip, np.ones((1, 8)), axis)
        hip.compound_bprop_ln(e, dg, db, e, e, s, s, g, EPS, axis=axis)
        assert not dg.get().any() and not db.get().any()


def test_layer_norm_vectors_with_gaps(hip):
    """parameters and statistics that are columns of wider matrices"""
    be, n, f = hip, 33, 65
    x, dy, gamma, beta = ln_inputs(n, f, F32)
    want = run_ln(be, x, dy, gamma, beta, 1, "plain", F32)
    params, stats, grads = be.empty((3, 2 * f)), be.empty((n, 4)), be.zeros((2, 3 * f))
    g, b = params[0:1, ::2], params[2:3, ::2]
    g[:], b[:] = vec(be, gamma, 1), vec(be, beta, 1)
    mean, var = stats[:, 1:2], stats[:, 3:4]
    y = be.empty((n, f))
    tx, td = place(be, x, 1, "plain", F32), place(be, dy, 1, "plain", F32)
    be.compound_fprop_ln(tx, mean, var, g, b, y, EPS, axis=1)
    dg, db = grads[0:1, ::3], grads[1:2, 1::3]
    dx = be.empty((n, f))
    be.compound_bprop_ln(dx, dg, db, td, tx, mean, var, g, EPS, axis=1)
    for t, w in zip((y, mean, var, dx, dg, db), want):
        assert np.array_equal(host(t, 1), w)
    assert not grads.get()[0, 1::3].any()


def test_layer_norm_is_reproducible(hip):
    for n, f in ((5000, 300), (700, 1100)):
        x, dy, gamma, beta = ln_inputs(n, f, BF16)
        for axis in (0, 1):
            a, b = (run_ln(hip, x, dy, gamma, beta, axis, "plain", BF16) for _ in range(2))
            for p, q in zip(a, b):
                assert np.array_equal(p, q)


# ---- embedding -----------------------------------------------------------------------------------
def ids_of(kind, count, vocab, rs):
    if kind == "uniform":
        return rs.randint(0, vocab, count)
    if kind == "one":
        return np.full(count, vocab // 2)
    if kind == "skewed":
        return np.minimum((rs.pareto(0.6, count)).astype(np.int64), vocab - 1)
    if kind == "outside":
        ids = rs.randint(0, vocab, count)
        ids[::3] = rs.choice([-1, vocab, -2 ** 31, 2 ** 31 - 1, vocab + 1], len(ids[::3]))
        return ids
    if kind == "sorted":
        return np.sort(rs.randint(0, vocab, count))
    if kind == "runs":                  # words that end exactly where runs of 32 sorted positions do
        return np.repeat(np.arange(count // 32 + 1) % vocab, 32)[:count]
    raise ValueError(kind)


def run_lut(be, W, err, dW, ids, axis, how, name, pad, scale, beta):
    (vocab, embed), n = W.shape, len(ids)
    tw, ti = place(be, W, 1, "plain", name), be.array(ids.reshape(1, -1).astype(np.int32), dtype=np.int32)
    out = place(be, (n, embed), axis, how, name)
    be.compound_fprop_lut(ti, tw, out, pad_idx=pad, scale=scale, axis=axis)
    te, td = place(be, err, axis, how, name), place(be, dW, 1, "plain", name)
    be.compound_update_lut(ti, te, td, pad_idx=pad, scale=scale, beta=beta, axis=axis)
    return host(out, axis), host(td, 1)


def check_lut(got, W, err, dW, ids, name, pad, scale, beta):
    s = float(np.float32(scale))
    want = ref.lookup(W, ids, s, pad)
    ref.within(got[0], want, ref.stored(want, name, np.abs(want) * ref.U), "lookup")
    b = float(np.float32(beta))
    want = ref.table_grad(dW, err, ids, s, b, pad)
    ref.within(got[1], want, ref.stored(want, name, ref.table_grad_bound(dW, err, ids, s, b, pad)), "table gradient")


def lut_inputs(vocab, embed, count, name, kind, seed=0):
    rs = np.random.RandomState(seed + vocab + embed + count)
    W, dW = quantise(rs.standard_normal((vocab, embed)), name), quantise(rs.standard_normal((vocab, embed)), name)
    return W, quantise(rs.standard_normal((count, embed)), name), dW, ids_of(kind, count, vocab, rs)


@pytest.mark.parametrize("name", DTYPES)
@pytest.mark.parametrize("kind", ["uniform", "one", "skewed", "outside", "sorted", "runs"])
@pytest.mark.parametrize("vocab,embed,count", [(1, 1, 1), (2, 3, 31), (255, 8, 32), (256, 64, 33), (257, 65, 64),
                                               (1000, 300, 1000), (70000, 20, 5000), (300, 1030, 700), (50, 513, 2000)])
def test_embedding(hip, vocab, embed, count, kind, name):
    W, err, dW, ids = lut_inputs(vocab, embed, count, name, kind)
    for axis in (0, 1):
        for pad, scale, beta in ((None, 1.0, 0.0), (vocab // 2, 3.5, 0.0), (0, 0.75, 1.0)):
            got = run_lut(hip, W, err, dW, ids, axis, "plain", name, pad, scale, beta)
            check_lut(got, W, err, dW, ids, name, pad, scale, beta)


@pytest.mark.parametrize("how", ["turned", "window", "sparse"])
def test_embedding_on_views(hip, how):
    for name in (F32, BF16):
        W, err, dW, ids = lut_inputs(400, 77, 300, name, "skewed")
        for axis in (0, 1):
            check_lut(run_lut(hip, W, err, dW, ids, axis, how, name, 3, 2.0, 0.5), W, err, dW, ids, name, 3, 2.0, 0.5)


def test_embedding_table_views(hip):
    """tables that are windows of larger ones: neighbours keep their values"""
    be, vocab, embed, count = hip, 90, 50, 333
    W, err, dW, ids = lut_inputs(vocab, embed, count, F32, "skewed")
    big = be.array(np.full((vocab + 4, embed + 7), 5.0, np.float32))
    ti = be.array(ids.reshape(-1, 1).astype(np.int32), dtype=np.int32)
    te = place(be, err, 1, "plain", F32)
    for beta in (0.0, 1.0, -0.5):
        big[:] = 5.0
        win = big[2:2 + vocab, 3:3 + embed]
        win[:] = place(be, dW, 1, "plain", F32)
        be.compound_update_lut(ti, te, win, scale=1.5, beta=beta, axis=1)
        got = big.get()
        want = ref.table_grad(dW, err, ids, 1.5, beta, None)
        ref.within(got[2:2 + vocab, 3:3 + embed], want, ref.table_grad_bound(dW, err, ids, 1.5, beta, None))
        got[2:2 + vocab, 3:3 + embed] = 5.0
        assert (got == 5.0).all()
        # a transposed table, and ids with a stride
        turned = place(be, dW, 1, "turned", F32)
        wide = be.zeros((count, 3), dtype=np.int32)
        wide.set(np.stack([ids * 0 + 1, ids, ids * 0 + 2], 1).astype(np.int32))
        be.compound_update_lut(wide[:, 1:2], te, turned, scale=1.5, beta=beta, axis=1)
        ref.within(host(turned, 1), want, ref.table_grad_bound(dW, err, ids, 1.5, beta, None))
        out = be.empty((count, embed))
        be.compound_fprop_lut(wide[:, 1:2], turned, out, axis=1)
        assert np.array_equal(out.get(), turned.get()[ids])


def test_embedding_gradient_without_positions(hip):
    for beta, want in ((0.0, 0.0), (1.0, 3.0), (0.5, 1.5)):
        dW = hip.empty((70, 9))
        dW[:] = 3.0
        hip.compound_update_lut(hip.empty((1, 0), dtype=np.int32), hip.empty((9, 0)), dW, beta=beta)
        assert (dW.get() == want).all()
    W = hip.ones((70, 9))
    hip.compound_fprop_lut(hip.empty((1, 0), dtype=np.int32), W, hip.empty((9, 0)))


def test_embedding_padding_hides_bad_values(hip):
    """NaN and infinities in padded positions' errors and in the padding row"""
    be, vocab, embed, count = hip, 40, 24, 200
    W, err, dW, ids = lut_inputs(vocab, embed, count, F32, "uniform")
    ids[::4] = 7
    W[7] = np.nan
    err[::8], err[4::8] = np.nan, np.inf
    ids[1::50], err[1::50] = -1, np.nan
    for axis in (0, 1):
        out, grad = run_lut(be, W, err, dW, ids, axis, "plain", F32, 7, 2.0, 0.0)
        assert np.isfinite(out).all() and np.isfinite(grad).all()
        assert not grad[7].any() and not out[ids == 7].any() and not out[ids == -1].any()
    # and beta = 0 does not read what dW held
    dW[:] = np.nan
    assert np.isfinite(run_lut(be, W, err, dW, ids, 1, "plain", F32, 7, 2.0, 0.0)[1]).all()


def test_embedding_gradient_of_ones_counts(hip):
    for vocab, count in ((3000, 40000), (100000, 60000)):
        rs = np.random.RandomState(1)
        ids = ids_of("skewed", count, vocab, rs)
        dW = hip.empty((vocab, 5))
        hip.compound_update_lut(hip.array(ids.reshape(1, -1).astype(np.int32), dtype=np.int32), hip.ones((5, count)), dW)
        assert np.array_equal(dW.get(), np.repeat(np.bincount(ids, minlength=vocab)[:, None], 5, 1).astype(np.float32))


def test_embedding_gradient_is_reproducible(hip):
    W, err, dW, ids = lut_inputs(500, 130, 9000, F32, "skewed")
    a, b = (run_lut(hip, W, err, dW, ids, 0, "plain", F32, 1, 0.3, 0.0)[1] for _ in range(2))
    assert np.array_equal(a, b)


# ---- distillation ------------------------------------------------------------------------------------
def distill_inputs(n, vocab, k, name, t_name, seed=0, spread=3.0):
    rs = np.random.RandomState(seed + n + vocab + k)
    z = quantise(rs.standard_normal((n, vocab)) * spread, name)
    t = quantise(rs.standard_normal((n, k)) * 2 + 4, t_name)
    ids = rs.randint(0, vocab, (n, k))
    if k:
        ids[rs.rand(n, k) < 0.2] = -1                                  # entries that stand for nothing
        ids[rs.rand(n, k) < 0.05] = vocab + 3
        ids[n // 2] = -1                                               # a position without entries
        if k > 2:
            ids[0, 2] = ids[0, 0] = vocab - 1                          # a word named twice
    weight = (rs.rand(n, 1) + 0.5).astype(np.float32).astype(np.float64)
    return z, ids, t, weight


def run_distill(be, z, ids, t, weight, tau, axis, how, name, t_name):
    n, vocab = z.shape
    k = ids.shape[1]
    tz = place(be, z, axis, how, name)
    ti = be.array(np.ascontiguousarray(ids.T if axis == 0 else ids).astype(np.int32), dtype=np.int32) if k else \
        be.empty((0, n) if axis == 0 else (n, 0), dtype=np.int32)
    tt = place(be, t, axis, "plain", t_name) if k else be.empty((0, n) if axis == 0 else (n, 0), dtype=np_dtype(t_name))
    loss = be.empty((1, n) if axis == 0 else (n, 1))
    stats = be.empty((4, n) if axis == 0 else (n, 4))
    be.compound_fprop_distill(tz, ti, tt, loss, stats, temperature=tau, axis=axis)
    delta = place(be, (n, vocab), axis, how, name)
    tw = vec(be, weight, axis) if isinstance(weight, np.ndarray) else weight
    be.compound_bprop_distill(delta, tz, ti, tt, stats, tw, temperature=tau, axis=axis)
    return host(loss, axis), host(stats, axis), host(delta, axis)


def check_distill(got, z, ids, t, weight, tau, name):
    loss, stats, delta = got
    tau = float(np.float32(tau))
    want = ref.distill(z, ids, t, tau)
    e = ref.distill_bounds(z, ids, t, tau)
    ref.within(stats, want[1], e[1], "stats")
    ref.within(loss, want[0], e[0], "loss")
    grad = ref.distill_grad(z, ids, t, stats, weight, tau)
    ref.within(delta, grad, ref.stored(grad, name, ref.distill_grad_bound(z, ids, t, stats, weight, tau)), "delta")


@pytest.mark.parametrize("name", DTYPES)
@pytest.mark.parametrize("n,vocab,k", [(1, 1, 1), (2, 2, 3), (5, 7, 2), (3, 64, 0), (64, 63, 5), (65, 65, 64), (130, 257, 3),
                                       (33, 1000, 65), (6, 4097, 257), (2, 32001, 32), (70, 9000, 16), (1, 70000, 1024)])
def test_distillation(hip, n, vocab, k, name):
    z, ids, t, weight = distill_inputs(n, vocab, k, name, name)
    for axis in (0, 1):
        for how in ("plain", "turned"):
            for tau in (1.0, 3.0):
                check_distill(run_distill(hip, z, ids, t, weight, tau, axis, how, name, name), z, ids, t, weight, tau, name)


@pytest.mark.parametrize("n,vocab,k", [(4100, 70, 9), (4097, 50, 600), (4099, 33, 1024), (9, 3, 300), (300, 40, 1024), (2, 20000, 1000)])
def test_distillation_of_many_positions_and_repeated_words(hip, n, vocab, k):
    """entries of 16 positions at a time; words named once, many times, by every entry"""
    z, ids, t, weight = distill_inputs(n, vocab, k, F32, F32)
    ids[1] = vocab - 1
    for axis in (0, 1):
        check_distill(run_distill(hip, z, ids, t, weight, 1.0, axis, "plain", F32, F32), z, ids, t, weight, 1.0, F32)


@pytest.mark.parametrize("how", ["window", "sparse"])
@pytest.mark.parametrize("name,t_name", [(F32, F16), (F16, F32), (BF16, F32)])
def test_distillation_on_views(hip, how, name, t_name):
    for n, vocab, k in ((9, 130, 4), (67, 1031, 20)):
        z, ids, t, weight = distill_inputs(n, vocab, k, name, t_name)
        for axis in (0, 1):
            check_distill(run_distill(hip, z, ids, t, weight, 0.5, axis, how, name, t_name), z, ids, t, weight, 0.5, name)


def test_distillation_of_small_tensors_with_gaps(hip):
    """ids, teacher logits, loss, statistics and weights as parts of larger tensors"""
    be, n, vocab, k = hip, 21, 300, 6
    z, ids, t, weight = distill_inputs(n, vocab, k, F32, F32)
    for axis in (0, 1):
        want = run_distill(be, z, ids, t, weight, 2.0, axis, "plain", F32, F32)
        cut = (slice(1, None, 2), slice(None, None, 3)) if axis == 0 else (slice(None, None, 3), slice(1, None, 2))

        def wide(rows, cols, dtype=np.float32):
            shape = (2 * rows + 1, 3 * cols) if axis == 0 else (3 * cols, 2 * rows + 1)
            big = be.empty(shape, dtype=dtype)
            big[:] = 9
            return big, big[cut]
        (bi, wi), (bt, wt) = wide(k, n, np.int32), wide(k, n)
        h = np.full(bi.shape, 9, np.int32)
        h[cut] = ids.T if axis == 0 else ids
        bi.set(h)
        h = np.full(bt.shape, 9, np.float32)
        h[cut] = t.T if axis == 0 else t
        bt.set(h)
        (bl, wl), (bs, ws), (bw, ww) = wide(1, n), wide(4, n), wide(1, n)
        h = np.full(bw.shape, 9, np.float32)
        h[cut] = weight.T if axis == 0 else weight
        bw.set(h)
        tz, delta = place(be, z, axis, "plain", F32), place(be, z.shape, axis, "plain", F32)
        be.compound_fprop_distill(tz, wi, wt, wl, ws, temperature=2.0, axis=axis)
        be.compound_bprop_distill(delta, tz, wi, wt, ws, ww, temperature=2.0, axis=axis)
        assert np.array_equal(host(wl, axis), want[0]) and np.array_equal(host(ws, axis), want[1])
        assert np.array_equal(host(delta, axis), want[2])
        for big, view in ((bl, wl), (bs, ws)):
            g = big.get()
            g[cut] = 9
            assert (g == 9).all()


def test_distillation_masks(hip):
    """-inf among the student's and the teacher's logits, NaN where nothing counts"""
    n, vocab, k = 8, 500, 10
    z, ids, t, weight = distill_inputs(n, vocab, k, F32, F32)
    ids[:] = np.arange(k) * 7
    z[1, 100:400] = -np.inf                      # words the student may not use
    z[2] = -3.4028234663852886e38                # all at the lowest value of the type
    z[3, :] = -np.inf
    z[3, 7] = 1.0                                # one word left
    t[3, [0] + list(range(2, k))] = -np.inf
    t[4] = -np.inf                               # a teacher that says nothing: no loss, no gradient
    t[5, 3:] = -np.inf
    ids[6] = -1
    z[6] = np.nan                                # padding behind the end of a sequence
    t[6] = np.nan
    ids[7, 5:] = -5
    t[7, 5:] = np.nan
    for axis in (0, 1):
        for tau in (1.0, 2.0):
            got = run_distill(hip, z, ids, t, weight, tau, axis, "plain", F32, F32)
            check_distill(got, z, ids, t, weight, tau, F32)
            assert not got[2][[4, 6]].any() and not got[0][[4, 6]].any()
            assert abs(got[0][3, 0]) < 1e-5
    # what reaches a position that counts stays there
    z[0, 3], z[1, 499] = np.nan, np.inf
    for axis in (0, 1):
        loss, stats, delta = run_distill(hip, z, ids, t, weight, 1.0, axis, "plain", F32, F32)
        assert np.isnan(loss[:2]).all() and np.isnan(delta[:2]).all() and np.isfinite(loss[[4, 5, 6, 7]]).all()
    # a word with no probability left that the teacher wants: an infinite loss
    z[0, 3], z[1, 499] = 0.0, 0.0
    z[0, 14] = -np.inf
    for axis in (0, 1):
        loss, _, delta = run_distill(hip, z, ids, t, weight, 1.0, axis, "plain", F32, F32)
        assert loss[0, 0] == np.inf and np.isfinite(delta[0]).all()


@pytest.mark.parametrize("size", [40.0, 2000.0, 1e6])
def test_distillation_of_large_logits(hip, size):
    z, ids, t, weight = distill_inputs(7, 900, 12, F32, F32, spread=size)
    z = quantise(z + size, F32)           # (the values the tensor will hold)
    for axis in (0, 1):
        check_distill(run_distill(hip, z, ids, t, weight, 1.0, axis, "plain", F32, F32), z, ids, t, weight, 1.0, F32)


def test_distillation_with_one_weight_for_all(hip):
    z, ids, t, _ = distill_inputs(12, 400, 5, F16, F16)
    for axis in (0, 1):
        for w in (1.0, 0.25, 0.0, -2):
            check_distill(run_distill(hip, z, ids, t, w, 1.0, axis, "plain", F16, F16), z, ids, t, w, 1.0, F16)


def test_distillation_without_positions(hip):
    for axis in (0, 1):
        def e(rows, dtype=np.float32):
            return hip.empty((rows, 0) if axis == 0 else (0, rows), dtype=dtype)
        hip.compound_fprop_distill(e(50), e(3, np.int32), e(3), e(1), e(4), axis=axis)
        hip.compound_bprop_distill(e(50), e(50), e(3, np.int32), e(3), e(4), axis=axis)


def test_distillation_gradient_against_differences(hip):
    """central differences of the kernel's own loss along random directions"""
    rs = np.random.RandomState(3)
    z, ids, t, weight = distill_inputs(6, 40, 5, F32, F32, spread=1.0)
    for axis in (0, 1):
        _, _, delta = run_distill(hip, z, ids, t, weight, 2.0, axis, "plain", F32, F32)
        for _ in range(4):
            v = rs.standard_normal(z.shape)
            h = 2.0 ** -6
            hi, lo = (quantise(z + s * h * v, F32) for s in (1, -1))
            up, down = (run_distill(hip, w, ids, t, weight, 2.0, axis, "plain", F32, F32)[0] for w in (hi, lo))
            slope = ((up - down) * weight).sum() / (2 * h)
            # third derivatives of a log-sum-exp along v are at most max|v|^3 / T^3 (T^2 in front); fp32
            # losses of size L are off by some 1e-6 L each
            bound = h * h * (np.abs(v).max(1) ** 3).sum() * 1.5 / 2.0 + 1e-5 * np.abs(up).sum() / h
            assert abs(slope - (delta * v).sum()) <= bound


# ---- offsets behind 2^32 bytes and 2^31 elements --------------------------------------------------------
def test_lines_far_apart(hip):
    """operands whose lines lie 1.2e9 elements apart in one large allocation"""
    be, ld, lines, width = hip, 1200000000, 4, 300
    big = [be.empty((lines, ld), dtype=np.float16) for _ in range(2)]

    def put(k, a):
        for i in range(lines):
            be.rt.memcpy_h2d(big[k].gpudata + 2 * (i * ld + 7), np.ascontiguousarray(a[i].astype(np.float16)))
        return big[k][:, 7:7 + width]

    def got(k):
        out = np.empty((lines, width), np.float16)
        be.synchronize()
        for i in range(lines):
            be.rt.memcpy_d2h(out[i], big[k].gpudata + 2 * (i * ld + 7))
        return out.astype(np.float64)

    def plain(a, dtype=np.float16):
        return be.array(np.ascontiguousarray(a).astype(np.float32), dtype=dtype)
    for axis in (1, 0):               # lines are positions, then features
        x, dy, gamma, beta = ln_inputs(lines, width, F16) if axis == 1 else ln_inputs(width, lines, F16)
        X, D = (a if axis == 1 else a.T for a in (x, dy))
        one_n = (lines, 1) if axis == 1 else (1, width)
        g, b, mean, var = vec(be, gamma, axis), vec(be, beta, axis), be.empty(one_n), be.empty(one_n)
        tx, ty = put(0, X), put(1, X)
        be.compound_fprop_ln(tx, mean, var, g, b, ty, EPS, axis=axis)
        y = got(1)
        dg, db = be.empty(g.shape), be.empty(g.shape)
        be.compound_bprop_ln(ty, dg, db, plain(D), tx, mean, var, g, EPS, axis=axis)
        dx = got(1)
        check_ln([y if axis == 1 else y.T, host(mean, axis), host(var, axis), dx if axis == 1 else dx.T, host(dg, axis),
                  host(db, axis)], x, dy, gamma, beta, F16)
    W, err, dW, ids = lut_inputs(lines, width, 50, F16, "outside")
    ti, out = be.array(ids.reshape(1, -1).astype(np.int32), dtype=np.int32), be.empty((50, width), dtype=np.float16)
    be.compound_fprop_lut(ti, put(0, W), out, axis=1)
    be.compound_update_lut(ti, plain(err), put(1, dW), beta=1.0, axis=1)
    check_lut([host(out, 1), got(1)], W, err, dW, ids, F16, None, 1.0, 1.0)
    for axis in (1, 0):
        z, tids, t, weight = distill_inputs(lines, width, 5, F16, F16) if axis == 1 else \
            distill_inputs(width, lines, 5, F16, F16)
        n = len(z)
        Z = z if axis == 1 else z.T
        tt, loss = plain(t if axis == 1 else t.T), be.empty((n, 1) if axis == 1 else (1, n))
        td = be.array(np.ascontiguousarray(tids if axis == 1 else tids.T).astype(np.int32), dtype=np.int32)
        stats = be.empty((n, 4) if axis == 1 else (4, n))
        tz, delta = put(0, Z), put(1, Z)
        be.compound_fprop_distill(tz, td, tt, loss, stats, axis=axis)
        be.compound_bprop_distill(delta, tz, td, tt, stats, vec(be, weight, axis), axis=axis)
        d = got(1)
        check_distill([host(loss, axis), host(stats, axis), d if axis == 1 else d.T], z, tids, t, weight, 1.0, F16)


# ---- in a row, as they are used ------------------------------------------------------------------------
def test_a_training_step(hip):
    """embedding -> layer norm -> product -> distillation, and back to the table,
    in the backend's own layout, against float64"""
    be = hip
    rs = np.random.RandomState(11)
    vocab, embed, n, k, tau, scale, pad = 301, 48, 90, 7, 2.0, np.sqrt(48.0), 0
    ids = ids_of("skewed", n, vocab, rs).astype(np.int32)
    W = (rs.standard_normal((vocab, embed)) * 0.2).astype(np.float32)
    P = (rs.standard_normal((vocab, embed)) * 0.1).astype(np.float32)
    gamma, beta = (rs.rand(embed, 1) + 0.5).astype(np.float32), (rs.standard_normal((embed, 1)) * 0.1).astype(np.float32)
    tids, t = rs.randint(0, vocab, (k, n)).astype(np.int32), (rs.standard_normal((k, n)) * 2).astype(np.float32)
    tids[:, ids == pad] = -1                                            # padding does not train
    d = {name: be.array(a, dtype=a.dtype) for name, a in dict(W=W, P=P, gamma=gamma, beta=beta, t=t).items()}
    dids, dtids = be.array(ids.reshape(1, n), dtype=np.int32), be.array(tids, dtype=np.int32)
    x, y, z = be.empty((embed, n)), be.empty((embed, n)), be.empty((vocab, n))
    mean, var, loss, stats = be.empty((1, n)), be.empty((1, n)), be.empty((1, n)), be.empty((4, n))
    dz, dyy, dxx = be.empty((vocab, n)), be.empty((embed, n)), be.empty((embed, n))
    dP, dW, dg, db = be.empty((vocab, embed)), be.empty((vocab, embed)), be.empty((embed, 1)), be.empty((embed, 1))

    def step():
        be.compound_fprop_lut(dids, d["W"], x, pad_idx=pad, scale=scale)
        be.compound_fprop_ln(x, mean, var, d["gamma"], d["beta"], y, EPS)
        be.compound_dot(d["P"], y, z)
        be.compound_fprop_distill(z, dtids, d["t"], loss, stats, temperature=tau)
        be.compound_bprop_distill(dz, z, dtids, d["t"], stats, 1.0, temperature=tau)
        be.compound_dot(dz, y.T, dP)
        be.compound_dot(d["P"].T, dz, dyy)
        be.compound_bprop_ln(dxx, dg, db, dyy, x, mean, var, d["gamma"], EPS)
        be.compound_update_lut(dids, dxx, dW, pad_idx=pad, scale=scale)

    def formula(W, P, gamma, beta):
        X = ref.lookup(W, ids, scale, pad)
        Y, m, v = ref.ln(X, gamma.T, beta.T, EPS)
        Z = Y @ P.T
        return (X, Y, m, v, Z) + ref.distill(Z, tids.T, t.T.astype(np.float64), tau)

    step()
    X, Y, m, v, Z, L, stat = formula(*(a.astype(np.float64) for a in (W, P, gamma, beta)))
    dZ = ref.distill_grad(Z, tids.T, t.T.astype(np.float64), stat, 1.0, tau)
    dY = dZ @ P
    dX, G, B = ref.ln_grad(dY, X, m, v, gamma.T.astype(np.float64), EPS)
    want = dict(loss=L.T, dP=dZ.T @ Y, dgamma=G.T, dbeta=B.T, dW=ref.table_grad(W * 0.0, dX, ids, scale, 0.0, pad))
    got = dict(loss=loss, dP=dP, dgamma=dg, dbeta=db, dW=dW)
    for name in want:
        a, b = got[name].get().astype(np.float64), want[name]
        # fp32 through five stages: some hundred roundings each, 300 u relative to the whole
        assert np.linalg.norm(a - b) <= 300 * ref.U * np.linalg.norm(b), name
    assert not dW.get()[pad].any() and np.linalg.norm(want["dW"]) > 0
    # the formulas' gradients against differences of the formulas' loss
    for name, at in (("dW", 0), ("dP", 1), ("dgamma", 2), ("dbeta", 3)):
        args = [a.astype(np.float64) for a in (W, P, gamma, beta)]
        u = rs.standard_normal(args[at].shape)
        h, sums = 1e-5, []
        for s in (1, -1):
            moved = list(args)
            moved[at] = args[at] + s * h * u
            sums.append(formula(*moved)[5].sum())
        slope = (sums[0] - sums[1]) / (2 * h)
        # (rounding of the sums over 2h; the quadratic term of a smooth function at h = 1e-5)
        assert abs(slope - (want[name] * u).sum()) <= 1e-6 * np.abs(want[name] * u).sum() + 1e-9 * abs(sums[0]) / h
    # a second step on the same tensors gives the same bits
    first = {name: got[name].get() for name in got}
    step()
    for name in got:
        assert np.array_equal(first[name], got[name].get())
    # inside an open fusion scope: what was queued runs first, in order
    with be.fused():
        x[:] = x * 0.0 + 1.0
        be.compound_fprop_ln(x, mean, var, d["gamma"], d["beta"], y, EPS)
        y[:] = y * 2.0
    assert np.array_equal(y.get(), np.broadcast_to(2 * beta, (embed, n)))


# ---- through the C ABI: a stream of the caller's, a graph ------------------------------------------------
class Hip(object):
    """the few runtime calls that record and replay a graph, in the runtime the
    library itself is linked to"""

    def __init__(self):
        self.lib = ctypes.CDLL("libamdhip64.so.7")

    def __getattr__(self, name):
        fn = getattr(self.lib, name)

        def call(*args):
            assert fn(*args) == 0, name
        return call


def test_captured_and_replayed(hip):
    """all operators recorded into one graph on a stream of their own, replayed
    with new inputs between eager calls that have workspaces of their own"""
    be, lib, api = hip, hip.rt.lib, Hip()
    n, f, vocab, embed, k = 300, 200, 500, 64, 5
    rs = np.random.RandomState(0)
    x, dy, gamma, beta = be.empty((f, n)), be.empty((f, n)), be.empty((f, 1)), be.empty((f, 1))
    W, err, z, t = be.empty((vocab, embed)), be.empty((embed, n)), be.empty((vocab, n)), be.empty((k, n))
    ids, tids = be.empty((1, n), dtype=np.int32), be.empty((k, n), dtype=np.int32)

    def fill():
        for v in (x, dy, gamma, beta, W, err, z, t):
            v.set(rs.standard_normal(v.shape).astype(np.float32))
        for v in (ids, tids):
            v.set(rs.randint(0, vocab, v.shape).astype(np.int32))

    def outputs():
        return dict(y=be.empty((f, n)), mean=be.empty((1, n)), var=be.empty((1, n)), dx=be.empty((f, n)), dg=be.empty((f, 1)),
                    db=be.empty((f, 1)), out=be.empty((embed, n)), dW=be.empty((vocab, embed)), loss=be.empty((1, n)),
                    stats=be.empty((4, n)), dz=be.empty((vocab, n)))
    need = [lib.nh_ln_workspace_bytes(b, 0, 0, f, n) for b in (0, 1)] + \
        [lib.nh_embed_update_workspace_bytes(0, 0, n, embed, vocab)] + \
        [lib.nh_distill_workspace_bytes(0, 0, vocab, n)]
    scratch = [[be.empty((b // 4 + 1, 1)) for b in need] for _ in range(2)]
    strides, strides_b = hiprt.int64s(n, 1, n, 1, 1, n, 1), hiprt.int64s(n, 1, n, 1, n, 1, 0)

    def enqueue(o, scratch, s):
        p = {a: v.gpudata for a, v in o.items()}
        w = [(a.gpudata, a.nbytes) for a in scratch]
        X, DY, G, B, TW, E, Z, TT, I, TI = (v.gpudata for v in (x, dy, gamma, beta, W, err, z, t, ids, tids))
        for rc in (
                lib.nh_ln_fprop(p["y"], p["mean"], p["var"], X, G, B, EPS, 0, 0, f, n, n, n, w[0][0], w[0][1], s),
                lib.nh_ln_bprop(p["dx"], p["dg"], p["db"], DY, X, p["mean"], p["var"], G, EPS, 0, 0, f, n, n, n, n,
                                w[1][0], w[1][1], s),
                lib.nh_embed_fprop(p["out"], TW, I, 2.0, 0, 0, n, embed, vocab, embed, n, -1, s),
                lib.nh_embed_update(p["dW"], E, I, 2.0, 0.0, 0, 0, n, embed, vocab, embed, n, 3, w[2][0], w[2][1], s),
                lib.nh_distill_fprop(p["loss"], p["stats"], Z, TI, TT, 2.0, 0, 0, 0, vocab, n, k, n, strides,
                                     w[3][0], w[3][1], s),
                lib.nh_distill_bprop(p["dz"], Z, TI, TT, p["stats"], None, 1.0, 2.0, 0, 0, 0, vocab, n, k, n, n, strides_b,
                                     s)):
            assert rc == 0, lib.nh_last_error()
    eager, recorded = outputs(), outputs()
    fill()
    be.synchronize()
    stream, graph, ready = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
    hiprt.check(lib.nh_stream_create(ctypes.byref(stream)))
    api.hipStreamBeginCapture(stream, 2)                    # relaxed: other calls of the process are not looked at
    enqueue(recorded, scratch[0], stream)
    api.hipStreamEndCapture(stream, ctypes.byref(graph))
    api.hipGraphInstantiate(ctypes.byref(ready), graph, None, None, ctypes.c_size_t(0))
    try:
        for turn in range(4):
            fill()
            for v in recorded.values():
                v[:] = -123.0
            be.synchronize()
            api.hipGraphLaunch(ready, stream)
            enqueue(eager, scratch[1], None)
            hiprt.check(lib.nh_stream_sync(stream))
            be.synchronize()
            for name in eager:
                assert np.array_equal(eager[name].get(), recorded[name].get()), (turn, name)
    finally:
        api.hipGraphExecDestroy(ready)
        api.hipGraphDestroy(graph)
        hiprt.check(lib.nh_stream_destroy(stream))
