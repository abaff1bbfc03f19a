"""The loops of the language-model kernels that only large calls enter, on
positions that repeat 16 different ones: those are checked against the float64
formulas, the others have to give the same bits.  Error bounds count the
additions that the kernels' geometry makes at these sizes (``lm_reference``'s
own count is for short sums)."""
import numpy as np
import pytest

import lm_reference as ref
from test_lm_ops import BF16, EPS, F16, F32, distill_inputs, ln_inputs, np_dtype, place, quantise, vec

pytestmark = pytest.mark.gpu

SAME = 16


def repeated(be, a, n, name, axis=1):
    """positions 0 .. n - 1 of a device matrix with a's 16 positions over and over"""
    f = a.shape[1]
    t = be.empty((n, f) if axis == 1 else (f, n), dtype=np_dtype(name))
    lines = (lambda lo, hi: t[lo:hi]) if axis == 1 else (lambda lo, hi: t[:, lo:hi])
    lines(0, SAME)[:] = vec(be, a, axis, name)
    have = SAME
    while have < n:
        more = min(have, n - have)
        lines(have, have + more)[:] = lines(0, more)
        have += more
    return t


def first_of(t, n, axis=1):
    """the first 16 positions, as float64; the others equal them to the bit"""
    got = t.get()
    got = got if axis == 1 else got.T
    assert n % SAME == 0 and len(got) == n
    tiles = got.reshape(n // SAME, -1)
    for lo in range(0, len(tiles), 256):
        block = tiles[lo:lo + 256]
        assert np.array_equal(block, np.broadcast_to(tiles[0], block.shape), equal_nan=True)
    return got[:SAME].astype(np.float64)


# 16 KB of logits are a batch of a workgroup's loads in the forward pass: an even and an odd number of
# batches, with a rest and without; logits (and logits with their gradients) below and above the 256 MB from
# which the caches are bypassed
@pytest.mark.parametrize("name,n,vocab", [(F32, 1104, 20001), (BF16, 1104, 33000), (F16, 1104, 25000), (F16, 1104, 65536),
                                          (BF16, 1104, 130001), (F32, 1104, 65536)])
def test_distillation_of_long_rows(hip, monkeypatch, name, n, vocab):
    be, k, tau = hip, 40, 2.0
    z, ids, t, weight = distill_inputs(SAME, vocab, k, name, name)
    # a thread adds every 256th logit, and corrects its sum by a factor (6 roundings with its exponent's) where
    # a batch of 16 KB, or one of the vectors behind the last batch, holds a larger one
    batch = 16384 // (4 if name == F32 else 2)
    monkeypatch.setattr(ref, "depth", lambda count: -(-count // 256) + 6 * (-(-count // batch) + 4))
    tz = repeated(be, z, n, name)
    ti = be.array(np.tile(ids, (n // SAME, 1)).astype(np.int32), dtype=np.int32)
    tt, tw = repeated(be, t, n, name), repeated(be, weight, n, F32)
    loss, stats, delta = be.empty((n, 1)), be.empty((n, 4)), be.empty((n, vocab), dtype=np_dtype(name))
    delta[:] = 77.0
    be.compound_fprop_distill(tz, ti, tt, loss, stats, temperature=tau, axis=1)
    be.compound_bprop_distill(delta, tz, ti, tt, stats, tw, temperature=tau, axis=1)
    loss, stats, delta = first_of(loss, n), first_of(stats, n), first_of(delta, n)
    want, bound = ref.distill(z, ids, t, tau), ref.distill_bounds(z, ids, t, tau)
    ref.within(stats, want[1], bound[1], "stats")
    ref.within(loss, want[0], bound[0], "loss")
    grad = ref.distill_grad(z, ids, t, stats, weight, tau)
    ref.within(delta, grad, ref.stored(grad, name, ref.distill_grad_bound(z, ids, t, stats, weight, tau)), "delta")


# ---- layer normalisation -------------------------------------------------------------------
def ceil_div(a, b):
    return -(-a // b)


def position_depth(name, n, f, axis):
    """additions that a position's share of dgamma and dbeta passes through:
    within a thread (and the lanes and waves that share a feature), then over the
    partial rows, of which a thread adds every 128th before 4 + 32 are joined"""
    if axis == 0:                                           # a partial row per strip of 64 bytes of positions
        columns = 16 if name == F32 else 32
        return columns // 4 + 2 + ceil_div(ceil_div(n, columns), 128) + 8
    if f > (8192 if name == F32 else 16384):                # 64 runs of rows
        return ceil_div(n, 64) + 1 + 8
    threads = 64 if f <= 1024 else 256 if f <= 2048 else 512 if f <= 4096 else 1024
    rows = 4 if threads == 64 else 1                        # of a workgroup at a time
    blocks = min(ceil_div(n, 3 * rows), 256 if threads == 1024 else 512)
    return ceil_div(n, blocks * rows) + rows - 1 + ceil_div(blocks, 128) + 8


# 16 features per thread of a whole workgroup (16-bit rows of more than 8192); every number of threads per row
# with more rows than workgroups, outputs that bypass the caches; the form of rows too long for registers
# over many of them; strips of columns by the thousand
@pytest.mark.parametrize("name,n,f,axis", [(F16, 1040, 8200, 1), (BF16, 1040, 16384, 1), (BF16, 131072, 1100, 1),
                                           (F32, 46000, 1500, 1), (F16, 16800, 4000, 1), (F16, 16400, 4104, 1),
                                           (BF16, 340000, 200, 1), (F32, 20000, 8200, 1), (F16, 262144, 100, 0)])
def test_layer_norm_of_many_repeated_positions(hip, monkeypatch, name, n, f, axis):
    be, times = hip, n // SAME
    x, dy, gamma, beta = ln_inputs(SAME, f, name)
    short = ref.depth
    monkeypatch.setattr(ref, "depth", lambda count: position_depth(name, n, f, axis) if count == SAME else short(count))
    tx, td = repeated(be, x, n, name, axis), repeated(be, dy, n, name, axis)
    g, b = vec(be, gamma, axis), vec(be, beta, axis)
    out = be.empty(tx.shape, dtype=np_dtype(name))
    mean, var = (be.empty((n, 1) if axis == 1 else (1, n)) for _ in range(2))
    be.compound_fprop_ln(tx, mean, var, g, b, out, EPS, axis=axis)
    y, mu, v = (first_of(t, n, axis) for t in (out, mean, var))
    want, e = ref.ln(x, gamma, beta, EPS), ref.ln_bounds(x, gamma, beta, EPS)
    ref.within(mu, want[1], e[1], "mean")
    ref.within(v, want[2], e[2], "var")
    ref.within(y, want[0], ref.stored(want[0], name, e[0]), "y")
    out[:] = 77.0
    dg, db = be.empty(g.shape), be.empty(g.shape)
    be.compound_bprop_ln(out, dg, db, td, tx, mean, var, g, EPS, axis=axis)
    dx = first_of(out, n, axis)
    want, e = ref.ln_grad(dy, x, mu, v, gamma, EPS), ref.ln_grad_bounds(dy, x, mu, v, gamma, EPS)
    ref.within(dx, want[0], ref.stored(want[0], name, e[0]), "dx")
    for got, k, what in ((dg, 1, "dgamma"), (db, 2, "dbeta")):
        ref.within(got.get().reshape(1, -1), want[k] * times, e[k] * times, what)


# ---- table gradient ---------------------------------------------------------------------------
def table_depth(counts, positions, embed, name):
    """additions that a position's error passes through: sorted positions are
    added by runs; of a word in several of them, up to 24 partial sums one after
    another, more by sixteen shares"""
    run, tiles = 32, ceil_div(embed, 256 if name == F32 else 512)
    while run > 8 and ceil_div(positions, run) * tiles < 2048:
        run //= 2
    parts = -(-counts // run) + 1
    return np.minimum(counts, np.minimum(counts, run) + np.where(parts <= 25, parts, -(-parts // 16) + 16))


@pytest.mark.parametrize("name,positions,embed", [(F32, 65600, 256), (BF16, 65600, 512), (F32, 9000, 300), (F16, 700, 64)])
def test_table_gradient_of_frequent_words(hip, name, positions, embed):
    """words of 23, 24 and 25 whole runs, and of a third of all positions"""
    be, vocab, scale = hip, 1500, 1.5
    rs = np.random.RandomState(positions)
    run = 32 if positions > 10000 else 8
    ids = rs.randint(0, vocab, positions)
    at = 0
    for word, count in ((7, 23 * run + 5), (700, 24 * run + 3), (1499, 25 * run + 9), (301, positions // 3)):
        count = min(count, positions // 4 if word != 301 else count)
        ids[at:at + count] = word
        at = min(at + count, positions)
    rs.shuffle(ids)
    err = quantise(rs.standard_normal((positions, embed)), name)
    ti = be.array(ids.reshape(1, -1).astype(np.int32), dtype=np.int32)
    counts = np.bincount(ids, minlength=vocab)[:, None]
    want = ref.table_grad(np.zeros((vocab, embed)), err, ids, scale, 0.0, None)
    # (two more roundings: scale times the sum, and the partial sums' own first element)
    bound = (table_depth(counts, positions, embed, name) + 2) * ref.U * scale * ref.table_sums(np.abs(err), ids, vocab, None)
    for axis in (0, 1):
        dW = be.empty((vocab, embed), dtype=np_dtype(name))
        be.compound_update_lut(ti, place(be, err, axis, "plain", name), dW, scale=scale, axis=axis)
        ref.within(dW.get(), want, ref.stored(want, name, bound), "table gradient")


# words of more than 24 bits take three passes of the sort; more than 4 million positions are more slices than a
# class's workgroup has threads.  Errors are ones, or the position's parity: sums that fp32 holds exactly
@pytest.mark.parametrize("vocab,positions,embed,same", [(2 ** 24 + 777, 3000, 3, 0.0), (2 ** 24 + 777, 40000, 2, 0.4),
                                                        (900, 4300000, 2, 0.1), (70000, 4200001, 1, 0.3)])
def test_table_gradient_of_large_tables_and_many_positions(hip, vocab, positions, embed, same):
    be = hip
    rs = np.random.RandomState(7)
    ids = rs.randint(0, vocab, positions).astype(np.int32)
    ids[rs.rand(positions) < same] = vocab - 5                        # a class that does not fit the LDS
    ids[::1000] = -1
    ti = be.array(ids.reshape(1, -1), dtype=np.int32)
    err = np.ones((embed, positions), np.float32)
    err[-1] = np.arange(positions) % 2
    ok = ids >= 0
    want = [np.bincount(ids[ok], weights=err[e][ok], minlength=vocab) for e in range(embed)]
    for axis in (0, 1):
        dW = be.empty((vocab, embed))
        dW[:] = 77.0
        be.compound_update_lut(ti, be.array(err if axis == 0 else np.ascontiguousarray(err.T)), dW, axis=axis)
        got = dW.get()
        for e in range(embed):
            assert np.array_equal(got[:, e], want[e].astype(np.float32))
        out = be.empty((embed, positions) if axis == 0 else (positions, embed))
        be.compound_fprop_lut(ti, dW, out, axis=axis)
        out = out.get() if axis == 0 else out.get().T
        assert np.array_equal(out, np.where(ok, got[np.where(ok, ids, 0)].T, 0.0))
