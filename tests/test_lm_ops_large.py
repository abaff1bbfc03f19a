"""The loops of the language-model kernels that only large calls enter, on
positions that repeat 16 different ones: those are checked against the float64
formulas, the others have to give the same bits.  Error bounds count the
additions that the kernels' geometry makes at these sizes (``lm_reference``'s
own count is for short sums)."""
import numpy as np
import pytest

import lm_reference as ref
from test_lm_ops import BF16, F16, F32, distill_inputs, np_dtype, vec

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
