"""float64 formulas of the language-model operators, positions along the first
axis, and how far fp32 arithmetic may be from them.

Bounds.  u = 2^-24 is half a unit of fp32.  A sum of terms t_i in which no term
passes through more than d additions is off by at most d u sum|t_i| (first
order); a product or quotient adds u per operation.  ``depth(n)`` is d for sums over
n values of which a thread adds at most 128 in a row before lanes and waves are joined (6 + 16
additions): so it is at the lengths of test_lm_ops.py, and no longer where a thread adds more (dgamma and dbeta:
a 512th, 256th or 64th of the positions; a vocabulary in one chunk: a 256th of it), which
test_lm_ops_large.py counts.  Storage types round once, by at
most ``half(dtype)`` relative, or half the smallest subnormal."""
import numpy as np

U = 2.0 ** -24
HALF = {"float32": 0.0, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float32": 2.0 ** -149, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -134}


def depth(n):
    return min(n, 128) + 22


def stored(value, name, error):
    """bound on the error of a value stored in a type of that name"""
    return error * (1 + HALF[name]) + np.abs(value) * HALF[name] + TINY[name]


# ---- layer normalisation ----------------------------------------------------------------
def ln(x, gamma, beta, eps):
    mean = x.mean(1, keepdims=True)
    var = ((x - mean) ** 2).mean(1, keepdims=True)
    return gamma * (x - mean) / np.sqrt(var + eps) + beta, mean, var


def ln_bounds(x, gamma, beta, eps):
    """(y, mean, var) errors before y is stored"""
    f = x.shape[1]
    y, mean, var = ln(x, gamma, beta, eps)
    d = depth(f)
    e_mean = (d + 2) * U * np.abs(x).mean(1, keepdims=True)
    dev = np.abs(x - mean)
    # each deviation is off by e_mean and a rounding; the shift of the mean enters squared
    # (deviations add up to nothing), the roundings of the deviations do not
    e_var = (d + 6) * U * (dev ** 2).mean(1, keepdims=True) + 2 * U * (dev * np.abs(mean)).mean(1, keepdims=True) \
        + e_mean ** 2 + 4 * e_mean * U * dev.mean(1, keepdims=True)
    rs = 1.0 / np.sqrt(var + eps)
    e_rs = rs * (0.5 * e_var / (var + eps) + 4 * U)
    e_y = np.abs(gamma) * (rs * (e_mean + 2 * U * dev + U * np.abs(mean)) + dev * e_rs) + 4 * U * (np.abs(y) + np.abs(beta))
    return e_y, e_mean, e_var


def ln_grad(dy, x, mean, var, gamma, eps):
    rs = 1.0 / np.sqrt(var + eps)
    h = (x - mean) * rs
    u = dy * gamma
    dx = rs * (u - u.mean(1, keepdims=True) - h * (u * h).mean(1, keepdims=True))
    return dx, (dy * h).sum(0, keepdims=True), dy.sum(0, keepdims=True)


def ln_grad_bounds(dy, x, mean, var, gamma, eps):
    n, f = x.shape
    rs = 1.0 / np.sqrt(var + eps)
    h, u = np.abs(x - mean) * rs, np.abs(dy * gamma)
    # h: the difference (1 unit of x - mean, exact operands), the reciprocal root (4) and the product (1)
    e_h = 6 * U * h
    a1, a2 = u.mean(1, keepdims=True), (u * h).mean(1, keepdims=True)
    e1, e2 = (depth(f) + 3) * U * a1, (depth(f) + 9) * U * a2
    s1, s2 = np.abs((dy * gamma).mean(1, keepdims=True)), np.abs((dy * gamma * (x - mean) * rs).mean(1, keepdims=True))
    e_dx = rs * (e1 + h * e2 + e_h * s2 + 12 * U * (u + s1 + h * s2))
    e_dg = ((depth(n) + 9) * U * np.abs(dy) * h).sum(0, keepdims=True)
    e_db = ((depth(n) + 2) * U * np.abs(dy)).sum(0, keepdims=True)
    return e_dx, e_dg, e_db


# ---- embedding -------------------------------------------------------------------------------
def live(ids, vocab, pad):
    return (ids >= 0) & (ids < vocab) & (ids != (-1 if pad is None else pad))


def lookup(W, ids, scale, pad):
    ok = live(ids, W.shape[0], pad)
    return np.where(ok[:, None], W[np.where(ok, ids, 0)] * scale, 0.0)


def table_sums(err, ids, vocab, pad):
    g = np.zeros((vocab, err.shape[1]))
    ok = live(ids, vocab, pad)
    np.add.at(g, ids[ok], err[ok])
    return g


def table_grad(dW, err, ids, scale, beta, pad):
    return (beta * dW if beta else 0.0) + scale * table_sums(err, ids, dW.shape[0], pad)


def table_grad_bound(dW, err, ids, scale, beta, pad):
    vocab = dW.shape[0]
    counts = np.bincount(ids[live(ids, vocab, pad)], minlength=vocab)[:, None]
    # 32 positions in a row, the partial sums of runs of 32 in eight shares, the shares (the kernel adds up to 24
    # partial sums one after another and more in sixteen shares, of runs of 8 to 32: test_lm_ops_large.py)
    d = np.minimum(counts, 32 + (counts // 32 + 2 + 7) // 8 + 8) + 3
    return d * U * np.abs(scale) * table_sums(np.abs(err), ids, vocab, pad) + (2 * U * np.abs(beta * dW) if beta else 0.0)


# ---- distillation ----------------------------------------------------------------------------
def _log_sum(z, temperature):
    """per row: the largest value, log sum exp((z - largest) / temperature), the
    exponents (z - largest) / temperature"""
    with np.errstate(all="ignore"):
        top = z.max(1, keepdims=True, initial=-np.inf)
        e = (z - np.where(top == -np.inf, 0.0, top)) / temperature
        return top, np.log(np.exp(e).sum(1, keepdims=True)), e


def _counts(ids, vocab):
    return (ids >= 0) & (ids < vocab)


def distill(z, ids, t, temperature):
    """(loss, stats)"""
    ok = _counts(ids, z.shape[1])
    top, log_sum, e = _log_sum(z, temperature)
    t_top, t_log_sum, te = _log_sum(np.where(ok, t, -np.inf), temperature)
    some = t_top != -np.inf
    with np.errstate(all="ignore"):
        log_p = np.where(ok & some, te - np.where(some, t_log_sum, 0.0), -np.inf)
        p = np.exp(log_p)
        # (where every z is -inf, q is no distribution)
        log_q = np.where(top == -np.inf, np.nan, np.take_along_axis(e, np.where(ok, ids, 0), 1) - log_sum)
        loss = np.where(p != 0, p * (log_p - log_q), 0.0).sum(1, keepdims=True)
    return temperature ** 2 * np.where(some, loss, 0.0), np.concatenate((top, log_sum, t_top, t_log_sum), 1)


def _distributions(z, ids, t, stats, temperature):
    """(counts, some, exponents of q, q, exponents of p, p) from saved statistics"""
    ok = _counts(ids, z.shape[1])
    top, log_sum, t_top, t_log_sum = (stats[:, i:i + 1] for i in range(4))
    some = t_top != -np.inf
    with np.errstate(all="ignore"):
        eq = (z - top) / temperature - log_sum
        ep = np.where(ok & some, (t - np.where(some, t_top, 0.0)) / temperature - np.where(some, t_log_sum, 0.0), -np.inf)
        return ok, some, eq, np.where(some, np.exp(eq), 0.0), ep, np.exp(ep)


def distill_grad(z, ids, t, stats, weight, temperature):
    ok, some, _, d, _, p = _distributions(z, ids, t, stats, temperature)
    row = np.broadcast_to(np.arange(len(z))[:, None], ids.shape)
    np.subtract.at(d, (row[ok], ids[ok]), p[ok])
    return np.where(some, weight * temperature * d, 0.0)


def distill_bounds(z, ids, t, temperature):
    """(loss, stats) errors"""
    ok, k = _counts(ids, z.shape[1]), ids.shape[1]
    top, log_sum, e = _log_sum(z, temperature)
    t_top, t_log_sum, te = _log_sum(np.where(ok, t, -np.inf), temperature)
    some = t_top != -np.inf
    none = np.zeros_like(top)
    with np.errstate(all="ignore"):
        # an exponent d = (z - m) / T is off by |d| times 5 u (difference, 1 / T, log2 e, their product, the
        # product); weighted by its own exponential that is at most 5 u / e per term, 5 u |d| e^d <= 2 u; exp2
        # adds 2 u; then the additions, and up to 12 joins of two partial sums with 5 u each.  Relative to
        # the sum; its logarithm adds 2 u of itself
        e_log = (4 + depth(z.shape[1]) + 128 + 60) * U + 2 * U * np.abs(log_sum)
        e_tlog = (4 + k / 64 + 8) * U + 2 * U * np.abs(np.where(some, t_log_sum, 0.0))
        log_p = np.where(ok & some, te - np.where(some, t_log_sum, 0.0), -np.inf)
        p = np.exp(log_p)
        ez = np.take_along_axis(e, np.where(ok, ids, 0), 1)
        # an entry's log p and log q: exponent (3 u), logarithm of the sum, difference (1 u); p is off by
        # the error of log p and 2 u; difference, product and the sum over the entries
        e_lq = e_log + U * (3 * np.abs(ez) + np.abs(ez - log_sum))
        e_lp = e_tlog + U * (3 * np.abs(te) + np.abs(log_p))
        near = np.abs(log_p - (ez - log_sum))
        terms = np.where(p > 0, p * (e_lq + e_lp + (e_lp + (2 + 3 + k / 64 + 8 + 3) * U) * near), 0.0)
        loss = np.where(some, terms.sum(1, keepdims=True), 0.0)
    # (a second-order term, and 2^-126 where an exponential is below the normal range)
    return temperature ** 2 * (1.01 * loss + k * 2.0 ** -120), np.concatenate((none, e_log, none, e_tlog), 1)


def distill_grad_bound(z, ids, t, stats, weight, temperature):
    """error before delta is stored"""
    ok, some, eq, q, ep, p = _distributions(z, ids, t, stats, temperature)
    with np.errstate(all="ignore"):
        log_sum, t_log_sum = stats[:, 1:2], stats[:, 3:4]
        # exponents: the difference and 1 / T (2 u of (z - m) / T), the fma and log2 e (3 u of the whole); the
        # teacher's: two more roundings.  exp2, expf: 3 u
        e = np.where(q == 0, 0.0, q * U * (2 * np.abs(eq + log_sum) + 3 * np.abs(eq) + 3))
        e_p = np.where(p == 0, 0.0, p * U * (3 * np.abs(ep + np.where(some, t_log_sum, 0.0)) + 2 * np.abs(ep) + 3 + ids.shape[1]))
    row = np.broadcast_to(np.arange(len(z))[:, None], ids.shape)
    np.add.at(e, (row[ok], ids[ok]), e_p[ok])
    d = np.abs(distill_grad(z, ids, t, stats, weight, temperature))
    # (2^-126: exponentials below the normal range may be flushed)
    return np.where(some, np.abs(weight) * temperature * (1.01 * e + 2.0 ** -125) + 4 * U * d, 0.0)


def within(got, want, bound, what=""):
    got, want, bound = (np.asarray(v, np.float64) for v in (got, want, np.broadcast_to(bound, np.shape(want))))
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what + ": NaN in other places"
    odd = ~fine & ~np.isnan(want)
    assert np.array_equal(got[odd], want[odd]), what + ": infinities differ"
    off = np.abs(got[fine] - want[fine]) - bound[fine]
    if off.size and not (off <= 0).all():
        i = np.argmax(np.where(np.isnan(off), np.inf, off))
        raise AssertionError("%s: %d of %d outside the bound; worst got %r want %r bound %r" % (
            what, int((~(off <= 0)).sum()), off.size, got[fine][i], want[fine][i], bound[fine][i]))
