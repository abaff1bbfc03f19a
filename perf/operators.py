"""
The language-model operators of the hip backend, as measured: layer
normalisation, embedding lookup and distillation from a teacher's top logits,
each forward and backward.

``columns`` is the backend's usual layout (features, positions): one position is
one column and memory runs along the positions.  ``rows`` is (positions,
features).  ``run`` computes an operator either in its plain form from
elementary torch operations, or (``own``) through the backend's entry points.
"""
import math

import torch

own = False

_DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}
_EPS = 1e-5


# ---- cases ---------------------------------------------------------------------------
def _ln(name, direction, dtype, layout, features, positions):
    return dict(name=name, op="ln", dir=direction, dtype=dtype, layout=layout, features=features, positions=positions)


def _lut(name, direction, dtype, layout, vocab, embed, positions, skew, pad):
    return dict(name=name, op="lut", dir=direction, dtype=dtype, layout=layout, vocab=vocab, embed=embed,
                positions=positions, skew=skew, pad=pad)


def _distill(name, direction, dtype, layout, vocab, positions, top, temperature):
    return dict(name=name, op="distill", dir=direction, dtype=dtype, layout=layout, vocab=vocab, positions=positions,
                top=top, temperature=temperature)


def listed():
    return [
        # a few sequences that generate one token each: launch latency
        _ln("ln decode", "fwd", "bf16", "rows", 4096, 5),
        # one minibatch of 128 behind a layer of 1000 units, the backend's own layout
        _ln("ln minibatch", "fwd", "fp32", "columns", 1000, 128),
        # the positions of a training step, one after another
        _ln("ln train fwd", "fwd", "bf16", "rows", 5000, 16384),
        _ln("ln train bwd", "bwd", "bf16", "rows", 2048, 16384),
        # 128 sequences of 196 steps in the backend's own layout
        _ln("ln columns bwd", "bwd", "fp16", "columns", 1024, 25088),
        # a short batch whose rows are no whole number of vectors
        _ln("ln ragged bwd", "bwd", "fp32", "rows", 1537, 777),
        # embedding layer of a training step into the backend's own layout
        _lut("lut train fwd", "fwd", "fp16", "columns", 32000, 1024, 16384, 1.0, True),
        # its gradient; text repeats a few tokens very often
        _lut("lut train bwd", "bwd", "bf16", "rows", 50000, 1024, 32768, 1.1, True),
        # word vectors of 300 over 128 sequences of 128
        _lut("lut columns bwd", "bwd", "fp32", "columns", 10000, 300, 16384, 0.9, False),
        # cost of one minibatch of 256 over 32000 words, the backend's own layout
        _distill("distill columns fwd", "fwd", "fp32", "columns", 32000, 256, 32, 2.0),
        # student logits of a training step; an odd vocabulary
        _distill("distill train fwd", "fwd", "bf16", "rows", 50001, 4096, 64, 1.0),
        _distill("distill train bwd", "bwd", "bf16", "rows", 32000, 8192, 64, 2.0),
    ]


_MOST_BYTES = 1.0e9     # of a drawn case; the largest listed one moves 1.05e9


def _log(rng, low, high):
    """a whole number, spread evenly over its logarithm"""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("ln", "lut", "distill"))
    common = dict(op=op, dir=rng.choice(("fwd", "bwd")), dtype=rng.choice(("fp32", "fp16", "bf16")),
                  layout=rng.choice(("rows", "columns")))
    size = _BYTES[common["dtype"]]
    if op == "ln":
        features = _log(rng, 32, 16384)
        most = int(_MOST_BYTES / (3 * size * features))
        return dict(common, features=features, positions=min(most, _log(rng, 1, 131072)))
    if op == "lut":
        embed = _log(rng, 16, 4096)
        vocab = min(_log(rng, 100, 130000), int(_MOST_BYTES / (3 * size * embed)))
        most = int(_MOST_BYTES / (3 * size * embed))
        return dict(common, vocab=vocab, embed=embed, positions=min(most, _log(rng, 1, 131072)),
                    skew=rng.choice((0.0, 0.9, 1.1)), pad=rng.choice((True, False)))
    vocab = _log(rng, 1000, 160000)
    most = int(_MOST_BYTES / (2 * size * vocab))
    return dict(common, vocab=vocab, positions=min(most, _log(rng, 1, 32768)), top=_log(rng, 1, 256),
                temperature=rng.choice((1.0, 2.0, 4.0)))


# ---- inputs --------------------------------------------------------------------------
def _oriented(t, layout):
    """(positions, features) values in the memory order of ``layout``"""
    return t.contiguous() if layout == "rows" else t.t().contiguous()


def _by_position(t, layout):
    return t if layout == "rows" else t.t()


def _token_weights(vocab, skew):
    return torch.arange(1, vocab + 1, dtype=torch.float64).pow(-skew)


def _make_ln(case, g, dev):
    n, f, dt, lay = case["positions"], case["features"], _DTYPES[case["dtype"]], case["layout"]
    x = torch.randn((n, f), generator=g, device=dev) * 2.0 + 0.5
    s = {"x": _oriented(x.to(dt), lay)}
    del x
    feature = (1, f) if lay == "rows" else (f, 1)
    position = (n, 1) if lay == "rows" else (1, n)
    s["gamma"] = torch.rand(feature, generator=g, device=dev) + 0.5
    s["beta"] = torch.randn(feature, generator=g, device=dev) * 0.1
    if case["dir"] == "fwd":
        s["y"] = torch.empty_like(s["x"])
        s["mean"] = torch.empty(position, device=dev)
        s["var"] = torch.empty(position, device=dev)
    else:
        dy = torch.randn((n, f), generator=g, device=dev) * 0.1
        s["dy"] = _oriented(dy.to(dt), lay)
        del dy
        axis = 1 if lay == "rows" else 0
        var, mean = torch.var_mean(s["x"].double(), dim=axis, keepdim=True, unbiased=False)
        s["mean"], s["var"] = mean.float(), var.float()
        s["dx"] = torch.empty_like(s["x"])
        s["dgamma"] = torch.empty(feature, device=dev)
        s["dbeta"] = torch.empty(feature, device=dev)
    return s


def _make_lut(case, g, dev):
    n, v, e, dt, lay = case["positions"], case["vocab"], case["embed"], _DTYPES[case["dtype"]], case["layout"]
    cdf = _token_weights(v, case["skew"]).cumsum(0).to(dev)
    u = torch.rand((n,), generator=g, device=dev, dtype=torch.float64) * cdf[-1]
    ids = torch.searchsorted(cdf, u).clamp_(max=v - 1).int()
    s = {"scale": math.sqrt(e), "pad": None}
    if case["pad"]:
        # the ends of short sequences
        s["pad"] = 0
        ids = torch.where(torch.rand((n,), generator=g, device=dev) < 0.1, torch.zeros_like(ids), ids)
    s["ids"] = ids.reshape(1, n)
    shape = (n, e) if lay == "rows" else (e, n)
    if case["dir"] == "fwd":
        s["W"] = (torch.randn((v, e), generator=g, device=dev) * 0.05).to(dt)
        s["out"] = torch.empty(shape, dtype=dt, device=dev)
    else:
        s["err"] = _oriented((torch.randn((n, e), generator=g, device=dev) * 0.01).to(dt), lay)
        s["dW"] = torch.empty((v, e), dtype=dt, device=dev)
    return s


def _log_sum(z, temperature):
    """largest value of each row, logarithm of the sum of exp((z - largest) / temperature)"""
    top = z.amax(1, keepdim=True)
    shifted = torch.where(z == -math.inf, z, z - top)
    return top, torch.log(torch.exp(shifted / temperature).sum(1, keepdim=True))


def _make_distill(case, g, dev):
    n, v, k, dt, lay = case["positions"], case["vocab"], case["top"], _DTYPES[case["dtype"]], case["layout"]
    z = (torch.randn((n, v), generator=g, device=dev) * 3.0).to(dt)
    # distinct words, the teacher's logits falling from the best one
    gaps = torch.randint(1, max(2, v // k), (n, k), generator=g, device=dev)
    first = torch.randint(0, v, (n, 1), generator=g, device=dev)
    ids = ((first + gaps.cumsum(1)) % v).int()
    t = (torch.rand((n, k), generator=g, device=dev) * 8.0).sort(dim=1, descending=True).values + 4.0
    # lists shorter than the longest, and positions behind the end of their sequence
    length = torch.randint((k + 1) // 2, k + 1, (n, 1), generator=g, device=dev)
    length = torch.where(torch.rand((n, 1), generator=g, device=dev) < 0.05, torch.zeros_like(length), length)
    ids = torch.where(torch.arange(k, device=dev)[None, :] < length, ids, torch.full_like(ids, -1))
    position = (n, 1) if lay == "rows" else (1, n)
    s = {"z": _oriented(z, lay), "ids": _oriented(ids, lay), "t": _oriented(t.to(dt), lay),
         "temperature": case["temperature"]}
    del z
    if case["dir"] == "fwd":
        s["loss"] = torch.empty(position, device=dev)
        s["stats"] = torch.empty((n, 4) if lay == "rows" else (4, n), device=dev)
    else:
        zp, tp, ip = (_by_position(s[a], lay) for a in ("z", "t", "ids"))
        tt = torch.where(ip >= 0, tp.double(), torch.full(tp.shape, -math.inf, device=dev).double())
        parts = [torch.cat(_log_sum(zp[i:i + 1024].double(), case["temperature"]) + _log_sum(tt[i:i + 1024], case["temperature"]), 1)
                 for i in range(0, n, 1024)]
        s["stats"] = _oriented(torch.cat(parts).float(), lay)
        # the weight of each position in the cost (the optimizer divides by the batch size)
        s["weight"] = torch.rand(position, generator=g, device=dev) + 0.5
        s["dz"] = torch.empty_like(s["z"])
    return s


_MAKE = {"ln": _make_ln, "lut": _make_lut, "distill": _make_distill}


def _backend():
    from neon_amd import NervanaObject
    from neon_amd.backends import gen_backend
    return gen_backend("hip", rng_seed=0) if NervanaObject.be is None else NervanaObject.be


def _handles(s):
    """the backend's tensors over the same memory: what a program built on the backend holds"""
    from neon_amd.backends import bfloat16
    be = _backend()
    names = {torch.float32: "float32", torch.float16: "float16", torch.int32: "int32", torch.bfloat16: bfloat16}
    return be, {k: be.tensor_cls(be, tuple(t.shape), dtype=names[t.dtype], gpudata=t.data_ptr(), strides=t.stride())
                for k, t in s.items() if isinstance(t, torch.Tensor)}


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    s = _MAKE[case["op"]](case, g, dev)
    s["case"] = case
    if own:
        s["be"], s["h"] = _handles(s)
    return s


# ---- the plain forms -----------------------------------------------------------------
def _plain_ln(s, case):
    axis, other = (1, 0) if case["layout"] == "rows" else (0, 1)
    x = s["x"].float()
    if case["dir"] == "fwd":
        mean = x.mean(axis, keepdim=True)
        xc = x - mean
        var = (xc * xc).mean(axis, keepdim=True)
        y = xc * (1.0 / torch.sqrt(var + _EPS)) * s["gamma"] + s["beta"]
        return y.to(s["x"].dtype), mean, var
    dy = s["dy"].float()
    r = 1.0 / torch.sqrt(s["var"] + _EPS)
    h = (x - s["mean"]) * r
    u = dy * s["gamma"]
    dx = r * (u - u.mean(axis, keepdim=True) - h * (u * h).mean(axis, keepdim=True))
    return dx.to(s["x"].dtype), (dy * h).sum(other, keepdim=True), dy.sum(other, keepdim=True)


def _plain_lut(s, case):
    ids = s["ids"].reshape(-1).long()
    live = torch.ones_like(ids, dtype=torch.bool) if s["pad"] is None else ids != s["pad"]
    if case["dir"] == "fwd":
        rows = s["W"][ids].float() * s["scale"] * live[:, None]
        out = rows.to(s["W"].dtype)
        return out if case["layout"] == "rows" else out.t().contiguous()
    err = _by_position(s["err"], case["layout"]).float() * (s["scale"] * live[:, None])
    return torch.zeros(s["dW"].shape, device=err.device).index_add_(0, ids, err).to(s["dW"].dtype)


def _plain_distill(s, case):
    axis = 1 if case["layout"] == "rows" else 0
    inv = 1.0 / s["temperature"]
    valid = s["ids"] >= 0
    ids = s["ids"].clamp(min=0).long()
    some = valid.any(axis, keepdim=True)
    z = s["z"].float()
    t = torch.where(valid, s["t"].float(), torch.full((), -math.inf, device=z.device))
    if case["dir"] == "fwd":
        top = z.max(axis, keepdim=True).values
        z = (z - top) * inv
        log_sum = torch.log(torch.exp(z).sum(axis, keepdim=True))
        ttop = t.max(axis, keepdim=True).values
        t = (t - torch.where(some, ttop, torch.zeros_like(ttop))) * inv
        tlog_sum = torch.log(torch.exp(t).sum(axis, keepdim=True))
        logp = torch.where(valid, t - tlog_sum, torch.zeros_like(t))
        terms = torch.where(valid, torch.exp(logp) * (logp - (z.gather(axis, ids) - log_sum)), torch.zeros_like(t))
        return terms.sum(axis, keepdim=True) * s["temperature"] ** 2, torch.cat((top, log_sum, ttop, tlog_sum), axis)
    top, log_sum, ttop, tlog_sum = s["stats"].split(1, axis)
    p = torch.where(valid, torch.exp((t - ttop) * inv - tlog_sum), torch.zeros_like(t))
    d = torch.where(some, torch.exp((z - top) * inv - log_sum), torch.zeros_like(z)).scatter_add_(axis, ids, -p)
    return (d * (s["weight"] * s["temperature"])).to(s["z"].dtype)


_PLAIN = {"ln": _plain_ln, "lut": _plain_lut, "distill": _plain_distill}


# ---- the backend's operators ---------------------------------------------------------
def _own_ln(s, case):
    be, h, axis = s["be"], s["h"], 1 if case["layout"] == "rows" else 0
    if case["dir"] == "fwd":
        be.compound_fprop_ln(h["x"], h["mean"], h["var"], h["gamma"], h["beta"], h["y"], _EPS, axis=axis)
        return s["y"], s["mean"], s["var"]
    be.compound_bprop_ln(h["dx"], h["dgamma"], h["dbeta"], h["dy"], h["x"], h["mean"], h["var"], h["gamma"], _EPS, axis=axis)
    return s["dx"], s["dgamma"], s["dbeta"]


def _own_lut(s, case):
    be, h, axis = s["be"], s["h"], 1 if case["layout"] == "rows" else 0
    if case["dir"] == "fwd":
        be.compound_fprop_lut(h["ids"], h["W"], h["out"], pad_idx=s["pad"], scale=s["scale"], axis=axis)
        return s["out"]
    be.compound_update_lut(h["ids"], h["err"], h["dW"], pad_idx=s["pad"], scale=s["scale"], axis=axis)
    return s["dW"]


def _own_distill(s, case):
    be, h, axis = s["be"], s["h"], 1 if case["layout"] == "rows" else 0
    if case["dir"] == "fwd":
        be.compound_fprop_distill(h["z"], h["ids"], h["t"], h["loss"], h["stats"], temperature=s["temperature"], axis=axis)
        return s["loss"], s["stats"]
    be.compound_bprop_distill(h["dz"], h["z"], h["ids"], h["t"], h["stats"], h["weight"], temperature=s["temperature"], axis=axis)
    return s["dz"]


_OWN = {"ln": _own_ln, "lut": _own_lut, "distill": _own_distill}


def run(state):
    case = state["case"]
    return (_OWN if own else _PLAIN)[case["op"]](state, case)


# ---- what a pass cannot do without ---------------------------------------------------
def work(case):
    n, size, fwd = case["positions"], _BYTES[case["dtype"]], case["dir"] == "fwd"
    if case["op"] == "ln":
        f = case["features"]
        return {"bytes": (2 if fwd else 3) * n * f * size + 8 * n + (8 if fwd else 12) * f,
                "flops": (8 if fwd else 16) * n * f}
    if case["op"] == "lut":
        v, e = case["vocab"], case["embed"]
        p = _token_weights(v, case["skew"])
        p = p / p.sum()
        words = float((1.0 - (1.0 - p).pow(n)).sum())       # different words among the positions, on average
        live = n * (0.9 if case["pad"] else 1.0)
        return {"bytes": 4 * n + ((words + n) if fwd else (live + v)) * e * size, "flops": n * e}
    v, k = case["vocab"], case["top"]
    return {"bytes": (1 if fwd else 2) * n * v * size + n * k * (4 + size) + 20 * n, "flops": 6 * n * v}


# ---- the definitions in 64 bits, position by position -------------------------------------
def _exact_ln(s, case):
    lay, dt = case["layout"], torch.float64
    x = _by_position(s["x"], lay)
    gamma, beta = s["gamma"].reshape(-1).to(dt), s["beta"].reshape(-1).to(dt)
    f = case["features"]
    parts, sums = [], [torch.zeros(f, dtype=dt, device=x.device) for _ in range(2)]
    step = max(1, (1 << 26) // f)
    for i in range(0, case["positions"], step):
        xi = x[i:i + step].to(dt)
        if case["dir"] == "fwd":
            mu = xi.sum(1) / f
            sq = (xi - mu[:, None]).square().sum(1) / f
            parts.append(((xi - mu[:, None]) / (sq + _EPS).sqrt()[:, None] * gamma + beta, mu, sq))
        else:
            mu = s["mean"].reshape(-1)[i:i + step].to(dt)
            sd = (s["var"].reshape(-1)[i:i + step].to(dt) + _EPS).sqrt()
            e = _by_position(s["dy"], lay)[i:i + step].to(dt)
            xhat = (xi - mu[:, None]) / sd[:, None]
            a = (e * gamma).sum(1) / f
            b = (e * xhat * gamma).sum(1) / f
            parts.append(((e * gamma - a[:, None] - xhat * b[:, None]) / sd[:, None],))
            sums[0] += (e * xhat).sum(0)
            sums[1] += e.sum(0)
    whole = [torch.cat(p) for p in zip(*parts)]
    if case["dir"] == "fwd":
        column = (lambda v: v[:, None]) if lay == "rows" else (lambda v: v[None, :])
        return _oriented(whole[0], lay), column(whole[1]), column(whole[2])
    feature = (lambda v: v[None, :]) if lay == "rows" else (lambda v: v[:, None])
    return _oriented(whole[0], lay), feature(sums[0]), feature(sums[1])


def _exact_lut(s, case):
    ids = s["ids"].reshape(-1).long()
    dead = torch.zeros_like(ids, dtype=torch.bool) if s["pad"] is None else ids == s["pad"]
    if case["dir"] == "fwd":
        out = torch.index_select(s["W"], 0, ids).double() * s["scale"]
        out[dead] = 0.0
        return _oriented(out, case["layout"])
    # words in order, running sums over the sorted positions, differences at the words' ends: per
    # block of columns, in 64 bits
    err = _by_position(s["err"], case["layout"])
    v, e = case["vocab"], case["embed"]
    keep = (~dead).nonzero()[:, 0]
    word, order = torch.sort(ids[keep], stable=True)
    ends = torch.searchsorted(word, torch.arange(v + 1, device=ids.device))
    dw = torch.empty((v, e), dtype=torch.float64, device=ids.device)
    for c in range(0, e, 512):
        run_sum = torch.zeros((len(keep) + 1, min(512, e - c)), dtype=torch.float64, device=ids.device)
        torch.cumsum(err[keep[order], c:c + 512].double(), 0, out=run_sum[1:])
        dw[:, c:c + 512] = run_sum[ends[1:]] - run_sum[ends[:-1]]
    return dw * s["scale"]


def _exact_distill(s, case):
    lay, tau, n, v = case["layout"], case["temperature"], case["positions"], case["vocab"]
    z, ids, t = (_by_position(s[a], lay) for a in ("z", "ids", "t"))
    parts = []
    for i in range(0, n, 1024):
        zi, ki, ti = z[i:i + 1024].double() / tau, ids[i:i + 1024].long(), t[i:i + 1024].double() / tau
        real = (ki >= 0) & (ki < v)
        ti = ti.masked_fill(~real, -math.inf)
        if case["dir"] == "fwd":
            log_q = torch.log_softmax(zi, 1)
            best, tbest = zi.max(1).values, ti.max(1).values
            rest, trest = torch.logsumexp(zi, 1) - best, torch.logsumexp(ti, 1) - tbest.clamp(min=-1e300)
            log_p = torch.log_softmax(ti, 1)
            cross = log_p - torch.gather(log_q, 1, ki.clamp(0, v - 1))
            terms = torch.where(real, log_p.exp() * cross, torch.zeros_like(cross))
            parts.append((tau * tau * terms.sum(1), torch.stack((best * tau, rest, tbest * tau, trest), 1)))
        else:
            best, rest, tbest, trest = _by_position(s["stats"], lay)[i:i + 1024].double().unbind(1)
            some = real.any(1)
            d = torch.zeros_like(zi)
            d[some] = (zi[some] - (best / tau + rest)[some, None]).exp()
            p = torch.where(real, (ti - (tbest / tau + trest)[:, None]).exp(), torch.zeros_like(ti))
            row, col = real.nonzero(as_tuple=True)
            d.index_put_((row, ki[row, col]), -p[row, col], accumulate=True)
            parts.append((d * (_by_position(s["weight"], lay)[i:i + 1024].double() * tau),))
    whole = [torch.cat(p) for p in zip(*parts)]
    if case["dir"] == "fwd":
        return (whole[0][:, None] if lay == "rows" else whole[0][None, :]), _oriented(whole[1], lay)
    return _oriented(whole[0], lay)


def exact(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = _MAKE[case["op"]](case, g, torch.device("cuda"))
    return {"ln": _exact_ln, "lut": _exact_lut, "distill": _exact_distill}[case["op"]](s, case)
