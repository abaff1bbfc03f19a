"""
Language-model operators of the ``hip`` backend: layer normalisation, embedding
lookup with its table's gradient, and distillation from a teacher's top logits.

The methods of ``LanguageModelOps`` are the backend class's.  A matrix argument holds
one position (token, sample) per column for ``axis=0`` -- the layout the
reference's layers use, (features, batch size) -- and one per row for
``axis=1``; ``axis`` is the axis a position's values lie along.  Either way its
memory may run along the features or along the positions (``x.T`` is as good as
``x``); views the kernels cannot read in place (gather views, strides along both
axes) go through a temporary.  Work is enqueued on the backend's stream.

The reference has batch normalisation (neon/backends/nervanagpu.py:2463-2588),
a lookup table's gradient (:2591-2660) and cross-entropy
(neon/transforms/cost.py:112-173) in these places; the calling conventions
follow those.
"""
import numpy as np

from neon_amd.backends.hip import bf16
from neon_amd.backends.hip import runtime as hiprt

ROWS, COLUMNS = 1, 0        # how memory runs: along a position's values / along the positions (the C ABI's axis)

_F32 = np.dtype(np.float32)
_I32 = np.dtype(np.int32)
_STORAGE = {_F32: 0, np.dtype(np.float16): 1, bf16.bfloat16: 2}


def _storage(what, t):
    code = _STORAGE.get(t.dtype)
    if code is None:
        raise TypeError("%s is %s: float32, float16 or bfloat16 expected" % (what, t.dtype))
    return code


def _shaped(what, t, shape, dtype=None):
    if t.shape != shape:
        raise ValueError("%s has shape %s: %s expected" % (what, t.shape, shape))
    if dtype is not None and t.dtype != dtype:
        raise TypeError("%s is %s: %s expected" % (what, t.dtype, dtype))


def _along(axis, features, positions):
    return (features, positions) if axis == 0 else (positions, features)


def _leading(t, axis, layout):
    """elements between the lines of ``t`` if its memory runs as ``layout``
    says, else None"""
    if t.take_array:
        return None
    features, positions = t.shape[axis], t.shape[1 - axis]
    step_f, step_p = t.strides[axis], t.strides[1 - axis]
    if layout == COLUMNS:
        features, positions, step_f, step_p = positions, features, step_p, step_f
    # now: `features` values side by side, `positions` lines
    if features > 1 and step_f != 1:
        return None
    if positions <= 1:
        return features
    return step_p if step_p >= features else None


def _dense(t, axis):
    """a vector along ``axis`` without gaps"""
    return not t.take_array and (t.shape[axis] == 1 or t.strides[axis] == 1)


def _interleaved(a, b):
    """two views into one range of memory that certainly share no element:
    strided alike (columns of one matrix, windows of one), at offsets no pair of
    indices bridges"""
    if a.take_array or b.take_array or a.dtype.itemsize != b.dtype.itemsize:
        return False
    diff, rest = divmod(b.gpudata - a.gpudata, a.dtype.itemsize)
    if rest:
        return False
    dims = []
    for na, nb, sa, sb in zip(a.shape, b.shape, a.strides, b.strides):
        if na > 1 or nb > 1:
            if (na > 1 and nb > 1 and sa != sb) or min(sa, sb) <= 0:
                return False
            dims.append((sa if na > 1 else sb, na, nb))
    if len(dims) == 1:
        dims.append((1, 1, 1))
    if not dims:
        return diff != 0
    (s0, a0, b0), (s1, a1, b1) = sorted(dims, reverse=True)
    # an element in both: diff = i * s0 + j * s1 with -b0 < i < a0, -b1 < j < a1
    low, high = -((s1 * (a1 - 1) - diff) // s0), (diff + s1 * (b1 - 1)) // s0
    low, high = max(low, 1 - b0), min(high, a0 - 1)
    if high - low > 16:
        return False
    return not any((diff - i * s0) % s1 == 0 and -b1 < (diff - i * s0) // s1 < a1 for i in range(low, high + 1))


class LanguageModelOps(object):
    """see the module's docstring"""

    # -- calls seen before --------------------------------------------------------------
    # A call whose tensors have the shapes, strides and types of an earlier one needs none of that
    # looked at again: ``_lm_forms`` keeps, by these and by nothing else, the constant arguments of
    # the library call.  What depends on addresses (overlap) and on attributes a program may change
    # (rounding) is looked at every time.
    def _lm_form(self, name, axis, tensors, outputs):
        """(key, constant arguments or None) of a call whose first ``outputs``
        tensors are written"""
        try:
            key = (name, axis) + tuple([t._geom[1:] for t in tensors])
            tail = self._lm_forms.get(key)
        except (AttributeError, TypeError):
            return None, None
        if tail is None:
            return key, None
        for t in tensors[:outputs]:
            if t.rounding:
                return key, None
        # (every tensor of a kept form is read and written in place; where two might share memory the
        # long way decides)
        end = 0
        for low, high in sorted([(t.gpudata, t.gpudata + t.nbytes) if t.is_contiguous else self._lm_byte_span(t)
                                 for t in tensors]):
            if low < end:
                return key, None
            end = high
        if self._deferred or self._pending:
            self._flush()
        return key, tail

    def _lm_keep(self, key, temps, tail):
        if key is not None and not temps:
            if len(self._lm_forms) >= 4096:         # a program of ever new shapes
                self._lm_forms.clear()
            self._lm_forms[key] = tail

    # -- arguments ----------------------------------------------------------------------
    def _lm_tensors(self, axis, outputs, inputs, aliases=()):
        """Checks every operator makes: tensors of this backend with two
        dimensions, no output asking for stochastic rounding, no output sharing
        memory with another argument -- except the (output, input) pairs in
        ``aliases``, which may be the very same view."""
        if axis not in (0, 1):
            raise ValueError("axis is 0 or 1, not %r" % (axis,))
        base = self._lm_tensor_base
        for t in outputs + inputs:
            if not isinstance(t, base):
                raise TypeError("a tensor of the hip backend expected, not %s" % type(t).__name__)
            if len(t.shape) != 2:
                raise ValueError("tensors with two dimensions expected, not %s" % (t.shape,))
        spans = [(t.gpudata, t.gpudata + t.nbytes) if t.is_contiguous else self._lm_byte_span(t)
                 for t in outputs + inputs]
        for i, out in enumerate(outputs):
            if out.rounding:
                raise NotImplementedError("stochastic rounding of this operator's outputs")
            if out.take_array:
                raise NotImplementedError("a gather view as this operator's output")
            if 0 in out.strides and not out.is_contiguous and \
                    any(s == 0 and n > 1 for s, n in zip(out.strides, out.shape)):
                raise ValueError("an output whose elements share memory")
            lo, hi = spans[i]
            for k in range(i + 1, len(spans)):
                if lo < spans[k][1] and spans[k][0] < hi:
                    other = inputs[k - len(outputs)] if k >= len(outputs) else None
                    if other is not None and any(out is a and other is b for a, b in aliases) and \
                            out._geom == other._geom:
                        continue
                    if _interleaved(out, other if other is not None else outputs[k]):
                        continue
                    raise ValueError("an output of this operator overlaps another argument")

    def _lm_layout(self, axis, tensors):
        """the way memory runs in all of ``tensors``; where they disagree, in
        the first one that has a way (the others go through temporaries)"""
        first = tensors[0]
        features, positions = first.shape[axis], first.shape[1 - axis]
        order = (ROWS, COLUMNS) if features >= positions else (COLUMNS, ROWS)
        best, count = order[0], -1
        for layout in order:
            n = sum(_leading(t, axis, layout) is not None for t in tensors)
            if n > count:
                best, count = layout, n
        return best

    def _lm_temp(self, t, axis, layout, temps):
        """an uninitialised temporary of ``t``'s shape whose memory runs as
        ``layout`` says"""
        if (layout == ROWS) == (axis == 1):
            return self._temp(t.shape, t.dtype, temps)
        return self._temp(t.shape[::-1], t.dtype, temps).T

    def _lm_in(self, t, axis, layout, temps):
        """(tensor, leading dimension) the kernels can read"""
        ld = _leading(t, axis, layout)
        if ld is None:
            tmp = self._lm_temp(t, axis, layout, temps)
            self._run([self._stmt(tmp, t)])
            t, ld = tmp, _leading(tmp, axis, layout)
        return t, ld

    def _lm_out(self, t, axis, layout, temps, back, keep=False):
        """(tensor, leading dimension) the kernels can write; ``back`` collects
        (destination, temporary) pairs to copy afterwards"""
        ld = _leading(t, axis, layout)
        if ld is None:
            tmp = self._lm_temp(t, axis, layout, temps)
            if keep:
                self._run([self._stmt(tmp, t)])
            back.append((t, tmp))
            t, ld = tmp, _leading(tmp, axis, layout)
        return t, ld

    def _lm_vector_in(self, t, axis, temps):
        if _dense(t, axis):
            return t
        tmp = self._temp(t.shape, t.dtype, temps)
        self._run([self._stmt(tmp, t)])
        return tmp

    def _lm_vector_out(self, t, axis, temps, back):
        if _dense(t, axis):
            return t
        tmp = self._temp(t.shape, t.dtype, temps)
        back.append((t, tmp))
        return tmp

    def _lm_copy_back(self, back):
        for dst, tmp in back:
            self._run([self._stmt(dst, tmp)])

    def _lm_release(self, temps):
        for t in temps:
            self._temp_release(t)

    def _lm_workspace(self, need):
        """scratch of at least ``need`` bytes, the backend's own: its operators
        run one after another on its stream"""
        if not need:
            return 0, 0
        have = self._lm_ws
        if have is None or have[1] < need:
            if have is not None:
                self.synchronize()
                self._lm_ws = None
                self.rt.free(have[0])
            size = (need + (1 << 20) - 1) >> 20 << 20
            have = self._lm_ws = (self.rt.malloc(size), size)
        return have

    # -- layer normalisation -------------------------------------------------------------
    def compound_fprop_ln(self, x, xmean, xvar, gamma, beta, y, eps, axis=0):
        """Layer normalisation: ``y = gamma * (x - xmean) / sqrt(xvar + eps) +
        beta`` with the mean and the (biased) variance of every position over
        its features, which are also stored for the backward pass.

        With ``axis=0``: x, y (features, positions), gamma and beta (features,
        1), xmean and xvar (1, positions); with ``axis=1`` all of them
        transposed.  x and y are float32, float16 or bfloat16 alike, the rest is
        float32.  y may be x."""
        eps = float(eps)
        key, tail = self._lm_form("ln", axis, (y, xmean, xvar, x, gamma, beta), 3)
        if tail is not None:
            ws, ws_bytes = self._lm_workspace(tail[6])
            hiprt.check(self.rt.lib.nh_ln_fprop(y.gpudata, xmean.gpudata, xvar.gpudata, x.gpudata, gamma.gpudata,
                                                beta.gpudata, eps, *tail[:6], ws, ws_bytes, self.rt.stream))
            return
        self._lm_tensors(axis, (y, xmean, xvar), (x, gamma, beta), ((y, x),))
        code = _storage("x", x)
        features, positions = x.shape[axis], x.shape[1 - axis]
        _shaped("y", y, x.shape, x.dtype)
        per_feature, per_position = _along(axis, features, 1), _along(axis, 1, positions)
        _shaped("gamma", gamma, per_feature, _F32)
        _shaped("beta", beta, per_feature, _F32)
        _shaped("xmean", xmean, per_position, _F32)
        _shaped("xvar", xvar, per_position, _F32)
        if features == 0:
            raise ValueError("positions without features have no mean")
        self._flush()
        if positions == 0:
            return
        temps, back = [], []
        try:
            layout = self._lm_layout(axis, (x, y))
            xin, ld_x = self._lm_in(x, axis, layout, temps)
            out, ld_y = self._lm_out(y, axis, layout, temps, back)
            gamma, beta = self._lm_vector_in(gamma, axis, temps), self._lm_vector_in(beta, axis, temps)
            mean, var = (self._lm_vector_out(t, 1 - axis, temps, back) for t in (xmean, xvar))
            rt = self.rt
            need = rt.lib.nh_ln_workspace_bytes(0, code, layout, features, positions)
            ws, ws_bytes = self._lm_workspace(need)
            tail = (code, layout, features, positions, ld_x, ld_y)
            hiprt.check(rt.lib.nh_ln_fprop(out.gpudata, mean.gpudata, var.gpudata, xin.gpudata, gamma.gpudata,
                                           beta.gpudata, eps, *tail, ws, ws_bytes, rt.stream))
            self._lm_keep(key, temps, tail + (need,))
            self._lm_copy_back(back)
        finally:
            self._lm_release(temps)

    def compound_bprop_ln(self, delta_out, grad_gamma, grad_beta, delta_in, x, xmean, xvar, gamma, eps, axis=0):
        """Gradients of ``compound_fprop_ln``: ``delta_out`` with respect to x,
        ``grad_gamma`` and ``grad_beta`` (overwritten) from the error
        ``delta_in`` with respect to y and the saved statistics.  Shapes and
        types as there; sums over positions are taken in a fixed order.
        delta_out may be delta_in or x."""
        eps = float(eps)
        key, tail = self._lm_form("ln grad", axis, (delta_out, grad_gamma, grad_beta, delta_in, x, xmean, xvar, gamma), 3)
        if tail is not None:
            ws, ws_bytes = self._lm_workspace(tail[7])
            hiprt.check(self.rt.lib.nh_ln_bprop(delta_out.gpudata, grad_gamma.gpudata, grad_beta.gpudata, delta_in.gpudata,
                                                x.gpudata, xmean.gpudata, xvar.gpudata, gamma.gpudata, eps, *tail[:7],
                                                ws, ws_bytes, self.rt.stream))
            return
        self._lm_tensors(axis, (delta_out, grad_gamma, grad_beta), (delta_in, x, xmean, xvar, gamma),
                         ((delta_out, delta_in), (delta_out, x)))
        code = _storage("x", x)
        features, positions = x.shape[axis], x.shape[1 - axis]
        _shaped("delta_in", delta_in, x.shape, x.dtype)
        _shaped("delta_out", delta_out, x.shape, x.dtype)
        per_feature, per_position = _along(axis, features, 1), _along(axis, 1, positions)
        for what, t, shape in (("gamma", gamma, per_feature), ("grad_gamma", grad_gamma, per_feature),
                               ("grad_beta", grad_beta, per_feature), ("xmean", xmean, per_position),
                               ("xvar", xvar, per_position)):
            _shaped(what, t, shape, _F32)
        if features == 0:
            raise ValueError("positions without features have no mean")
        self._flush()
        temps, back = [], []
        try:
            layout = self._lm_layout(axis, (x, delta_in, delta_out))
            xin, ld_x = self._lm_in(x, axis, layout, temps)
            dy, ld_dy = self._lm_in(delta_in, axis, layout, temps)
            dx, ld_dx = self._lm_out(delta_out, axis, layout, temps, back)
            gamma = self._lm_vector_in(gamma, axis, temps)
            mean, var = (self._lm_vector_in(t, 1 - axis, temps) for t in (xmean, xvar))
            dgamma, dbeta = (self._lm_vector_out(t, axis, temps, back) for t in (grad_gamma, grad_beta))
            rt = self.rt
            need = rt.lib.nh_ln_workspace_bytes(1, code, layout, features, positions)
            ws, ws_bytes = self._lm_workspace(need)
            tail = (code, layout, features, positions, ld_x, ld_dy, ld_dx)
            hiprt.check(rt.lib.nh_ln_bprop(dx.gpudata, dgamma.gpudata, dbeta.gpudata, dy.gpudata, xin.gpudata,
                                           mean.gpudata, var.gpudata, gamma.gpudata, eps, *tail, ws, ws_bytes, rt.stream))
            self._lm_keep(key, temps, tail + (need,))
            self._lm_copy_back(back)
        finally:
            self._lm_release(temps)

    # -- embedding ---------------------------------------------------------------------------
    def _lm_ids(self, inputs, temps):
        """word ids as one run of int32"""
        if inputs.dtype != _I32:
            raise TypeError("word ids are %s: int32 expected" % inputs.dtype)
        if inputs.is_contiguous:
            return inputs
        if inputs.take_array or min(inputs.strides) < 0:
            raise NotImplementedError("word ids in a gather view or a reversed one")
        tmp = self._temp(inputs.shape, inputs.dtype, temps)
        self.copy_transpose(inputs, tmp, axes=(0, 1))
        return tmp

    def compound_fprop_lut(self, inputs, W, outputs, pad_idx=None, scale=1.0, axis=0):
        """Embedding lookup: the values of position j are ``scale * W[w]`` for
        its word ``w = inputs[j]`` -- zeros where w is ``pad_idx`` or no row of
        W.  inputs holds int32 ids, in row-major order whatever its shape; W is
        (vocabulary, embedding size); outputs (embedding size, positions) for
        ``axis=0``, (positions, embedding size) for ``axis=1``."""
        pad, scale = -1 if pad_idx is None else int(pad_idx), float(scale)
        key, tail = self._lm_form("lut", axis, (outputs, inputs, W), 1)
        if tail is not None:
            hiprt.check(self.rt.lib.nh_embed_fprop(outputs.gpudata, W.gpudata, inputs.gpudata, scale, *tail, pad,
                                                   self.rt.stream))
            return
        self._lm_tensors(axis, (outputs,), (inputs, W))
        code = _storage("W", W)
        vocab, embed = W.shape
        count = inputs.size
        if vocab == 0 or embed == 0:
            raise ValueError("an empty table")
        _shaped("outputs", outputs, _along(axis, embed, count), W.dtype)
        temps, back = [], []
        self._flush()
        try:
            ids = self._lm_ids(inputs, temps)
            if count == 0:
                return
            table, ld_w = self._lm_in(W, 1, ROWS, temps)
            layout = self._lm_layout(axis, (outputs,))
            out, ld_out = self._lm_out(outputs, axis, layout, temps, back)
            rt = self.rt
            tail = (code, layout, count, embed, vocab, ld_w, ld_out)
            hiprt.check(rt.lib.nh_embed_fprop(out.gpudata, table.gpudata, ids.gpudata, scale, *tail, pad, rt.stream))
            self._lm_keep(key, temps, tail)
            self._lm_copy_back(back)
        finally:
            self._lm_release(temps)

    def compound_update_lut(self, inputs, error, dW, pad_idx=None, scale=1.0, beta=0.0, axis=0):
        """Gradient of ``compound_fprop_lut`` with respect to its table:
        ``dW = beta * dW + scale * G`` where ``G[w]`` is the sum of the errors of
        the positions that hold word w, zero for ``pad_idx`` and for words that
        do not occur.  ``beta=0`` defines every row of dW, ``beta=1`` adds to it.
        error has the shape outputs had; sums are taken in a fixed order, in
        float32."""
        pad, scale, beta = -1 if pad_idx is None else int(pad_idx), float(scale), float(beta)
        key, tail = self._lm_form("lut grad", axis, (dW, inputs, error), 1)
        if tail is not None:
            ws, ws_bytes = self._lm_workspace(tail[7])
            hiprt.check(self.rt.lib.nh_embed_update(dW.gpudata, error.gpudata, inputs.gpudata, scale, beta, *tail[:7], pad,
                                                    ws, ws_bytes, self.rt.stream))
            return
        self._lm_tensors(axis, (dW,), (inputs, error))
        code = _storage("dW", dW)
        vocab, embed = dW.shape
        count = inputs.size
        if vocab == 0 or embed == 0:
            raise ValueError("an empty table")
        _shaped("error", error, _along(axis, embed, count), dW.dtype)
        temps, back = [], []
        self._flush()
        try:
            ids = self._lm_ids(inputs, temps)
            table, ld_dw = self._lm_out(dW, 1, ROWS, temps, back, keep=beta != 0)
            layout = self._lm_layout(axis, (error,))
            err, ld_err = self._lm_in(error, axis, layout, temps)
            rt = self.rt
            need = rt.lib.nh_embed_update_workspace_bytes(code, layout, count, embed, vocab)
            ws, ws_bytes = self._lm_workspace(need)
            tail = (code, layout, count, embed, vocab, ld_dw, ld_err)
            hiprt.check(rt.lib.nh_embed_update(table.gpudata, err.gpudata, ids.gpudata, scale, beta, *tail, pad,
                                               ws, ws_bytes, rt.stream))
            self._lm_keep(key, temps, tail + (need,))
            self._lm_copy_back(back)
        finally:
            self._lm_release(temps)

    # -- distillation ------------------------------------------------------------------------
    def _lm_entries(self, axis, y, ids, t):
        positions = y.shape[1 - axis]
        entries = ids.shape[axis]
        _shaped("ids", ids, _along(axis, entries, positions), _I32)
        _shaped("t", t, ids.shape)
        if ids.take_array:
            raise NotImplementedError("word ids in a gather view")
        if y.shape[axis] == 0:
            raise ValueError("an empty vocabulary")
        return entries, positions

    def _lm_temperature(self, temperature):
        temperature = float(temperature)
        if not 2.0 ** -60 <= temperature <= 2.0 ** 60:
            raise ValueError("the temperature lies between 2**-60 and 2**60, not %r" % temperature)
        return temperature

    def compound_fprop_distill(self, y, ids, t, loss, stats, temperature=1.0, axis=0):
        """Distillation from a teacher's top logits.  Per position, with the
        student's logits y over the vocabulary, the words ``ids`` the teacher
        rates highest and its logits t for them:

            p = softmax(t / temperature)  over the entries with 0 <= id < vocabulary
            q = softmax(y / temperature)  over the vocabulary
            loss = temperature**2 * sum_k p_k * (log p_k - log q[ids_k])

        Entries with another id (-1, say) fill up shorter lists; a position
        without entries has loss 0.  A word may be named twice.  ``stats``
        receives what the backward pass starts from: the largest y and the
        logarithm of sum(exp((y - largest) / temperature)), and the same two of
        the entries' t (largest -inf without entries).

        With ``axis=0``: y (vocabulary, positions), ids (int32) and t (entries,
        positions), loss (1, positions), stats (4, positions); with ``axis=1``
        all of them transposed.  y and t are float32, float16 or bfloat16, loss
        and stats float32; at most 1024 entries, a temperature between 2**-60
        and 2**60."""
        key, tail = self._lm_form("distill", axis, (loss, stats, y, ids, t), 2)
        if tail is not None:
            ws, ws_bytes = self._lm_workspace(tail[8])
            hiprt.check(self.rt.lib.nh_distill_fprop(loss.gpudata, stats.gpudata, y.gpudata, ids.gpudata, t.gpudata,
                                                     self._lm_temperature(temperature), *tail[:8], ws, ws_bytes,
                                                     self.rt.stream))
            return
        self._lm_tensors(axis, (loss, stats), (y, ids, t))
        code, t_code = _storage("y", y), _storage("t", t)
        temperature = self._lm_temperature(temperature)
        entries, positions = self._lm_entries(axis, y, ids, t)
        _shaped("loss", loss, _along(axis, 1, positions), _F32)
        _shaped("stats", stats, _along(axis, 4, positions), _F32)
        self._flush()
        if positions == 0:
            return
        temps = []
        try:
            layout = self._lm_layout(axis, (y,))
            z, ld_z = self._lm_in(y, axis, layout, temps)
            if t.take_array:
                t, _ = self._lm_in(t, axis, layout, temps)
            rt, vocab = self.rt, y.shape[axis]
            need = rt.lib.nh_distill_workspace_bytes(code, layout, vocab, positions)
            ws, ws_bytes = self._lm_workspace(need)
            strides = hiprt.int64s(ids.strides[axis], ids.strides[1 - axis], t.strides[axis], t.strides[1 - axis],
                                   loss.strides[1 - axis], stats.strides[axis], stats.strides[1 - axis])
            tail = (code, t_code, layout, vocab, positions, entries, ld_z, strides)
            hiprt.check(rt.lib.nh_distill_fprop(loss.gpudata, stats.gpudata, z.gpudata, ids.gpudata, t.gpudata, temperature,
                                                *tail, ws, ws_bytes, rt.stream))
            self._lm_keep(key, temps, tail + (need,))
        finally:
            self._lm_release(temps)

    def compound_bprop_distill(self, delta, y, ids, t, stats, weight=1.0, temperature=1.0, axis=0):
        """Gradient of ``compound_fprop_distill``'s loss with respect to y, each
        position's times its weight (a number, or a float32 tensor shaped like
        the loss):

            delta_v = weight * temperature * (q_v - sum of p_k over the entries with ids_k == v)

        and 0 at positions without entries.  delta is shaped and typed like y
        and must not share its memory; stats is what the forward pass left."""
        tensor_weight = isinstance(weight, self._lm_tensor_base)
        key, tail = self._lm_form("distill grad" if tensor_weight else "distill grad, one weight", axis,
                                  (delta, y, ids, t, stats) + ((weight,) if tensor_weight else ()), 1)
        if tail is not None:
            hiprt.check(self.rt.lib.nh_distill_bprop(delta.gpudata, y.gpudata, ids.gpudata, t.gpudata, stats.gpudata,
                                                     weight.gpudata if tensor_weight else None,
                                                     1.0 if tensor_weight else float(weight),
                                                     self._lm_temperature(temperature), *tail, self.rt.stream))
            return
        self._lm_tensors(axis, (delta,), (y, ids, t, stats) + ((weight,) if tensor_weight else ()))
        code, t_code = _storage("y", y), _storage("t", t)
        temperature = self._lm_temperature(temperature)
        entries, positions = self._lm_entries(axis, y, ids, t)
        _shaped("delta", delta, y.shape, y.dtype)
        _shaped("stats", stats, _along(axis, 4, positions), _F32)
        if tensor_weight:
            _shaped("weight", weight, _along(axis, 1, positions), _F32)
        self._flush()
        if positions == 0:
            return
        temps, back = [], []
        try:
            layout = self._lm_layout(axis, (y, delta))
            z, ld_z = self._lm_in(y, axis, layout, temps)
            dz, ld_dz = self._lm_out(delta, axis, layout, temps, back)
            if t.take_array:
                t, _ = self._lm_in(t, axis, layout, temps)
            if stats.take_array:
                stats, _ = self._lm_in(stats, axis, layout, temps)
            if tensor_weight and weight.take_array:
                weight = self._lm_vector_in(weight, 1 - axis, temps)
            rt, vocab = self.rt, y.shape[axis]
            strides = hiprt.int64s(ids.strides[axis], ids.strides[1 - axis], t.strides[axis], t.strides[1 - axis],
                                   stats.strides[axis], stats.strides[1 - axis], weight.strides[1 - axis] if tensor_weight else 0)
            tail = (code, t_code, layout, vocab, positions, entries, ld_z, ld_dz, strides)
            hiprt.check(rt.lib.nh_distill_bprop(dz.gpudata, z.gpudata, ids.gpudata, t.gpudata, stats.gpudata,
                                                weight.gpudata if tensor_weight else None,
                                                1.0 if tensor_weight else float(weight), temperature, *tail, rt.stream))
            self._lm_keep(key, temps, tail)
            self._lm_copy_back(back)
        finally:
            self._lm_release(temps)
