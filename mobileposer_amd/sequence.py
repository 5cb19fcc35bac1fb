"""Sequence operators of the facade: the gated delta rule over ragged batches (``delta_rule``) and per tick of S streams
(``delta_rule_online``), and a linear layer with a low-rank adapter per sequence (``linear_adapted``) -- the parts of a personalised
recurrent block, over mp_delta_rule / mp_delta_rule_online / mp_linear_adapted (include/mobileposer_hip.h).

They take torch tensors on the model's device, fp32 or bf16, run on the current stream, and return fresh tensors without waiting.
Inference only, as the rest of the package: a tensor that requires a gradient is refused while gradients are recorded, and one that
carries a tangent (forward-mode derivatives) always.
No counterpart in the reference."""
import ctypes as C

import torch
from torch.autograd import forward_ad

from . import _lib

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}
_INT_MAX = 2 ** 31 - 1
_stream_of = torch._C._cuda_getCurrentRawStream       # the current stream's handle (torch.cuda.current_stream builds an object around it: 2 us)


def _no_grad(*tensors):
    for t in tensors:
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("the sequence operators have no backward pass: call them under torch.no_grad() or detach their inputs")
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("the sequence operators have no forward-mode derivative: a tensor carries a tangent")


def _rows(t):
    """The tensor itself when its last dimension is contiguous, else a contiguous copy."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


class SequenceOps:
    """Methods of ``MobilePoserNet``, on its device.  They need none of its weights: a model that has not loaded any serves them
    through its body model's handle.  A tick's call is host time first: the checks read each property once."""

    _device_index = None         # set with the model's handle

    def _find_device(self):
        self._device_index = self.device.index if self.device.index is not None else torch.cuda.current_device()

    def _failed(self, rc, h):
        if h is self._h:
            self._check(rc)
        _lib.check(rc, h)

    def _dtype(self, what, first, *more):
        """The common type of the tensors, as the library numbers it; all of them on this model's device."""
        dtype, index = first.dtype, self._device_index
        if dtype not in _DTYPES:
            raise RuntimeError("%s takes float32 or bfloat16 tensors, got %s" % (what, dtype))
        if first.get_device() != index:
            raise RuntimeError("%s: a tensor on %s, the model is on %s" % (what, first.device, self.device))
        for t in more:
            if t.dtype is not dtype:
                raise RuntimeError("%s: tensors of one type expected, got %s and %s" % (what, dtype, t.dtype))
            if t.get_device() != index:
                raise RuntimeError("%s: a tensor on %s, the model is on %s" % (what, t.device, self.device))
        return _DTYPES[dtype]

    def _indices(self, what, value, n, lo, hi):
        """[n] int32 on the device.  A host sequence is checked against lo..hi; a device tensor is taken as it is (the kernels
        hold its values to the range: nothing waits for the device here)."""
        if torch.is_tensor(value) and value.is_cuda:
            if value.shape != (n,) or value.dtype not in (torch.int32, torch.int64):
                raise RuntimeError("%s: expected [%d] int32, got %s %s" % (what, n, tuple(value.shape), value.dtype))
            if value.get_device() != self._device_index:
                raise RuntimeError("%s: a tensor on %s, the model is on %s" % (what, value.device, self.device))
            if value.dtype is torch.int64:
                value = value.clamp(-1, _INT_MAX).to(torch.int32)
            return value.contiguous()
        ints = [int(i) for i in value]
        if len(ints) != n:
            raise RuntimeError("%s: %d values for %d sequences" % (what, len(ints), n))
        if any(i < lo or i > hi for i in ints):
            raise RuntimeError("%s: values outside of %d..%d" % (what, lo, hi))
        return torch.tensor(ints, dtype=torch.int32, device="cuda:%d" % self._device_index)

    def _heads(self, what, q, k, v, g, beta, lead):
        qs, vs = q.shape, v.shape
        if len(qs) != lead + 2 or len(vs) != lead + 2 or k.shape != qs or vs[:lead] != qs[:lead]:
            raise RuntimeError("%s: q, k [.., Hk, dk] and v [.., Hv, dv] expected, got %s, %s, %s" % (what, tuple(qs), tuple(k.shape), tuple(vs)))
        Hk, dk, Hv, dv = qs[lead], qs[lead + 1], vs[lead], vs[lead + 1]
        if Hk < 1 or Hv < 1 or Hv % Hk or not 1 <= dk <= 256 or dv < 1:
            raise RuntimeError("%s: %d value heads over %d key heads, head sizes %d / %d (Hv a multiple of Hk, dk at most 256)" % (what, Hv, Hk, dk, dv))
        gate = vs[:lead + 1]
        if g.shape != gate or beta.shape != gate:
            raise RuntimeError("%s: g and beta %s expected, got %s and %s" % (what, tuple(gate), tuple(g.shape), tuple(beta.shape)))
        if g.dtype is not torch.float32 or beta.dtype is not torch.float32:
            raise RuntimeError("%s: g and beta are float32, got %s and %s" % (what, g.dtype, beta.dtype))
        return Hk, dk, Hv, dv

    def delta_rule(self, q, k, v, g, beta, input_lengths=None, state=None, scale=None):
        """The gated delta rule over B ragged sequences: per value head a state S [dk, dv] and per frame
        ``S = exp(g) S; u = beta (v - S^T k); S = S + k u^T; o = scale S^T q``.

        q, k [B, T, Hk, dk], v [B, T, Hv, dv] (fp32 or bf16; views of one projection's rows are fine, frames less than 2^24 elements
        apart; what lies behind a sequence's end is not read), g (<= 0), beta [B, T, Hv]
        fp32, ``input_lengths`` [B] (0..T; a list, or an int32 tensor on the device, whose values are clamped), ``state``
        [B, Hv, dk, dv] fp32 or None (zeros), ``scale`` (default dk ** -0.5).
        -> (o [B, T, Hv, dv], zeros behind a sequence's end; the state after each sequence's last frame, fp32)."""
        if self._device_index is None:
            self._find_device()
        _no_grad(q, k, v, g, beta, state)
        dtype = self._dtype("delta_rule", q, k, v)
        Hk, dk, Hv, dv = self._heads("delta_rule", q, k, v, g, beta, 2)
        self._dtype("delta_rule", g, beta)
        B, T = q.shape[0], q.shape[1]
        if state is not None:
            if state.shape != (B, Hv, dk, dv) or state.dtype != torch.float32:
                raise RuntimeError("delta_rule: state [%d, %d, %d, %d] float32 expected, got %s %s" % (B, Hv, dk, dv, tuple(state.shape), state.dtype))
            self._dtype("delta_rule", state)
            state = state.contiguous()
        lens = None if input_lengths is None else self._indices("delta_rule: input_lengths", input_lengths, B, 0, T)
        q, k, v = _rows(q), _rows(k), _rows(v)
        dev = q.device
        o = torch.empty(B, T, Hv, dv, device=dev, dtype=q.dtype)
        out = torch.empty(B, Hv, dk, dv, device=dev, dtype=torch.float32)
        need = self._lib.mp_delta_rule_workspace(B, T, Hv, dk, dv)
        ws = torch.empty(need, device=dev, dtype=torch.uint8)
        st = (C.c_int64 * 15)(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *g.stride(), *beta.stride())
        h = self._h or self.bodymodel._handle()[1]
        rc = self._lib.mp_delta_rule(
            h, dtype, q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(), C.addressof(st),
            0 if lens is None else lens.data_ptr(), B, T, Hk, Hv, dk, dv, dk ** -0.5 if scale is None else float(scale), o.data_ptr(),
            0 if state is None else state.data_ptr(), out.data_ptr(), ws.data_ptr(), need, _stream_of(self._device_index))
        if rc:
            self._failed(rc, h)
        return o, out

    def delta_rule_online(self, q, k, v, g, beta, state, slots=None, scale=None):
        """One frame of S streams on states that stay in place: q, k [S, Hk, dk], v [S, Hv, dv], g, beta [S, Hv], ``state``
        [n, Hv, dk, dv] fp32 contiguous, updated; ``slots`` [S]: the state of each stream (None: stream s has state s).  A negative
        slot is a stream without a frame (zeros, no state changes); a slot that is not there, or that an earlier stream of the
        call has, gives a row of NaN and changes no state.  -> o [S, Hv, dv]."""
        if self._device_index is None:
            self._find_device()
        _no_grad(q, k, v, g, beta, state)
        dtype = self._dtype("delta_rule_online", q, k, v)
        Hk, dk, Hv, dv = self._heads("delta_rule_online", q, k, v, g, beta, 1)
        self._dtype("delta_rule_online", g, beta, state)
        S = q.shape[0]
        if state.dim() != 4 or state.shape[1:] != (Hv, dk, dv) or not state.is_contiguous():
            raise RuntimeError("delta_rule_online: contiguous state [n, %d, %d, %d] expected, got %s" % (Hv, dk, dv, tuple(state.shape)))
        n = state.shape[0]
        if slots is None:
            if S > n:
                raise RuntimeError("delta_rule_online: %d streams on %d states" % (S, n))
        else:
            slots = self._indices("delta_rule_online: slots", slots, S, -_INT_MAX, n - 1)
        q, k, v = _rows(q), _rows(k), _rows(v)
        o = torch.empty(S, Hv, dv, device=q.device, dtype=q.dtype)
        st = (C.c_int64 * 10)(*q.stride()[:2], *k.stride()[:2], *v.stride()[:2], *g.stride(), *beta.stride())
        h = self._h or self.bodymodel._handle()[1]
        rc = self._lib.mp_delta_rule_online(
            h, dtype, q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(), C.addressof(st),
            0 if slots is None else slots.data_ptr(), S, n, Hk, Hv, dk, dv, dk ** -0.5 if scale is None else float(scale), o.data_ptr(),
            state.data_ptr(), _stream_of(self._device_index))
        if rc:
            self._failed(rc, h)
        return o

    def _block_adapters(self, adapters, ids, B, shapes):
        """``rnn_forward``'s adapters, checked: per layer its four arguments of mp_rnn_forward_adapted; the number of adapters, the
        larger rank, the ids on the device, and the tensors those addresses belong to."""
        if set(adapters) - set(shapes) or not adapters:
            raise RuntimeError("rnn_forward: adapters of linear1 and / or linear2 expected, got %s" % sorted(adapters))
        if ids is None:
            raise RuntimeError("rnn_forward: adapters without ids")
        args, n, rank, keep = {name: (0, 0, 0, 0) for name in shapes}, None, 0, []
        for name, (down, up, scale) in adapters.items():
            K, M = shapes[name]
            _no_grad(down, up, scale)
            if self._dtype("rnn_forward: adapters", down, up, *(() if scale is None else (scale,))) != _lib.F32:
                raise RuntimeError("rnn_forward: adapters are float32, got %s" % down.dtype)
            if down.dim() != 3 or down.shape[2] != K or not 1 <= down.shape[1] <= 128 or up.shape != (down.shape[0], M, down.shape[1]) or \
                    down.shape[0] < 1 or down.shape[0] != (n or down.shape[0]) or (scale is not None and scale.shape != down.shape[:1]):
                raise RuntimeError("rnn_forward: %s: down [n, r, %d], up [n, %d, r] and scale [n] with r at most 128 and one n expected, got %s and %s" %
                                   (name, K, M, tuple(down.shape), tuple(up.shape)))
            n, rank = down.shape[0], max(rank, down.shape[1])
            down, up, scale = down.contiguous(), up.contiguous(), None if scale is None else scale.contiguous()
            keep += [down, up, scale]
            args[name] = (down.data_ptr(), up.data_ptr(), 0 if scale is None else scale.data_ptr(), down.shape[1])
        return args, n, rank, self._indices("rnn_forward: ids", ids, B, -_INT_MAX, n - 1), keep

    def linear_adapted(self, x, weight, bias, down, up, scale, ids, relu=False):
        """``act(x W^T + b + scale[a] (x down[a]^T) up[a]^T)`` with a = ids[sequence]: a linear layer (nn.Linear's weight [M, K] and
        bias [M] or None) with a low-rank adapter per sequence beside it.  x [B, T, K] or, one frame each, [B, K]; down [n, r, K],
        up [n, M, r], r at most 128; ``scale`` [n] fp32 or None (1); ``ids`` [B]: negative = the shared layer alone (a list, or an
        int32 tensor on the device: a value >= n gives rows of NaN); ``relu``: ReLU behind it.  -> [B, T, M] or [B, M]."""
        if self._device_index is None:
            self._find_device()
        _no_grad(x, weight, bias, down, up, scale)
        dtype = self._dtype("linear_adapted", x, weight, down, up, *(() if bias is None else (bias,)))
        if x.dim() not in (2, 3) or weight.dim() != 2 or weight.shape[1] != x.shape[-1]:
            raise RuntimeError("linear_adapted: x [B, T, K] or [B, K] and weight [M, K] expected, got %s and %s" % (tuple(x.shape), tuple(weight.shape)))
        M, K = weight.shape
        if down.dim() != 3 or down.shape[2] != K or up.shape != (down.shape[0], M, down.shape[1]) or down.shape[0] < 1 or not 1 <= down.shape[1] <= 128:
            raise RuntimeError("linear_adapted: down [n, r, %d] and up [n, %d, r] with r at most 128 expected, got %s and %s" % (K, M, tuple(down.shape), tuple(up.shape)))
        n, r = down.shape[0], down.shape[1]
        if bias is not None and bias.shape != (M,):
            raise RuntimeError("linear_adapted: bias [%d] expected, got %s" % (M, tuple(bias.shape)))
        if scale is not None:
            if scale.shape != (n,) or scale.dtype != torch.float32:
                raise RuntimeError("linear_adapted: scale [%d] float32 expected, got %s %s" % (n, tuple(scale.shape), scale.dtype))
            self._dtype("linear_adapted", scale)
            scale = scale.contiguous()
        B, T = x.shape[0], x.shape[1] if x.dim() == 3 else 1
        ids = self._indices("linear_adapted: ids", ids, B, -_INT_MAX, n - 1)
        x, weight, down, up = _rows(x), weight.contiguous(), down.contiguous(), up.contiguous()
        bias = None if bias is None else bias.contiguous()
        y = torch.empty(*x.shape[:-1], M, device=x.device, dtype=x.dtype)
        need = self._lib.mp_linear_adapted_workspace(B, T, r)
        ws = torch.empty(need, device=x.device, dtype=torch.uint8)
        st = (C.c_int64 * 2)(x.stride(0), x.stride(1) if x.dim() == 3 else 0)
        h = self._h or self.bodymodel._handle()[1]
        rc = self._lib.mp_linear_adapted(
            h, dtype, x.data_ptr(), C.addressof(st), weight.data_ptr(), 0 if bias is None else bias.data_ptr(), down.data_ptr(),
            up.data_ptr(), 0 if scale is None else scale.data_ptr(), ids.data_ptr(), B, T, K, M, n, r, int(bool(relu)), y.data_ptr(),
            ws.data_ptr(), need, _stream_of(self._device_index))
        if rc:
            self._failed(rc, h)
        return y
