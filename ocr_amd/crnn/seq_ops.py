"""Operators on sequences of states, on torch tensors in device memory: the torch face of crnn_linear, crnn_rms_norm,
crnn_cross_attention and crnn_states_device (include/crnn_hip.h), as methods of ``CRNN``.

They run on torch's current stream of the handle's device and return without waiting; outputs are new tensors unless
``out`` is given.  Tensors have to be on the handle's device, with the last dimension contiguous; anything else about their
strides is taken as it is.  Inference only: a call that autograd would have to record is refused.
"""
import collections
import ctypes as C

import numpy as np

from . import _capi

RmsNorm = collections.namedtuple("RmsNorm", ["y", "scale", "sum"])
RmsNorm.__doc__ = "What rms_norm returns: y, its row scales (8-bit outputs only, else None), the sum (with a residual only, else None)."

ACTS = {"none": 0, None: 0, "relu": 1, "leaky": 2, "gelu": 3, "silu": 4}

_t = None       # torch, imported by the first call: the recogniser itself does without
_types = None   # torch dtype -> CRNN_* type


def _torch():
    global _t, _types
    if _t is None:
        import torch
        _t, _types = torch, {torch.float32: _capi.FP32, torch.bfloat16: _capi.BF16, torch.float8_e4m3fn: _capi.E4M3}
    return _t


def _ptr(t):
    return None if t is None else t.data_ptr()


class SequenceOps(object):
    """Mixin of ``CRNN``: needs ``_h``, ``_lib``, ``device``, ``precision``."""

    def _tensors(self, what, **named):
        """Checks every tensor's device and gradient; the stream to run on."""
        torch = _t
        for name, t in named.items():
            if t is None:
                continue
            if not isinstance(t, torch.Tensor):
                raise TypeError("%s: %s is not a tensor" % (what, name))
            if not t.is_cuda or t.device.index != self.device:
                raise ValueError("%s: %s is on %s, the handle on cuda:%d" % (what, name, t.device, self.device))
            if t.requires_grad and torch.is_grad_enabled():
                raise ValueError("%s: %s requires a gradient; these operators are for inference (torch.no_grad())" % (what, name))
            if t.dim() and t.shape[-1] > 1 and t.stride(-1) != 1:
                raise ValueError("%s: the last dimension of %s is not contiguous" % (what, name))
        return torch.cuda.current_stream(self.device).cuda_stream

    @staticmethod
    def _rows(what, name, t, n):
        """(rows, row stride) of a tensor [..., n] whose rows are evenly spaced."""
        if t.dim() < 1 or t.shape[-1] != n:
            raise ValueError("%s: %s has shape %s, its last dimension should be %d" % (what, name, tuple(t.shape), n))
        if 0 in t.shape[:-1]:
            return 0, n
        if t.dim() == 2:
            m, ld = t.shape[0], t.stride(0)
        elif t.dim() == 1:
            return 1, n
        else:
            m, ld, at = 1, None, None
            for size, st in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
                if size == 1:
                    continue
                if ld is None:
                    ld = st
                elif st != at:
                    raise ValueError("%s: the rows of %s are not evenly spaced" % (what, name))
                m, at = m * size, st * size
            ld = n if ld is None else ld
        return m, ld if m > 1 else max(ld, n)

    def _vector(self, what, name, t, n):
        if t is not None and (t.dtype is not _t.float32 or t.dim() != 1 or t.shape[0] != n):
            raise ValueError("%s: %s has to be float32 [%d], got %s %s" % (what, name, n, t.dtype, tuple(t.shape)))

    def linear(self, x, w, bias=None, residual=None, act="none", x_scale=None, w_scale=None, out_dtype=None, out=None):
        """act(x w^T + bias) + residual: x [..., k], w [n, k], bias float32 [n], residual and the result [..., n].

        x and w are both float32 (multiplied with fp32 accuracy), bfloat16 or float8_e4m3fn; the latter with float32
        ``x_scale`` (one per row of x) and ``w_scale`` [n].  act: none, relu, leaky (0.2), gelu, silu.  ``out_dtype``
        float32 or bfloat16: of the result and the residual (default: x's, bfloat16 for float8).  ``out`` may be the
        residual itself."""
        torch = _torch()
        stream = self._tensors("linear", x=x, w=w, bias=bias, residual=residual, x_scale=x_scale, w_scale=w_scale, out=out)
        if w.dim() != 2 or x.dim() < 1 or x.dtype is not w.dtype or x.dtype not in _types:
            raise ValueError("linear: x and w have to be [..., k] and [n, k], both float32, bfloat16 or float8_e4m3fn; got %s %s, %s %s"
                             % (x.dtype, tuple(x.shape), w.dtype, tuple(w.shape)))
        if act not in ACTS:
            raise ValueError("linear: unknown activation %r" % (act,))
        n, k = w.shape
        m, ldx = self._rows("linear", "x", x, k)
        shape = x.shape[:-1] + (n,)
        if out_dtype is None:
            out_dtype = out.dtype if out is not None else torch.float32 if x.dtype is torch.float32 else torch.bfloat16
        if out_dtype is not torch.float32 and out_dtype is not torch.bfloat16:
            raise ValueError("linear: out_dtype has to be float32 or bfloat16, got %s" % (out_dtype,))
        self._vector("linear", "bias", bias, n)
        self._vector("linear", "w_scale", w_scale, n)
        if x_scale is not None:
            if x_scale.dtype is not torch.float32 or x_scale.numel() != m or not x_scale.is_contiguous():
                raise ValueError("linear: x_scale has to be contiguous float32, one per row of x")
        if out is None:
            out = torch.empty(shape, dtype=out_dtype, device=x.device)
        elif out.shape != shape or out.dtype is not out_dtype:
            raise ValueError("linear: out has to be %s %s, got %s %s" % (out_dtype, tuple(shape), out.dtype, tuple(out.shape)))
        ldr = 0
        if residual is not None:
            if residual.shape != shape or residual.dtype is not out_dtype:
                raise ValueError("linear: residual has to be %s %s, got %s %s" % (out_dtype, tuple(shape), residual.dtype, tuple(residual.shape)))
            ldr = self._rows("linear", "residual", residual, n)[1]
        ldy = self._rows("linear", "out", out, n)[1]
        if m == 0:
            return out
        a = _capi.LinearArgs(m, n, k, x.data_ptr(), w.data_ptr(), ldx, w.stride(0) if n > 1 else k, _ptr(x_scale), _ptr(w_scale), _ptr(bias),
                             _ptr(residual), ldr, out.data_ptr(), ldy, _types[x.dtype], _types[out_dtype], ACTS[act], 0)
        rc = self._lib.crnn_linear(self._h, C.byref(a), stream)
        if rc:
            _capi.check(self._h, rc)
        return out

    def rms_norm(self, x, gain, residual=None, eps=1e-6, out_dtype=None, out=None, sum_out=None):
        """t = x + residual, y = t / sqrt(mean(t^2) + eps) * gain over the last dimension: RmsNorm(y, scale, sum).

        x and residual float32 or bfloat16, gain float32 [n].  ``out_dtype``: x's (default) or float8_e4m3fn, which adds
        ``scale``, one float32 per row with y = values * scale (the operands ``linear`` takes).  ``sum`` is t in x's type;
        without a residual None.  ``sum_out`` may be x or residual themselves, ``out`` too where the types agree."""
        torch = _torch()
        stream = self._tensors("rms_norm", x=x, gain=gain, residual=residual, out=out, sum_out=sum_out)
        if x.dim() < 1 or (x.dtype is not torch.float32 and x.dtype is not torch.bfloat16):
            raise ValueError("rms_norm: x has to be float32 or bfloat16 [..., n], got %s %s" % (x.dtype, tuple(x.shape)))
        n = x.shape[-1]
        self._vector("rms_norm", "gain", gain, n)
        out_dtype = out_dtype or (out.dtype if out is not None else x.dtype)
        if out_dtype is not x.dtype and out_dtype is not torch.float8_e4m3fn:
            raise ValueError("rms_norm: out_dtype has to be x's or float8_e4m3fn, got %s" % (out_dtype,))
        m, ldx = self._rows("rms_norm", "x", x, n)
        for name, t, dt in (("residual", residual, x.dtype), ("out", out, out_dtype), ("sum_out", sum_out, x.dtype)):
            if t is not None and (t.shape != x.shape or t.dtype is not dt):
                raise ValueError("rms_norm: %s has to be %s %s, got %s %s" % (name, dt, tuple(x.shape), t.dtype, tuple(t.shape)))
        if sum_out is not None and residual is None:
            raise ValueError("rms_norm: sum_out without a residual")
        y = out if out is not None else torch.empty(x.shape, dtype=out_dtype, device=x.device)
        scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device) if out_dtype is torch.float8_e4m3fn else None
        total = sum_out
        ldr = lds = 0
        if residual is not None:
            if total is None:
                total = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            ldr, lds = self._rows("rms_norm", "residual", residual, n)[1], self._rows("rms_norm", "sum_out", total, n)[1]
        ldy = self._rows("rms_norm", "out", y, n)[1]
        if m and n:
            a = _capi.RmsNormArgs(m, n, x.data_ptr(), ldx, _ptr(residual), ldr, gain.data_ptr(), _ptr(total), lds, y.data_ptr(), ldy, _ptr(scale), eps,
                                  _types[x.dtype], _types[out_dtype], 0)
            rc = self._lib.crnn_rms_norm(self._h, C.byref(a), stream)
            if rc:
                _capi.check(self._h, rc)
        return RmsNorm(y, scale, total)

    def cross_attention(self, q, k, v, lengths=None, mask=None, scale=None, out=None):
        """Attention of q [b, t, heads, d] over k, v [b, s, kv_heads, d] -> [b, t, heads, d], float32 or bfloat16, d <= 128.

        Query head h reads key head h // (heads // kv_heads).  ``lengths`` int32 [b]: the keys of each entry that exist;
        ``mask`` bool or uint8 [b, s]: the keys that count (both may be given).  A row without any key gives zeros; what the
        left-out keys hold is never looked at.  ``scale``: d ** -0.5."""
        torch = _torch()
        stream = self._tensors("cross_attention", q=q, k=k, v=v, lengths=lengths, mask=mask, out=out)
        if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
            raise ValueError("cross_attention: expected q [b, t, heads, d], k and v [b, s, kv_heads, d], got %s, %s, %s"
                             % (tuple(q.shape), tuple(k.shape), tuple(v.shape)))
        dt = q.dtype
        if (dt is not torch.float32 and dt is not torch.bfloat16) or k.dtype is not dt or v.dtype is not dt:
            raise ValueError("cross_attention: q, k and v have to be all float32 or all bfloat16, got %s, %s, %s" % (dt, k.dtype, v.dtype))
        b, t, heads, d = q.shape
        s, kv_heads = k.shape[1], k.shape[2]
        if lengths is not None and (lengths.dtype is not torch.int32 or lengths.shape != (b,)):
            raise ValueError("cross_attention: lengths has to be int32 [%d], got %s %s" % (b, lengths.dtype, tuple(lengths.shape)))
        if mask is not None and (mask.dtype not in (torch.bool, torch.uint8) or mask.shape != (b, s)):
            raise ValueError("cross_attention: mask has to be bool or uint8 [%d, %d], got %s %s" % (b, s, mask.dtype, tuple(mask.shape)))
        if out is None:
            out = torch.empty(q.shape, dtype=dt, device=q.device)
        elif out.shape != q.shape or out.dtype is not dt:
            raise ValueError("cross_attention: out has to be %s %s, got %s %s" % (dt, tuple(q.shape), out.dtype, tuple(out.shape)))
        i3 = _capi.I64x3
        a = _capi.CrossAttentionArgs(b, t, s, heads, kv_heads, d, _types[dt], q.data_ptr(), _ptr(k), _ptr(v), out.data_ptr(), i3(*q.stride()[:3]),
                                     i3(*k.stride()[:3]), i3(*v.stride()[:3]), i3(*out.stride()[:3]), _ptr(lengths), _ptr(mask),
                                     mask.stride(0) if mask is not None else 0, None, 0, d ** -0.5 if scale is None else scale, 0)
        need = self._lib.crnn_cross_attention_workspace(self._h, C.byref(a))
        if need:
            _capi.check(self._h, need)
            ws = torch.empty(need, dtype=torch.uint8, device=q.device)   # stream-ordered, as the tensors: freed when this call returns
            a.workspace, a.workspace_bytes = ws.data_ptr(), need
        rc = self._lib.crnn_cross_attention(self._h, C.byref(a), stream)
        if rc:
            _capi.check(self._h, rc)
        return out

    def line_states(self, lines, widths=None):
        """The recogniser as an encoder: uint8 [n, 32, w] lines on the handle's device -> (states [n, T, 512], lengths
        int32 [n]), T = crnn_out_len(w).  ``widths``: valid width of each line (host).  States are what the classifier reads
        (float32, bfloat16 with precision='bf16'), zeros behind a line's own length; ready on torch's current stream."""
        torch = _torch()
        stream = self._tensors("line_states", lines=lines)
        if lines.dtype is not torch.uint8 or lines.dim() != 3 or lines.shape[1] != 32 or not lines.is_contiguous() or lines.shape[0] == 0:
            raise ValueError("line_states: expected contiguous uint8 [n, 32, w], got %s %s" % (lines.dtype, tuple(lines.shape)))
        n, _, w = lines.shape
        wv = None
        if widths is not None:
            wv = np.ascontiguousarray(widths, dtype=np.int32)
            if wv.shape != (n,):
                raise ValueError("line_states: widths has to be [%d], got %s" % (n, wv.shape))
        T = max(0, self._lib.crnn_out_len(w))
        states = torch.empty((n, T, 512), dtype=torch.bfloat16 if self.precision == "bf16" else torch.float32, device=lines.device)
        lengths = torch.empty(n, dtype=torch.int32, device=lines.device)
        _capi.check(self._h, self._lib.crnn_states_device(self._h, lines.data_ptr(), n, w, wv.ctypes.data if wv is not None else None,
                                                          states.data_ptr(), lengths.data_ptr(), stream))
        return states, lengths
