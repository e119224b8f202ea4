"""Operators on sequences of states, on torch tensors in device memory: the torch face of crnn_linear, crnn_rms_norm,
crnn_cross_attention and crnn_states_device (include/crnn_hip.h), as methods of ``CRNN``.

They run on torch's current stream of the handle's device and return without waiting; outputs are new tensors unless
``out`` is given.  Tensors have to be on the handle's device, with the last dimension contiguous; anything else about their
strides is taken as it is.  Inference only: a call that autograd would have to record is refused, one on tensors with
forward-mode tangents too.
"""
import collections
import struct

import numpy as np

from . import _capi

RmsNorm = collections.namedtuple("RmsNorm", ["y", "scale", "sum"])
RmsNorm.__doc__ = "What rms_norm returns: y, its row scales (8-bit outputs only, else None), the sum (with a residual only, else None)."

ACTS = {"none": 0, None: 0, "relu": 1, "leaky": 2, "gelu": 3, "silu": 4}

_t = None       # torch, imported by the first call: the recogniser itself does without
_types = None   # torch dtype -> CRNN_* type
_f32 = _bf16 = _e4m3 = None
_stream = None  # device index -> its current stream
_forward = None  # torch.autograd.forward_ad

# The argument structs of include/crnn_hip.h as they lie in memory: packing a few integers costs a fifth of filling a
# ctypes.Structure, and a call's host time is what small operators cost.
_LINEAR = struct.Struct("@3q2P2q3PPqPq4i")
_RMS_NORM = struct.Struct("@2qPqPqPPqPqPf3i")
_CROSS_ATTENTION = struct.Struct("@3q4i4P12q2Pq" + "Pqfi")


def _torch():
    global _t, _types, _stream, _forward, _f32, _bf16, _e4m3
    if _t is None:
        import torch
        _f32, _bf16, _e4m3 = torch.float32, torch.bfloat16, torch.float8_e4m3fn
        _types = {_f32: _capi.FP32, _bf16: _capi.BF16, _e4m3: _capi.E4M3}
        _stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)
        import torch.autograd.forward_ad as _forward
        _t = torch
    return _t


def _ptr(t):
    return 0 if t is None else t.data_ptr()


class SequenceOps(object):
    """Mixin of ``CRNN``: needs ``_h``, ``_lib``, ``device``, ``precision``."""

    def _tensors(self, what, names, tensors):
        """Device, gradient and last dimension of every tensor; the stream to run on."""
        grad, dev = _t.is_grad_enabled(), self.device
        for t in tensors:
            if t is not None:
                try:
                    if t.get_device() == dev and t.stride(-1) == 1 and not (grad and t.requires_grad):
                        continue
                except (AttributeError, IndexError, TypeError):
                    pass
                self._refuse(what, names, tensors, grad)
                break
        if getattr(_forward, "_current_level", 0) >= 0:   # (within a level of forward-mode derivatives only)
            self._refuse_tangents(what, names, tensors)
        return _stream(dev)

    @staticmethod
    def _refuse_tangents(what, names, tensors):
        if not _t._C._is_fwd_grad_enabled():
            return
        for name, t in zip(names, tensors):
            if t is not None and _forward.unpack_dual(t).tangent is not None:
                raise ValueError("%s: %s has a forward-mode gradient; these operators are for inference" % (what, name))

    def _refuse(self, what, names, tensors, grad):
        """The check in full, for a call that did not pass at first sight (a last dimension of one may have any stride)."""
        for name, t in zip(names, tensors):
            if t is None:
                continue
            try:
                at = t.get_device()
            except AttributeError:
                raise TypeError("%s: %s is not a tensor" % (what, name)) from None
            if at != self.device:
                raise ValueError("%s: %s is on %s, the handle on cuda:%d" % (what, name, t.device, self.device))
            if grad and t.requires_grad:
                raise ValueError("%s: %s requires a gradient; these operators are for inference (torch.no_grad())" % (what, name))
            if t.dim() and t.stride(-1) != 1 and t.shape[-1] > 1:
                raise ValueError("%s: the last dimension of %s is not contiguous" % (what, name))

    @staticmethod
    def _rows(what, name, t, n):
        """(rows, row stride) of a tensor [..., n] whose rows are evenly spaced."""
        shape = t.shape
        if len(shape) == 2 and shape[1] == n:
            m = shape[0]
            return (m, t.stride(0)) if m > 1 else (m, n)
        if len(shape) < 1 or shape[-1] != n:
            raise ValueError("%s: %s has shape %s, its last dimension should be %d" % (what, name, tuple(shape), n))
        if 0 in shape[:-1]:
            return 0, n
        m, ld, at = 1, None, None
        for size, st in zip(reversed(shape[:-1]), reversed(t.stride()[:-1])):
            if size == 1:
                continue
            if ld is None:
                ld = st
            elif st != at:
                raise ValueError("%s: the rows of %s are not evenly spaced" % (what, name))
            m, at = m * size, st * size
        return m, n if ld is None else ld

    @staticmethod
    def _vector(what, name, t, n):
        if t.dtype is not _f32 or t.shape != (n,):
            raise ValueError("%s: %s has to be float32 [%d], got %s %s" % (what, name, n, t.dtype, tuple(t.shape)))

    @staticmethod
    def _like(what, name, t, shape, dtype):
        if t.shape != shape or t.dtype is not dtype:
            raise ValueError("%s: %s has to be %s %s, got %s %s" % (what, name, dtype, tuple(shape), t.dtype, tuple(t.shape)))

    def linear(self, x, w, bias=None, residual=None, act="none", x_scale=None, w_scale=None, out_dtype=None, out=None):
        """act(x w^T + bias) + residual: x [..., k], w [n, k], bias float32 [n], residual and the result [..., n].

        x and w are both float32 (each product to 2^-24), bfloat16 or float8_e4m3fn; the latter with float32
        ``x_scale`` (one per row of x) and ``w_scale`` [n].  act: none, relu, leaky (0.2), gelu, silu.  ``out_dtype``
        float32 or bfloat16: of the result and the residual (default: x's, bfloat16 for float8).  ``out`` may be the
        residual itself."""
        torch = _t or _torch()
        if x is None or w is None:
            raise TypeError("linear: x or w is missing")
        stream = self._tensors("linear", ("x", "w", "bias", "residual", "x_scale", "w_scale", "out"), (x, w, bias, residual, x_scale, w_scale, out))
        dt = x.dtype
        if w.dim() != 2 or w.dtype is not dt or dt not in _types:
            raise ValueError("linear: x and w have to be [..., k] and [n, k], both float32, bfloat16 or float8_e4m3fn; got %s %s, %s %s"
                             % (dt, tuple(x.shape), w.dtype, tuple(w.shape)))
        if act not in ACTS:
            raise ValueError("linear: unknown activation %r" % (act,))
        n, k = w.shape
        m, ldx = self._rows("linear", "x", x, k)
        shape = (m, n) if x.dim() == 2 else x.shape[:-1] + (n,)
        if out_dtype is None:
            out_dtype = out.dtype if out is not None else _f32 if dt is _f32 else _bf16
        if out_dtype is not _f32 and out_dtype is not _bf16:
            raise ValueError("linear: out_dtype has to be float32 or bfloat16, got %s" % (out_dtype,))
        if bias is not None:
            self._vector("linear", "bias", bias, n)
        if w_scale is not None:
            self._vector("linear", "w_scale", w_scale, n)
        if x_scale is not None and (x_scale.dtype is not _f32 or x_scale.numel() != m or not x_scale.is_contiguous()):
            raise ValueError("linear: x_scale has to be contiguous float32, one per row of x")
        if out is None:
            out = x.new_empty(shape) if out_dtype is dt else x.new_empty(shape, dtype=out_dtype)
            ldy = n
        else:
            self._like("linear", "out", out, shape, out_dtype)
            ldy = self._rows("linear", "out", out, n)[1]
        ldr = 0
        if residual is not None:
            self._like("linear", "residual", residual, shape, out_dtype)
            ldr = self._rows("linear", "residual", residual, n)[1]
        if m == 0:
            return out
        rc = self._lib.crnn_linear(self._h, _LINEAR.pack(
            m, n, k, x.data_ptr(), w.data_ptr(), ldx, w.stride(0) if n > 1 else k, _ptr(x_scale), _ptr(w_scale), _ptr(bias), _ptr(residual), ldr,
            out.data_ptr(), ldy, _types[dt], _types[out_dtype], ACTS[act], 0), stream)
        if rc:
            _capi.check(self._h, rc)
        return out

    def rms_norm(self, x, gain, residual=None, eps=1e-6, out_dtype=None, out=None, sum_out=None):
        """t = x + residual, y = t / sqrt(mean(t^2) + eps) * gain over the last dimension: RmsNorm(y, scale, sum).

        x and residual float32 or bfloat16, gain float32 [n].  ``out_dtype``: x's (default) or float8_e4m3fn, which adds
        ``scale``, one float32 per row with y = values * scale (the operands ``linear`` takes).  ``sum`` is t in x's type;
        without a residual None.  ``sum_out`` may be x or residual themselves, ``out`` too where the types agree."""
        torch = _t or _torch()
        if x is None or gain is None:
            raise TypeError("rms_norm: x or gain is missing")
        stream = self._tensors("rms_norm", ("x", "gain", "residual", "out", "sum_out"), (x, gain, residual, out, sum_out))
        dt, shape = x.dtype, x.shape
        if len(shape) < 1 or (dt is not _f32 and dt is not _bf16):
            raise ValueError("rms_norm: x has to be float32 or bfloat16 [..., n], got %s %s" % (dt, tuple(shape)))
        n = shape[-1]
        self._vector("rms_norm", "gain", gain, n)
        if not hasattr(eps, "__float__"):
            raise TypeError("rms_norm: eps is not a number, got %r" % (eps,))
        if out_dtype is None:
            out_dtype = out.dtype if out is not None else dt
        if out_dtype is not dt and out_dtype is not _e4m3:
            raise ValueError("rms_norm: out_dtype has to be x's or float8_e4m3fn, got %s" % (out_dtype,))
        m, ldx = self._rows("rms_norm", "x", x, n)
        if out is None:
            y, ldy = x.new_empty(shape) if out_dtype is dt else x.new_empty(shape, dtype=out_dtype), n
        else:
            self._like("rms_norm", "out", out, shape, out_dtype)
            y, ldy = out, self._rows("rms_norm", "out", out, n)[1]
        scale = x.new_empty(shape[:-1], dtype=_f32) if out_dtype is _e4m3 else None
        ldr = lds = 0
        total = None
        if residual is not None:
            self._like("rms_norm", "residual", residual, shape, dt)
            ldr = self._rows("rms_norm", "residual", residual, n)[1]
            if sum_out is None:
                total, lds = x.new_empty(shape), n
            else:
                self._like("rms_norm", "sum_out", sum_out, shape, dt)
                total, lds = sum_out, self._rows("rms_norm", "sum_out", sum_out, n)[1]
        elif sum_out is not None:
            raise ValueError("rms_norm: sum_out without a residual")
        if m and n:
            rc = self._lib.crnn_rms_norm(self._h, _RMS_NORM.pack(
                m, n, x.data_ptr(), ldx, _ptr(residual), ldr, gain.data_ptr(), _ptr(total), lds, y.data_ptr(), ldy, _ptr(scale), eps, _types[dt],
                _types[out_dtype], 0), stream)
            if rc:
                _capi.check(self._h, rc)
        elif m and scale is not None:
            scale.fill_(2.0 ** -126)   # rows without values: their largest is 0
        return RmsNorm(y, scale, total)

    def cross_attention(self, q, k, v, lengths=None, mask=None, scale=None, out=None):
        """Attention of q [b, t, heads, d] over k, v [b, s, kv_heads, d] -> [b, t, heads, d], float32 or bfloat16, d <= 128.

        Query head h reads key head h // (heads // kv_heads).  ``lengths`` int32 [b]: the keys of each entry that exist;
        ``mask`` bool or uint8 [b, s]: the keys that count (both may be given).  A row without any key gives zeros; what the
        left-out keys hold is never looked at.  ``scale``: d ** -0.5."""
        torch = _t or _torch()
        if q is None or k is None or v is None:
            raise TypeError("cross_attention: q, k or v is missing")
        stream = self._tensors("cross_attention", ("q", "k", "v", "lengths", "mask", "out"), (q, k, v, lengths, mask, out))
        qs, ks, dt = q.shape, k.shape, q.dtype
        if len(qs) != 4 or len(ks) != 4 or v.shape != ks or ks[0] != qs[0] or ks[3] != qs[3]:
            raise ValueError("cross_attention: expected q [b, t, heads, d], k and v [b, s, kv_heads, d], got %s, %s, %s" % (tuple(qs), tuple(ks), tuple(v.shape)))
        if (dt is not _f32 and dt is not _bf16) or k.dtype is not dt or v.dtype is not dt:
            raise ValueError("cross_attention: q, k and v have to be all float32 or all bfloat16, got %s, %s, %s" % (dt, k.dtype, v.dtype))
        b, t, heads, d = qs
        s, kv_heads = ks[1], ks[2]
        if lengths is not None and (lengths.dtype is not torch.int32 or lengths.shape != (b,)):
            raise ValueError("cross_attention: lengths has to be int32 [%d], got %s %s" % (b, lengths.dtype, tuple(lengths.shape)))
        if mask is not None and ((mask.dtype is not torch.bool and mask.dtype is not torch.uint8) or mask.shape != (b, s)):
            raise ValueError("cross_attention: mask has to be bool or uint8 [%d, %d], got %s %s" % (b, s, mask.dtype, tuple(mask.shape)))
        if out is None:
            out = q.new_empty(qs)
        else:
            self._like("cross_attention", "out", out, qs, dt)
        q1, q2, q3, _ = q.stride()
        k1, k2, k3, _ = k.stride()
        v1, v2, v3, _ = v.stride()
        o1, o2, o3, _ = out.stride()
        args = (b, t, s, heads, kv_heads, d, _types[dt], q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), q1, q2, q3, k1, k2, k3, v1, v2, v3,
                o1, o2, o3, _ptr(lengths), _ptr(mask), mask.stride(0) if mask is not None else 0)
        if scale is None:
            scale = d ** -0.5
        elif not hasattr(scale, "__float__"):
            raise TypeError("cross_attention: scale is not a number, got %r" % (scale,))
        a = _CROSS_ATTENTION.pack(*args, 0, 0, scale, 0)
        need = self._lib.crnn_cross_attention_workspace(self._h, a)
        if need:
            _capi.check(self._h, need)
            ws = q.new_empty(need, dtype=torch.uint8)   # stream-ordered, as all tensors: its memory is free again behind this call
            a = _CROSS_ATTENTION.pack(*args, ws.data_ptr(), need, scale, 0)
        rc = self._lib.crnn_cross_attention(self._h, a, stream)
        if rc:
            _capi.check(self._h, rc)
        return out

    def line_states(self, lines, widths=None):
        """The recogniser as an encoder: uint8 [n, 32, w] lines on the handle's device -> (states [n, T, 512], lengths
        int32 [n]), T = crnn_out_len(w).  ``widths``: valid width of each line (host).  States are what the classifier reads
        (float32, bfloat16 with precision='bf16'), zeros behind a line's own length; ready on torch's current stream."""
        torch = _torch()
        if lines is None:
            raise TypeError("line_states: lines are missing")
        stream = self._tensors("line_states", ("lines",), (lines,))
        if lines.dtype is not torch.uint8 or lines.dim() != 3 or lines.shape[1] != 32 or not lines.is_contiguous() or lines.shape[0] == 0:
            raise ValueError("line_states: expected contiguous uint8 [n, 32, w], got %s %s" % (lines.dtype, tuple(lines.shape)))
        n, _, w = lines.shape
        wv = None
        if widths is not None:
            wv = np.ascontiguousarray(widths, dtype=np.int32)
            if wv.shape != (n,):
                raise ValueError("line_states: widths has to be [%d], got %s" % (n, wv.shape))
        T = max(0, self._lib.crnn_out_len(w))
        states = torch.empty((n, T, 512), dtype=_bf16 if self.precision == "bf16" else _f32, device=lines.device)
        lengths = torch.empty(n, dtype=torch.int32, device=lines.device)
        _capi.check(self._h, self._lib.crnn_states_device(self._h, lines.data_ptr(), n, w, wv.ctypes.data if wv is not None else None,
                                                          states.data_ptr(), lengths.data_ptr(), stream))
        return states, lengths
