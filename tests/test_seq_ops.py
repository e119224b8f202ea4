"""Argument checks of the sequence operators and the error bounds their tests use: no GPU."""
import ctypes as C

import numpy as np
import pytest
import torch

from ocr_amd.crnn import _capi
from tests import seq_reference as R


@pytest.fixture(scope="module")
def handle():
    lib = _capi.lib()
    h = C.c_void_p()
    cfg = _capi.Config(32, 1, 65, 256, 0, 1, 0, 1, 0, 0)
    assert lib.crnn_create(C.byref(cfg), C.byref(h)) == 0
    yield lib, h
    lib.crnn_destroy(h)


def fields(struct, a, **change):
    d = dict(a, **change)
    return struct(*[d[n] for n, _ in struct._fields_])


P = 1 << 32      # a pointer that is never followed: every call here is refused, or has nothing to do
LIN = dict(m=4, n=8, k=16, x=P, w=P + 4096, ldx=16, ldw=16, x_scale=None, w_scale=None, bias=P + 8192, residual=None, ldr=0, y=P + 16384, ldy=8,
           in_type=_capi.BF16, out_type=_capi.BF16, act=0, reserved=0)


@pytest.mark.parametrize("change, word", [
    (dict(x=None), "null"), (dict(w=None), "null"), (dict(y=None), "null"), (dict(m=-1), "range"), (dict(n=0), "range"), (dict(k=0), "range"),
    (dict(m=1 << 31), "range"), (dict(in_type=3), "in_type"), (dict(out_type=_capi.E4M3), "out_type"), (dict(act=5), "activation"),
    (dict(act=-1), "activation"), (dict(ldy=7), "ldy"), (dict(ldx=-1), "stride"), (dict(ldw=-1), "stride"), (dict(x_scale=P + 9000), "scales"),
    (dict(x=P + 1), "aligned"), (dict(bias=P + 8193), "aligned"), (dict(y=P), "overlaps"), (dict(y=P + 4096), "overlaps"), (dict(y=P + 8192), "overlaps"),
    (dict(residual=P + 16386, ldr=8), "residual"), (dict(residual=P + 16384, ldr=9), "residual"), (dict(reserved=1), "reserved"),
    (dict(ldx=1 << 41), "stride"), (dict(m=1 << 30, ldy=1 << 30), "stride"), (dict(n=1 << 30, ldw=1 << 40), "stride"),
    (dict(y=P + 16, ldx=24, ldy=24, n=9), "overlaps"),      # columns 8..16 of the buffer whose columns 0..15 are x
])
def test_linear_refuses(handle, change, word):
    lib, h = handle
    a = fields(_capi.LinearArgs, LIN, **change)
    assert lib.crnn_linear(h, C.byref(a), None) == _capi.CRNN_ERR_ARG
    assert word in lib.crnn_last_error(h).decode()


NORM = dict(m=4, n=16, x=P, ldx=16, residual=P + 4096, ldr=16, gain=P + 8192, sum=P + 12288, lds=16, y=P + 16384, ldy=16, y_scale=None, eps=1e-6,
            in_type=_capi.BF16, out_type=_capi.BF16, reserved=0)


@pytest.mark.parametrize("change, word", [
    (dict(x=None), "null"), (dict(gain=None), "null"), (dict(y=None), "null"), (dict(m=-1), "range"), (dict(n=0), "range"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(in_type=_capi.E4M3), "in_type"), (dict(out_type=_capi.FP32), "out_type"), (dict(y_scale=P + 20000), "y_scale"),
    (dict(out_type=_capi.E4M3), "y_scale"), (dict(ldy=15), "overlap"), (dict(lds=15), "overlap"), (dict(ldx=-2), "stride"), (dict(x=P + 1), "aligned"),
    (dict(y=P + 2), "overlaps an input"), (dict(y=P, ldy=17), "overlaps an input"), (dict(sum=P + 16384), "two outputs"), (dict(y=P + 8192), "overlaps an input"),
    (dict(m=1 << 30, ldr=1 << 40), "stride"), (dict(reserved=7), "reserved"), (dict(out_type=_capi.E4M3, y_scale=P + 20000, y=P), "overlaps an input"),
])
def test_rms_norm_refuses(handle, change, word):
    lib, h = handle
    a = fields(_capi.RmsNormArgs, NORM, **change)
    assert lib.crnn_rms_norm(h, C.byref(a), None) == _capi.CRNN_ERR_ARG
    assert word in lib.crnn_last_error(h).decode()


ATT = dict(batch=2, q_len=3, kv_len=5, heads=4, kv_heads=2, head_dim=8, type=_capi.BF16, q=P, k=P + 4096, v=P + 8192, out=P + 16384,
           q_stride=_capi.I64x3(96, 32, 8), k_stride=_capi.I64x3(80, 16, 8), v_stride=_capi.I64x3(80, 16, 8), out_stride=_capi.I64x3(96, 32, 8),
           lengths=None, mask=None, mask_stride=0, workspace=None, workspace_bytes=0, scale=0.3, reserved=0)


@pytest.mark.parametrize("change, word", [
    (dict(q=None), "null"), (dict(k=None), "null"), (dict(v=None), "null"), (dict(out=None), "null"), (dict(heads=3), "multiple"), (dict(heads=0), "multiple"),
    (dict(kv_heads=0), "multiple"), (dict(head_dim=0), "head_dim"), (dict(head_dim=129), "head_dim"), (dict(batch=-1), "range"), (dict(kv_len=1 << 31), "range"),
    (dict(batch=1 << 20, q_len=1 << 20), "passes"), (dict(type=_capi.E4M3), "type"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(q_stride=_capi.I64x3(-1, 0, 0)), "stride"), (dict(out_stride=_capi.I64x3(96, 32, 7)), "rows of out"), (dict(out_stride=_capi.I64x3(95, 32, 8)), "rows of out"),
    (dict(out_stride=_capi.I64x3(0, 32, 8)), "rows of out"), (dict(out=P), "overlaps q"), (dict(out=P + 4096), "overlaps k"), (dict(out=P + 8192), "overlaps k"),
    (dict(mask=P + 16400, mask_stride=5), "mask"), (dict(mask=P, mask_stride=-1), "mask_stride"), (dict(lengths=P + 16388), "lengths"), (dict(lengths=P + 2), "aligned"),
    (dict(q=P + 1), "aligned"), (dict(reserved=1), "reserved"), (dict(kv_len=1 << 30, v_stride=_capi.I64x3(80, 1 << 40, 8)), "stride"),
    (dict(q_len=1 << 20, out_stride=_capi.I64x3(96, 1 << 40, 8)), "stride"), (dict(mask=P, mask_stride=1 << 41), "mask_stride"),
])
def test_cross_attention_refuses(handle, change, word):
    lib, h = handle
    a = fields(_capi.CrossAttentionArgs, ATT, **change)
    assert lib.crnn_cross_attention(h, C.byref(a), None) == _capi.CRNN_ERR_ARG
    assert word in lib.crnn_last_error(h).decode()


def test_nothing_to_do_is_no_error(handle):
    lib, h = handle
    assert lib.crnn_linear(h, C.byref(fields(_capi.LinearArgs, LIN, m=0, x=None, y=None)), None) == 0
    assert lib.crnn_rms_norm(h, C.byref(fields(_capi.RmsNormArgs, NORM, m=0, x=None)), None) == 0
    for none in (dict(batch=0), dict(q_len=0)):
        a = fields(_capi.CrossAttentionArgs, ATT, q=None, **none)
        assert lib.crnn_cross_attention(h, C.byref(a), None) == 0 and lib.crnn_cross_attention_workspace(h, C.byref(a)) == 0


def test_workspace_is_told_from_sizes_type_and_strides(handle):
    lib, h = handle
    ask = lambda **c: lib.crnn_cross_attention_workspace(h, C.byref(fields(_capi.CrossAttentionArgs, ATT, **dict(dict(q=None, k=None, v=None, out=None), **c))))
    assert ask() == 0                                               # five keys: nothing to share out
    splits = ask(kv_len=100000) / (2 * 4 * 3 * (8 + 2) * 4)         # batch, heads, q_len; head_dim values, maximum and sum in 32 bits
    assert splits == int(splits) and 2 <= splits <= 64
    assert ask(kv_len=100000, k_stride=_capi.I64x3(1600000, 17, 8)) == 0      # not in whole 16 bytes: the kernel that shares nothing
    assert ask(kv_len=(1 << 31) - 1) == 0                           # key numbers a step past these would not be ints
    assert ask(kv_len=100000, batch=1, k_stride=_capi.I64x3(3, 16, 8)) == ask(kv_len=100000, batch=1)   # a stride that no step is made by


def test_null_arguments(handle):
    lib, h = handle
    for f in (lib.crnn_linear, lib.crnn_rms_norm, lib.crnn_cross_attention):
        assert f(h, None, None) == _capi.CRNN_ERR_ARG and f(None, None, None) == _capi.CRNN_ERR_ARG
    assert lib.crnn_cross_attention_workspace(h, None) == _capi.CRNN_ERR_ARG
    assert lib.crnn_states_device(h, None, 1, 64, None, None, None, None) == _capi.CRNN_ERR_ARG
    assert lib.crnn_states_device(h, P, 1, 64, None, P + 8, None, None) == _capi.CRNN_ERR_ARG


def test_tensors_of_the_host_are_refused():
    from ocr_amd.crnn.network_hip import CRNN
    m = CRNN(32, 1, 65, 256, device=0)
    x = torch.zeros(2, 16)
    for call in (lambda: m.linear(x, x), lambda: m.rms_norm(x, x[0]), lambda: m.cross_attention(x.view(1, 2, 2, 8), x.view(1, 2, 2, 8), x.view(1, 2, 2, 8)),
                 lambda: m.line_states(torch.zeros(1, 32, 64, dtype=torch.uint8))):
        with pytest.raises(ValueError, match="on cpu"):
            call()
    with pytest.raises(TypeError):
        m.linear(x.numpy(), x)


def test_line_attention_checks_its_weights():
    from ocr_amd.crnn.attention import LineAttention
    w = {"norm.weight": torch.ones(64), "q.weight": torch.zeros(32, 64), "kv.weight": torch.zeros(64, 512), "out.weight": torch.zeros(64, 32)}
    assert LineAttention(None, w, heads=4).d == 8
    for bad in (dict(w, extra=w["norm.weight"]), {k: v for k, v in w.items() if k != "out.weight"}, dict(w, **{"kv.weight": torch.zeros(64, 511)}),
                dict(w, **{"q.weight": w["q.weight"].bfloat16()}), dict(w, **{"q.scale": torch.ones(32)}), dict(w, **{"norm.weight": torch.ones(63)})):
        with pytest.raises(ValueError):
            LineAttention(None, bad, heads=4)
    with pytest.raises(ValueError):
        LineAttention(None, w, heads=4, kv_heads=3)


def test_packed_arguments_are_the_structs():
    from ocr_amd.crnn import seq_ops
    for packer, struct in ((seq_ops._LINEAR, _capi.LinearArgs), (seq_ops._RMS_NORM, _capi.RmsNormArgs), (seq_ops._CROSS_ATTENTION, _capi.CrossAttentionArgs)):
        assert packer.size == C.sizeof(struct)
        values, flat = [], []
        for i, (name, kind) in enumerate(struct._fields_):
            v = i + 1.5 if kind is C.c_float else kind(i + 1, i + 51, i + 101) if kind is _capi.I64x3 else i + 1
            values.append(v)
            flat += list(v) if kind is _capi.I64x3 else [v]
        assert packer.pack(*flat) == bytes(struct(*values))


def test_rows_of_a_tensor():
    from ocr_amd.crnn.seq_ops import SequenceOps
    rows = SequenceOps._rows
    t = torch.zeros(6, 5, 32)
    assert rows("f", "t", t, 32) == (30, 32) and rows("f", "t", t[:, 0], 32) == (6, 160) and rows("f", "t", t[:, :, :16], 16) == (30, 32)
    assert rows("f", "t", t[0, 0], 32) == (1, 32) and rows("f", "t", t[:1, 0], 32) == (1, 32) and rows("f", "t", t[:, :0], 32)[0] == 0 and rows("f", "t", t[:1, 2:3], 32) == (1, 32)
    assert rows("f", "t", t[0, :1].expand(7, 32), 32) == (7, 0)
    with pytest.raises(ValueError):
        rows("f", "t", t[:, :4], 32)
    with pytest.raises(ValueError):
        rows("f", "t", t, 16)


@pytest.mark.parametrize("act", ["none", "relu", "leaky", "gelu", "silu"])
def test_the_linear_bound_holds_for_32_bit_sums_and_not_for_a_mistake(act):
    g = torch.Generator().manual_seed(1)
    x, w, b = torch.randn(9, 70, generator=g), torch.randn(13, 70, generator=g), torch.randn(13, generator=g)
    want, err = R.linear(x, w, b, act=act)
    got = R.act64((x @ w.t() + b), act)
    R.check(got, want, err)
    w2 = w.clone()
    w2[3, 69] = 0
    with pytest.raises(AssertionError):
        R.check(R.act64(x @ w2.t() + b, act), want, err)


def test_the_attention_bound_holds_for_32_bits_and_not_for_a_lost_key():
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(2, n, 4, 8, generator=g) for n in (3, 50, 50))
    want, err = R.attention(q, k, v, lengths=torch.tensor([50, 17]))
    z = torch.einsum("bthd,bshd->bhts", q, k) * 8 ** -0.5
    z[1, :, :, 17:] = -float("inf")
    R.check(torch.einsum("bhts,bshd->bthd", torch.softmax(z, 3), v), want, err)
    z[1, :, :, 16:] = -float("inf")
    with pytest.raises(AssertionError):
        R.check(torch.einsum("bhts,bshd->bthd", torch.softmax(z, 3), v), want, err)


def host_face(monkeypatch):
    """The torch face on host tensors with a library that only remembers its calls: what Python decides before and beside them."""
    from ocr_amd.crnn import seq_ops

    class Lib(object):
        def __init__(self):
            self.calls = []

        def __getattr__(self, name):
            return lambda *a: self.calls.append(name) or 0

    seq_ops._torch()
    monkeypatch.setattr(seq_ops, "_stream", lambda device: 0)
    face = seq_ops.SequenceOps()
    face.device, face._h, face._lib, face.precision = -1, None, Lib(), "fp32"
    return face


def test_rms_norm_of_rows_without_values_has_its_scale(monkeypatch):
    """The largest of no values counts as 0: the smallest scale, never what the memory held before."""
    face = host_face(monkeypatch)
    monkeypatch.setattr(torch.Tensor, "new_empty", lambda t, shape, dtype=None: torch.full(tuple(shape), 7.0).to(dtype or t.dtype))
    for shape in ((5, 0), (2, 3, 0)):
        got = face.rms_norm(torch.zeros(shape), torch.zeros(0), out_dtype=torch.float8_e4m3fn)
        assert got.y.shape == shape and got.scale.shape == shape[:-1] and (got.scale == 2.0 ** -126).all()
    assert face.rms_norm(torch.zeros(0, 0), torch.zeros(0), out_dtype=torch.float8_e4m3fn).scale.shape == (0,)
    assert face._lib.calls == []


def test_forward_mode_tangents_are_refused(monkeypatch):
    """A tensor with a tangent would come back without one: refused, as what requires a gradient is, unless such derivatives are off."""
    import torch.autograd.forward_ad as fwd
    face = host_face(monkeypatch)
    x, w, q = torch.ones(4, 16), torch.ones(8, 16), torch.ones(2, 3, 4, 8)
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))
        for call in (lambda: face.linear(dual(x), w), lambda: face.linear(x, dual(w)), lambda: face.linear(x, w, bias=dual(w[:, 0].contiguous())),
                     lambda: face.rms_norm(dual(x), x[0]), lambda: face.rms_norm(x, dual(x[0])), lambda: face.rms_norm(x, x[0], residual=dual(x)),
                     lambda: face.cross_attention(dual(q), q, q), lambda: face.cross_attention(q, q, dual(q))):
            with pytest.raises(ValueError, match="gradient"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="gradient"):      # (no_grad is of reverse mode only)
                call()
        assert face._lib.calls == []
        assert face.linear(x, w).shape == (4, 8)                                 # the level alone is no reason
        assert face.cross_attention(q, q, q, lengths=torch.ones(2, dtype=torch.int32), mask=torch.ones(2, 3, dtype=torch.bool)).shape == q.shape
        with torch.inference_mode():
            assert face.linear(x, w).shape == (4, 8)
    assert face.linear(x, w).shape == (4, 8) and face._lib.calls == ["crnn_linear", "crnn_cross_attention_workspace", "crnn_cross_attention"] + ["crnn_linear"] * 2


def test_line_attention_checks_head_size_biases_and_scales():
    """What no call of the layer could run on is refused where it is made."""
    from ocr_amd.crnn.attention import LineAttention

    def weights(dim=64, heads=4, d=8, dt=torch.float32, **more):
        return dict({"norm.weight": torch.ones(dim), "q.weight": torch.zeros(heads * d, dim, dtype=dt), "kv.weight": torch.zeros(2 * heads * d, 512, dtype=dt),
                     "out.weight": torch.zeros(dim, heads * d, dtype=dt), "q.bias": torch.zeros(heads * d), "kv.bias": torch.zeros(2 * heads * d),
                     "out.bias": torch.zeros(dim)}, **more)
    for d in (1, 20, 36, 128):
        assert LineAttention(None, weights(d=d), heads=4).d == d
    q8 = dict(weights(dt=torch.bfloat16), **{"q.weight": torch.zeros(32, 64).to(torch.float8_e4m3fn), "q.scale": torch.ones(32)})
    assert LineAttention(None, q8, heads=4).q8
    for bad in (weights(d=200), weights(d=129), weights(d=0)):
        with pytest.raises(ValueError, match="head"):
            LineAttention(None, bad, heads=4)
    for w, change in ((weights(), {"q.bias": torch.zeros(31)}), (weights(), {"kv.bias": torch.zeros(32)}), (weights(), {"out.bias": torch.zeros(1, 64)}),
                      (weights(), {"q.bias": torch.zeros(32).bfloat16()}), (weights(), {"norm.weight": torch.ones(64).bfloat16()}), (q8, {"q.scale": torch.ones(64)}),
                      (q8, {"q.scale": torch.ones(32).double()})):
        with pytest.raises(ValueError, match=next(iter(change))):
            LineAttention(None, dict(w, **change), heads=4)


def test_what_does_not_fit_is_a_type_or_value_error(monkeypatch):
    """Also a tensor that is missing, and what is no number."""
    face = host_face(monkeypatch)
    x, w, q = torch.ones(4, 16), torch.ones(8, 16), torch.ones(2, 3, 4, 8)
    for call in (lambda: face.linear(None, w), lambda: face.linear(x, None), lambda: face.rms_norm(None, x[0]), lambda: face.rms_norm(x, None),
                 lambda: face.cross_attention(None, q, q), lambda: face.cross_attention(q, None, q), lambda: face.cross_attention(q, q, None),
                 lambda: face.line_states(None), lambda: face.rms_norm(x, x[0], eps=None), lambda: face.cross_attention(q, q, q, scale="1")):
        with pytest.raises(TypeError):
            call()
    assert face._lib.calls == []
    face.rms_norm(x, x[0], eps=np.float32(1e-5))
    face.cross_attention(q, q, q, scale=torch.tensor(0.5))
    assert face._lib.calls == ["crnn_rms_norm", "crnn_cross_attention_workspace", "crnn_cross_attention"]
