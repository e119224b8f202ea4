"""The sequence operators on the GPU against plain 64-bit forms (seq_reference.py), and run together as a decoder's layer."""
import threading

import numpy as np
import pytest
import torch

from tests import seq_reference as R

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}


@pytest.fixture(scope="module")
def crnn():
    from ocr_amd.crnn.network_hip import CRNN
    return CRNN(32, 1, 65, 256, device=0)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dt="fp32"):
    return torch.randn(*shape, generator=g, device="cuda").to(DT[dt])


# ------------------------------------------------------------------------------------------------------- linear
SIZES = [(1, 512, 512), (1, 7, 3), (2, 64, 5530), (3, 33, 65), (7, 517, 129), (16, 2048, 64), (17, 8200, 48), (48, 512, 5530), (64, 128, 33), (130, 96, 260),
         (71, 1, 1), (255, 512, 511), (300, 1000, 256), (513, 256, 2048), (1000, 64, 70), (257, 4096, 512), (2500, 576, 640), (5000, 513, 255),
         (12500, 264, 1025), (17000, 80, 770), (3000, 1040, 4100)]


def linear_inputs(m, k, n, dt, seed):
    g = gen(seed)
    if dt == "e4m3":
        x, w = randn(g, m, k).to(DT[dt]), randn(g, n, k).to(DT[dt])
        return x, w, dict(x_scale=torch.rand(m, generator=g, device="cuda") + 0.1, w_scale=torch.rand(n, generator=g, device="cuda") + 0.1)
    return randn(g, m, k, dt=dt), randn(g, n, k, dt=dt), {}


@pytest.mark.parametrize("dt", ["fp32", "bf16", "e4m3"])
@pytest.mark.parametrize("m, k, n", SIZES)
def test_linear(crnn, m, k, n, dt):
    x, w, sc = linear_inputs(m, k, n, dt, m + k)
    act = ["none", "relu", "leaky", "gelu", "silu"][(m + n) % 5]
    bias = randn(gen(1), n) if (m + k) % 3 else None
    for out in ("fp32", "bf16") if m * k * n < 1e8 else ("bf16" if dt != "fp32" else "fp32",):
        res = randn(gen(2), m, n, dt=out) if n % 2 else None
        got = crnn.linear(x, w, bias=bias, residual=res, act=act, out_dtype=DT[out], **sc)
        assert got.dtype is DT[out] and got.shape == (m, n)
        R.check(got, *R.linear(x, w, bias, res, act, out_dtype=DT[out], **sc), what=(act, out))


@pytest.mark.parametrize("dt", ["fp32", "bf16", "e4m3"])
@pytest.mark.parametrize("act", ["none", "relu", "leaky", "gelu", "silu"])
def test_linear_activations_and_epilogues(crnn, act, dt):
    for m in (5, 200, 700):
        x, w, sc = linear_inputs(m, 192, 320, dt, 3)
        bias, res = randn(gen(1), 320), randn(gen(2), m, 320)
        for b, r in ((None, None), (bias, None), (None, res), (bias, res)):
            R.check(crnn.linear(x, w, bias=b, residual=r, act=act, out_dtype=torch.float32, **sc), *R.linear(x, w, b, r, act, **sc))


@pytest.mark.parametrize("dt", ["fp32", "bf16", "e4m3"])
@pytest.mark.parametrize("m", [1, 9, 40, 300, 800])
def test_linear_strides_and_alignments(crnn, m, dt):
    """Column slices, rows that are not a multiple of 16 bytes apart, bases off the 16-byte grid; what lies beside y stays."""
    g = gen(m)
    k, n = 256, 192
    for lead, pitch_x, pitch_w, lead_y, pitch_y in ((0, 320, 256, 0, 192), (1, 259, 261, 3, 197), (16, 512, 304, 8, 256), (3, 320, 320, 1, 193)):
        X, W = randn(g, m, lead + pitch_x).to(DT[dt]), randn(g, n, lead + pitch_w).to(DT[dt])
        x, w = X[:, lead:lead + k], W[:, lead:lead + k]
        Y = torch.full((m, lead_y + pitch_y), 7.0, dtype=torch.bfloat16, device="cuda")
        Rs = randn(g, m, lead_y + pitch_y, dt="bf16")
        y, res = Y[:, lead_y:lead_y + n], Rs[:, lead_y:lead_y + n]
        got = crnn.linear(x, w, residual=res, out=y)
        assert got is y
        R.check(y, *R.linear(x, w, None, res, out_dtype=torch.bfloat16))
        assert (Y[:, :lead_y] == 7).all() and (Y[:, lead_y + n:] == 7).all()


def test_linear_leading_dimensions_broadcast_rows_and_in_place(crnn):
    g = gen(4)
    x, w = randn(g, 5, 6, 64), randn(g, 48, 64)
    got = crnn.linear(x[:, 2], w)
    assert got.shape == (5, 48)
    R.check(got, *R.linear(x[:, 2], w))
    assert crnn.linear(x, w).shape == (5, 6, 48) and crnn.linear(x[0, 0], w).shape == (48,) and crnn.linear(x[:0], w).shape == (0, 6, 48)
    row = randn(g, 1, 64).expand(70, 64)
    R.check(crnn.linear(row, w), *R.linear(row, w))
    t = randn(g, 30, 48)
    want = R.linear(x, w, None, t)
    assert crnn.linear(x.view(30, 64), w, residual=t, out=t) is t
    R.check(t, *want)
    buf = randn(g, 40, 128)          # y and x are columns of the same buffer
    want = R.linear(buf[:, :64], w)
    crnn.linear(buf[:, :64], w, out=buf[:, 64:112])
    R.check(buf[:, 64:112], *want)


@pytest.mark.parametrize("dt", ["fp32", "bf16", "e4m3"])
@pytest.mark.parametrize("m, k, n", [(1, 80, 64), (40, 80, 64), (300, 320, 256), (700, 96, 512)])
def test_linear_nan_and_infinity_stay_in_their_row_and_column(crnn, m, k, n, dt):
    x, w, sc = linear_inputs(m, k, n, dt, 5)
    clean = crnn.linear(x, w, **sc)
    xf = x.float().clone()
    xf[0, k - 1] = float("nan")
    if m > 20 and dt != "e4m3":
        xf[17, 3] = float("inf")
    got = crnn.linear(xf.to(DT[dt]), w, **sc)
    assert torch.isnan(got[0]).all()
    if m > 20 and dt != "e4m3":
        want = torch.sign(w[:, 3].float()) * float("inf")
        assert torch.equal(got[17].float(), want)
    keep = [i for i in range(m) if i != 0 and i != 17]
    assert torch.equal(got[keep], clean[keep])
    wf = w.float().clone()
    wf[n - 1, 0] = float("nan")
    got = crnn.linear(x, wf.to(DT[dt]), **sc)
    assert torch.isnan(got[:, n - 1]).all() and torch.equal(got[:, :n - 1], clean[:, :n - 1])


@pytest.mark.parametrize("dt", ["fp32", "bf16", "e4m3"])
@pytest.mark.parametrize("act", ["none", "relu", "leaky", "gelu", "silu"])
def test_linear_activations_of_nan_and_infinity(crnn, act, dt):
    """NaN stays, infinities and what overflows nothing give the limits; through each of the kernels."""
    nan, inf = float("nan"), float("inf")
    z = torch.tensor([nan, inf, -inf, 1e30, -1e30, 200.0, -200.0, 0.0] * 8)
    neg = {"none": z, "leaky": 0.2 * z}.get(act, torch.zeros_like(z))
    want = torch.where(z < 0, neg, z)
    for m, k in ((1, 64), (3, 64), (9, 64), (40, 64), (300, 64), (700, 256), (9, 63), (300, 65)):
        x, w = torch.zeros(m, k, device="cuda").to(DT[dt]), torch.zeros(64, k, device="cuda").to(DT[dt])
        got = crnn.linear(x, w, bias=z.cuda(), act=act, out_dtype=torch.bfloat16)
        torch.testing.assert_close(got.cpu(), want.to(torch.bfloat16).expand(m, 64), rtol=2.0 ** -7, atol=0, equal_nan=True, msg=lambda t: "%d x %d: %s" % (m, k, t))


@pytest.mark.parametrize("dt", ["fp32", "bf16", "e4m3"])
@pytest.mark.parametrize("m, k, n", [(1, 4097, 33), (1, 63, 5003), (2, 515, 700), (4, 1031, 4099), (6, 3, 70), (13, 4093, 97), (100, 65, 2100), (4000, 261, 1030), (5000, 3, 2100),
                                     (2100, 1, 2050), (1500, 2047, 1500)])
def test_linear_rows_at_any_alignment(crnn, m, k, n, dt):
    """Odd lengths, and the same rows cut from wider ones at an odd place: what lies beside them (NaN) is not looked at."""
    x, w, sc = linear_inputs(m, k, n, dt, m + k)
    bias, res = randn(gen(1), n), randn(gen(2), m, n)
    for out in ("fp32", "bf16"):
        r = res.to(DT[out])
        got = crnn.linear(x, w, bias=bias, residual=r, act="silu", out_dtype=DT[out], **sc)
        R.check(got, *R.linear(x, w, bias, r, "silu", out_dtype=DT[out], **sc), what=out)
        X, W = (torch.full((t.shape[0], k + 7), float("nan"), device="cuda").to(DT[dt]) for t in (x, w))
        X[:, 3:3 + k], W[:, 3:3 + k] = x, w
        assert torch.equal(crnn.linear(X[:, 3:3 + k], W[:, 3:3 + k], bias=bias, residual=r, act="silu", out_dtype=DT[out], **sc), got)


@pytest.mark.parametrize("m, k, n", [(4600, 520, 512), (2500, 132, 1150), (8000, 4, 500), (6200, 520, 512), (2000, 76, 1700)])
def test_linear_fp32_tiles_that_share_k(crnn, m, k, n):
    x, w, _ = linear_inputs(m, k, n, "fp32", 3)
    bias, res = randn(gen(1), n), randn(gen(2), m, n)
    R.check(crnn.linear(x, w, bias=bias, residual=res, act="relu"), *R.linear(x, w, bias, res, "relu"))
    x[m - 1, 1] = float("inf")
    got = crnn.linear(x, w)
    assert torch.equal(got[m - 1], torch.sign(w[:, 1]) * float("inf"))
    R.check(got[:m - 1], *R.linear(x[:m - 1], w))


def test_linear_fp32_infinities_at_any_alignment(crnn):
    g = gen(12)
    x, w = randn(g, 700, 259), randn(g, 2060, 259)
    clean = crnn.linear(x, w)
    x[17, 3], x[650, 258] = float("inf"), -float("inf")
    got = crnn.linear(x, w)
    assert torch.equal(got[17], torch.sign(w[:, 3]) * float("inf")) and torch.equal(got[650], -torch.sign(w[:, 258]) * float("inf"))
    keep = [i for i in range(700) if i not in (17, 650)]
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("scale", [1e-30, 1e-10, 1e10, 1e18])
def test_linear_fp32_over_its_range(crnn, scale):
    g = gen(6)
    x, w = randn(g, 200, 128) * scale, randn(g, 128, 128)
    x[:, ::3] *= 1e-6                                  # values far apart in one row
    R.check(crnn.linear(x, w), *R.linear(x, w))
    R.check(crnn.linear(x[:3], w), *R.linear(x[:3], w))
    w[5] = 0
    x[7] = torch.finfo(torch.float32).max              # to the largest numbers: one product each, no overflow in between
    x[7, 1:] = 0
    w[:, 0] = 0.5
    got = crnn.linear(x, w)
    assert torch.equal(got[7], torch.full_like(got[7], torch.finfo(torch.float32).max / 2))


def test_linear_is_the_same_again(crnn):
    for m, k, n, dt in ((3, 4096, 512, "bf16"), (600, 1024, 512, "bf16"), (2500, 512, 512, "fp32"), (48, 8192, 256, "e4m3")):
        x, w, sc = linear_inputs(m, k, n, dt, 8)
        first = crnn.linear(x, w, **sc)
        for _ in range(3):
            assert torch.equal(first, crnn.linear(x, w, **sc))


# ------------------------------------------------------------------------------------------------------- rms_norm
def check_norm(crnn, x, gain, residual, eps, out_dtype, **kw):
    t, y, rel = R.rms_norm(x, gain, residual, eps)
    got = crnn.rms_norm(x, gain, residual=residual, eps=eps, out_dtype=out_dtype, **kw)
    if residual is None:
        assert got.sum is None
    else:
        R.check(got.sum, t, R.ROUND[x.dtype] * t.abs() + 2.0 ** -23 * t.abs() + R.TINY)
    if out_dtype is torch.float8_e4m3fn:
        top = y.abs().amax(-1).clamp(min=448 * 2.0 ** -126) / 448
        R.check(got.scale, top, (rel + 2.0 ** -22) * top)
        c = got.scale.double().cpu()[..., None]
        # 2 more roundings before the one to 8 bits: the scale's reciprocal and the product with it
        err = (1.01 * rel + 2.0 ** -22) * y.abs() + torch.maximum(2.0 ** -4 * 1.001 * y.abs(), 2.0 ** -10 * c)
        R.check(got.y.double().cpu() * c, y, err)
    else:
        assert got.scale is None and got.y.dtype is x.dtype
        R.check(got.y, y, 1.01 * rel * y.abs() + R.ROUND[x.dtype] * y.abs() + R.TINY)
    return got


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("m, n", [(1, 1), (1, 512), (3, 7), (8, 512), (5, 513), (33, 64), (70, 768), (9, 1000), (17, 2048), (130, 4096), (4, 5530), (3, 8192), (2, 16384),
                                  (2, 20001), (4000, 256)])
def test_rms_norm(crnn, m, n, dt):
    g = gen(m + n)
    x = randn(g, m, n, dt=dt)
    res, gain = randn(g, m, n, dt=dt), randn(g, n)
    for r in (None, res):
        for out in (None, torch.float8_e4m3fn):
            check_norm(crnn, x, gain, r, 1e-6, out)


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("m, n", [(3, 2), (9, 9), (300, 511), (2100, 1023), (41, 2047), (20, 4095), (9, 8191), (5, 8193)])
def test_rms_norm_rows_at_any_alignment(crnn, m, n, dt):
    g = gen(n)
    X, Y = (torch.full((m, n + 5), float("nan"), device="cuda").to(DT[dt]) for _ in range(2))
    X[:, 1:1 + n], Y[:, 3:3 + n] = randn(g, m, n, dt=dt), randn(g, m, n, dt=dt)
    x, r, gain = X[:, 1:1 + n], Y[:, 3:3 + n], 1 + 0.1 * randn(g, n)
    for out in (DT[dt], DT["e4m3"]):
        got = check_norm(crnn, x, gain, r, 1e-6, out)
        whole = crnn.rms_norm(x.contiguous(), gain, residual=r.contiguous(), out_dtype=out)
        bits = lambda t: t.view(torch.uint8) if t.dtype is DT["e4m3"] else t
        again = crnn.rms_norm(x, gain, residual=r, out_dtype=out)
        assert torch.equal(bits(again.y), bits(whole.y)) and torch.equal(again.sum, whole.sum)


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("n", [64, 512, 1024, 3000, 9000])
def test_rms_norm_strides_in_place_and_broadcast(crnn, n, dt):
    g = gen(n)
    gain = randn(g, n + 1)
    for lead, pitch in ((0, n + 64), (1, n + 3), (8, n + 8)):
        X, Rs = randn(g, 6, lead + pitch, dt=dt), randn(g, 6, lead + pitch, dt=dt)
        x, r = X[:, lead:lead + n], Rs[:, lead:lead + n]
        for out in (None, torch.float8_e4m3fn):
            Y = torch.zeros(6, lead + pitch, dtype=out or DT[dt], device="cuda")
            check_norm(crnn, x, gain[1:], r, 1e-5, out, out=Y[:, lead:lead + n])
            assert (Y.float()[:, :lead] == 0).all() and (Y.float()[:, lead + n:] == 0).all()
        x2, r2 = x.clone(), r.clone()       # (another layout may add its squares in another order)
        want = crnn.rms_norm(x2, gain[:n], residual=r2)
        got = crnn.rms_norm(x2, gain[:n], residual=r2, out=x2, sum_out=r2)
        assert got.y is x2 and torch.equal(x2, want.y) and torch.equal(r2, want.sum)
        row = x[:1].expand(6, n)
        check_norm(crnn, row, gain[:n], r, 1e-6, None)
    x3 = randn(g, 2, 3, n, dt=dt)
    assert torch.equal(crnn.rms_norm(x3[:, 1], gain[:n]).y, crnn.rms_norm(x3, gain[:n]).y[:, 1])
    assert crnn.rms_norm(x3, gain[:n], out_dtype=torch.float8_e4m3fn).scale.shape == (2, 3)
    assert crnn.rms_norm(x3[:0], gain[:n]).y.shape == (0, 3, n)


@pytest.mark.parametrize("n", [8, 512, 1024, 4097, 9000])
def test_rms_norm_zeros_extremes_and_nan(crnn, n):
    g = gen(3)
    gain = torch.ones(n, device="cuda")
    for dt in ("fp32", "bf16"):
        x = randn(g, 7, n, dt=dt)
        x[1] = 0
        x[2, n // 2] = float("nan")
        x[3, 0] = float("inf")
        x[4] = x[4] * 1e-25
        got, clean = crnn.rms_norm(x, gain), crnn.rms_norm(x[[0, 5, 6]], gain)
        assert (got.y[1] == 0).all() and torch.isnan(got.y[2]).all() and torch.equal(got.y[[0, 5, 6]], clean.y)
        assert torch.isnan(got.y[3, 0]) and (got.y[3, 1:] == 0).all()
        got, clean = (crnn.rms_norm(t, gain, out_dtype=torch.float8_e4m3fn) for t in (x, x[[0, 5, 6]]))
        y8 = got.y.float()
        assert (y8[1] == 0).all() and float(got.scale[1]) > 0 and torch.isnan(got.scale[2]) and torch.isnan(y8[2]).all() and torch.isnan(got.scale[3])
        assert torch.equal(y8[[0, 5, 6]], clean.y.float()) and torch.equal(got.scale[[0, 5, 6]], clean.scale)
        top = y8[[0, 5, 6]].abs().amax(1)
        assert (top == 448).all()
    check_norm(crnn, randn(g, 3, n) * 1e-22, gain, None, 0.0, None)      # no eps: squares near the smallest normal numbers


# ------------------------------------------------------------------------------------------------------- cross_attention
def qkv(g, b, t, s, heads, kvh, d, dt, spread=1.5):
    q = (randn(g, b, t, heads, d) * spread).to(DT[dt])
    kv = randn(g, b, s, 2, kvh, d, dt=dt)
    return q, kv[:, :, 0], kv[:, :, 1]


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("b, t, s, heads, kvh, d", [
    (1, 1, 1, 1, 1, 1), (2, 1, 71, 8, 8, 64), (3, 5, 33, 4, 2, 32), (2, 17, 64, 2, 1, 128), (1, 130, 257, 2, 2, 64), (2, 3, 1000, 4, 4, 64), (1, 1, 5000, 8, 2, 128),
    (2, 33, 129, 3, 3, 80), (1, 7, 31, 6, 2, 17), (4, 64, 32, 1, 1, 96), (1, 1, 20000, 2, 1, 64), (1, 300, 300, 4, 1, 128), (5, 2, 2, 2, 2, 8), (2, 16, 4096, 1, 1, 40),
    (1, 257, 65, 1, 1, 33), (3, 40, 700, 16, 1, 64), (32, 258, 400, 8, 4, 64), (16, 300, 330, 16, 8, 128), (40, 64, 300, 8, 2, 32),
    (33, 270, 260, 8, 8, 80)])
def test_cross_attention(crnn, b, t, s, heads, kvh, d, dt):
    g = gen(b + t + s)
    q, k, v = qkv(g, b, t, s, heads, kvh, d, dt)
    lengths = torch.randint(0, s + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
    mask = torch.rand(b, s, generator=g, device="cuda") < 0.7
    for L, M in ((None, None), (lengths, None), (None, mask), (lengths, mask)):
        got = crnn.cross_attention(q, k, v, lengths=L, mask=M)
        assert got.dtype is q.dtype and got.shape == q.shape
        R.check(got, *R.attention(q, k, v, L, M))


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("t, s, d", [(1, 71, 64), (1, 3000, 64), (40, 200, 64), (200, 200, 128), (1, 90, 48), (30, 513, 24)])
def test_cross_attention_never_looks_at_left_out_keys(crnn, t, s, d, dt):
    """Infinities and NaN in the keys and values that lengths and mask leave out, rows with no key at all, lengths out of range."""
    g = gen(t + s)
    b, h = 6, 2
    q, k, v = qkv(g, b, t, s, h, h, d, dt)
    lengths = torch.tensor([0, 1, s // 2, s, s + 100, -3], dtype=torch.int32, device="cuda")
    mask = torch.rand(b, s, generator=g, device="cuda") < 0.5
    mask[2] = False
    mask[1, 0] = True
    mask[3, : s - 1] = False
    mask[3, s - 1] = True
    want = crnn.cross_attention(q, k, v, lengths=lengths, mask=mask)
    R.check(want, *R.attention(q, k, v, lengths, mask))
    out = ~mask | (torch.arange(s, device="cuda") >= lengths[:, None])
    for poison in (float("nan"), float("inf"), -float("inf"), torch.finfo(DT[dt]).min):
        k2, v2 = k.clone(), v.clone()
        k2[out], v2[out] = poison, poison
        assert torch.equal(crnn.cross_attention(q, k2, v2, lengths=lengths, mask=mask), want)
        only_mask = crnn.cross_attention(q, k2, v2, mask=mask & ~out)
        assert torch.equal(only_mask[2], torch.zeros_like(only_mask[2]))
        R.check(only_mask, *R.attention(q, k, v, None, mask & ~out))
    for i in (0, 2, 5):
        assert (want[i] == 0).all()
    assert torch.equal(want[3], v[3, s - 1].expand(t, h, d))      # one key: its value
    assert torch.equal(crnn.cross_attention(q, k, v, lengths=lengths, mask=mask.to(torch.uint8) * 255), want)


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_cross_attention_without_keys(crnn, dt):
    q = randn(gen(1), 2, 3, 4, 64, dt=dt)
    k = randn(gen(2), 2, 0, 4, 64, dt=dt)
    assert torch.equal(crnn.cross_attention(q, k, k), torch.zeros_like(q))
    assert crnn.cross_attention(q[:0], k[:0], k[:0]).shape == (0, 3, 4, 64) and crnn.cross_attention(q[:, :0], k, k).shape == (2, 0, 4, 64)


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("t, s", [(1, 71), (1, 2500), (50, 130), (200, 600)])
def test_cross_attention_strides_and_alignments(crnn, t, s, dt):
    g = gen(t * s)
    b, h, d = 2, 3, 64
    Q, K, V = randn(g, b, h, t, d, dt=dt), randn(g, s, b, h, d + 3, dt=dt), randn(g, b, s, h * d + 1, dt=dt)
    q, k, v = Q.permute(0, 2, 1, 3), K.permute(1, 0, 2, 3)[..., 1:1 + d], V[..., 1:].unflatten(2, (h, d))
    Y = torch.full((b, t, h, d + 8), 7.0, dtype=DT[dt], device="cuda")
    got = crnn.cross_attention(q, k, v, out=Y[..., 4:4 + d])
    R.check(got, *R.attention(q, k, v))
    assert (Y[..., :4] == 7).all() and (Y[..., 4 + d:] == 7).all()
    one = randn(g, 1, s, 1, d, dt=dt)          # every entry and head reads the same keys
    q2 = q.contiguous()
    R.check(crnn.cross_attention(q2, one.expand(b, s, h, d), one.expand(b, s, h, d)), *R.attention(q2, one.expand(b, s, h, d), one.expand(b, s, h, d)))
    for sc in (0.0, -0.2, 3.0):
        R.check(crnn.cross_attention(q2, k, v, scale=sc), *R.attention(q2, k, v, scale=sc))


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("b, t, s, d", [(130, 1, 71, 64), (260, 3, 40, 24), (70, 48, 71, 64), (70, 33, 100, 32), (80, 20, 71, 64)])
def test_cross_attention_many_lines(crnn, b, t, s, d, dt):
    """More key heads than workgroups that fill the chip: fewer waves share the keys of one."""
    g = gen(b + t)
    q, k, v = qkv(g, b, t, s, 8, 8, d, dt)
    lengths = torch.randint(0, s + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
    got = crnn.cross_attention(q, k, v, lengths=lengths)
    some = [0, 1, b // 2, b - 1]
    R.check(got[some], *R.attention(q[some], k[some], v[some], lengths[some]))
    at = torch.arange(s, device="cuda") < lengths[:, None]
    assert torch.equal(crnn.cross_attention(q, k, v, mask=at), got)          # the same keys, said another way
    for i in range(0, b, 16):                                               # alone (other splits of the keys): the same within the bound
        R.check(crnn.cross_attention(q[i:i + 1], k[i:i + 1], v[i:i + 1], lengths=lengths[i:i + 1]), *R.attention(q[i:i + 1], k[i:i + 1], v[i:i + 1], lengths[i:i + 1]))


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("d", [16, 64, 72, 128])
@pytest.mark.parametrize("t, heads, kvh", [(1, 2, 2), (2, 2, 2), (1, 2, 1), (3, 2, 2), (1, 6, 2), (4, 1, 1), (2, 2, 1), (5, 2, 2)])
def test_cross_attention_one_to_five_rows_a_key_head(crnn, t, heads, kvh, d, dt):
    for b, s in ((3, 50), (2, 700), (3, 1)):
        g = gen(b + t + s)
        q, k, v = qkv(g, b, t, s, heads, kvh, d, dt)
        lengths = torch.tensor([s, s // 2, 1][:b], dtype=torch.int32, device="cuda")
        R.check(crnn.cross_attention(q, k, v, lengths=lengths), *R.attention(q, k, v, lengths))


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("b, t, s, heads, kvh, d", [(2, 300, 1500, 4, 2, 64), (1, 700, 2000, 3, 1, 128), (3, 130, 900, 4, 4, 40), (2, 520, 1100, 2, 2, 32), (1, 256, 3000, 4, 1, 8)])
def test_cross_attention_many_rows_over_splits(crnn, b, t, s, heads, kvh, d, dt):
    """Rows that several workgroups share, each part of the keys, more of them than are joined one by one; some without a key."""
    g = gen(b + t)
    q, k, v = qkv(g, b, t, s, heads, kvh, d, dt)
    lengths = torch.tensor([s, 0, s // 3][:b], dtype=torch.int32, device="cuda")
    mask = torch.rand(b, s, generator=g, device="cuda") < 0.7
    mask[0, : s // 2] = False                                     # whole splits without a key
    got = crnn.cross_attention(q, k, v, lengths=lengths, mask=mask)
    R.check(got, *R.attention(q, k, v, lengths, mask))
    if b > 1:
        assert (got[1] == 0).all()
    buf = torch.full((b, t, heads, d + 3), 7.0, dtype=q.dtype, device="cuda")     # results at any place
    out = buf[..., 1:1 + d]
    assert crnn.cross_attention(q, k, v, lengths=lengths, mask=mask, out=out) is out
    assert torch.equal(out, got) and (buf[..., 0] == 7).all() and (buf[..., 1 + d:] == 7).all()


@pytest.mark.parametrize("t, s", [(1, 1), (1, 300), (20, 1), (40, 300)])
def test_cross_attention_strides_of_single_dimensions_do_not_matter(crnn, t, s):
    g = gen(t + s)
    q, k, v = randn(g, 1, t, 1, 64), randn(g, 1, s, 1, 64), randn(g, 1, s, 1, 64)
    odd = lambda x: x.as_strided(x.shape, [3 if x.shape[i] == 1 else x.stride(i) for i in range(3)] + [1])
    want = crnn.cross_attention(q, k, v)
    R.check(want, *R.attention(q, k, v))
    assert torch.equal(crnn.cross_attention(odd(q), odd(k), odd(v)), want)


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("t, s", [(1, 40), (1, 4000), (64, 500)])
def test_cross_attention_scores_far_apart(crnn, t, s, dt):
    """Scores of several hundred: the running maximum, not the first tile's, decides; a maximum at the end, in the middle."""
    g = gen(9)
    q, k, v = qkv(g, 2, t, s, 2, 2, 64, dt, spread=12)
    k = k.clone()
    k[0, s - 1] *= 4
    k[1, s // 2] *= 4
    R.check(crnn.cross_attention(q, k, v), *R.attention(q, k, v))
    R.check(crnn.cross_attention(q, k, v, scale=-0.5), *R.attention(q, k, v, scale=-0.5))


def test_cross_attention_offsets_beyond_32_bits(crnn):
    free = torch.cuda.mem_get_info()[0]
    if free < 40 << 30:
        pytest.skip("needs 40 GB of device memory")
    g = gen(11)
    # positions far apart: 3000 keys, 2^20 elements from one to the next
    big = torch.empty(3000 << 20, dtype=torch.bfloat16, device="cuda")
    k = torch.as_strided(big, (1, 3000, 2, 64), (1 << 20, 1 << 20, 64, 1), 0)
    v = torch.as_strided(big, (1, 3000, 2, 64), (1 << 20, 1 << 20, 64, 1), 128)
    k.copy_(randn(g, 1, 3000, 2, 64))
    v.copy_(randn(g, 1, 3000, 2, 64))
    for t in (1, 70):
        q = randn(g, 1, t, 2, 64, dt="bf16")
        R.check(crnn.cross_attention(q, k, v), *R.attention(q, k, v))
        # entries far apart
        k3, v3 = (torch.as_strided(big, (3, 40, 1, 64), (1 << 30, 1 << 20, 64, 1), at) for at in (0, 128))
        k3.copy_(randn(g, 3, 40, 1, 64))
        v3.copy_(randn(g, 3, 40, 1, 64))
        q = randn(g, 3, t, 1, 64, dt="bf16")
        R.check(crnn.cross_attention(q, k3, v3), *R.attention(q, k3, v3))
        k.copy_(randn(g, 1, 3000, 2, 64))
        v.copy_(randn(g, 1, 3000, 2, 64))
    # rows of a matrix likewise
    x, w = torch.as_strided(big, (70, 64), (40 << 20, 1), 0), randn(g, 48, 64, dt="bf16")
    x.copy_(randn(g, 70, 64))
    R.check(crnn.linear(x, w), *R.linear(x, w, out_dtype=torch.bfloat16))
    R.check(crnn.linear(w, x), *R.linear(w, x, out_dtype=torch.bfloat16))
    check_norm(crnn, x, randn(g, 64), None, 1e-6, torch.float8_e4m3fn)


# ------------------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("k", [4096, 4095])
def test_rows_beyond_32_bits(crnn, k):
    """More than 2^31 values in x: aligned rows and rows at any place, linear and rms_norm, at both ends."""
    g, m, n = gen(5), 530000, 40
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
    ends = [0, 1, 2, m // 2, m - 3, m - 2, m - 1]
    x[ends] = randn(g, len(ends), k, dt="bf16")
    w, bias, gain = randn(g, n, k, dt="bf16"), randn(g, n), 1 + 0.1 * randn(g, k)
    y = crnn.linear(x, w, bias=bias)
    R.check(y[ends], *R.linear(x[ends], w, bias, out_dtype=torch.bfloat16))
    R.check(y[5:9], *R.linear(x[5:9], w, bias, out_dtype=torch.bfloat16))
    want = x[ends]
    norm = crnn.rms_norm(x, gain, out=x)
    assert norm.y is x
    t, y, rel = R.rms_norm(want, gain)
    R.check(x[ends], y, 1.01 * rel * y.abs() + R.ROUND[torch.bfloat16] * y.abs() + R.TINY)
    assert (x[5:9] == 0).all()
    del x, norm
    wide = torch.zeros(40, 1 << 26, dtype=torch.bfloat16, device="cuda")         # few rows, far apart
    a, out = wide[:, 3:3 + k], wide[:, 1 << 25:(1 << 25) + n]
    a.copy_(randn(g, 40, k, dt="bf16"))
    crnn.linear(a, w, bias=bias, out=out)
    R.check(out, *R.linear(a, w, bias, out_dtype=torch.bfloat16))
    assert (wide[:, (1 << 25) + n:(1 << 25) + 100] == 0).all() and (wide[:, (1 << 25) - 9:1 << 25] == 0).all()


@pytest.mark.parametrize("what", ["linear", "rms_norm", "attention"])
def test_operators_captured_beside_eager_calls(crnn, what):
    """Two graphs of one operator, replayed in turn with other eager calls of it between: each has its own outputs and workspace."""
    g = gen(9)
    if what == "linear":
        make = lambda: (randn(g, 70, 515, dt="bf16"), randn(g, 600, 515, dt="bf16"))
        call = lambda a: crnn.linear(a[0], a[1], act="gelu")
    elif what == "rms_norm":
        make = lambda: (randn(g, 70, 515, dt="bf16"), 1 + randn(g, 515))
        call = lambda a: crnn.rms_norm(a[0], a[1], residual=a[0], out_dtype=torch.float8_e4m3fn).scale
    else:
        make = lambda: tuple(randn(g, *t, dt="bf16") for t in ((2, 1, 8, 64), (2, 4000, 8, 64), (2, 4000, 8, 64)))      # splits: a workspace
        call = lambda a: crnn.cross_attention(*a)
    sets = [make() for _ in range(3)]
    want = [call(a).clone() for a in sets]
    graphs = []
    for a in sets[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(a)
        graphs.append((graph, out))
    for _ in range(4):
        for (graph, out), w in zip(graphs, want):
            out.zero_()
            graph.replay()
            eager = call(sets[2])
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, w) and torch.equal(eager, want[2])


def layer_weights(g, dim, heads, d, kvh, dt, q8=False):
    w = {"norm.weight": 1 + 0.1 * randn(g, dim), "q.weight": randn(g, heads * d, dim) / dim ** 0.5, "kv.weight": randn(g, 2 * kvh * d, 512) * 0.2,
         "out.weight": randn(g, dim, heads * d) / (heads * d) ** 0.5, "q.bias": randn(g, heads * d) * 0.1, "out.bias": randn(g, dim) * 0.1}
    for name in ("q.weight", "kv.weight", "out.weight"):
        w[name] = w[name].to(DT[dt])
    if q8:
        top = w["q.weight"].float().abs().amax(1) / 448
        w["q.weight"], w["q.scale"] = (w["q.weight"].float() / top[:, None]).to(torch.float8_e4m3fn), top
    return w


@pytest.fixture(scope="module")
def reader(synth_en):
    from ocr_amd.crnn import keys
    from ocr_amd.crnn.network_hip import CRNN
    m = CRNN(32, 1, 65, 256, alphabet=keys.alphabetEnglish, device=0)
    m.load_state_dict(synth_en)
    return m


def test_line_states_are_what_the_classifier_reads(reader, synth_en):
    rs = np.random.RandomState(5)
    lines = rs.randint(0, 256, size=(5, 32, 200)).astype(np.uint8)
    widths = [200, 8, 131, 64, 200]
    for i, w in enumerate(widths):
        lines[i, :, w:] = 0
    d = torch.from_numpy(lines).cuda()
    states, lengths = reader.line_states(d, widths)
    assert states.shape == (5, 51, 512) and lengths.tolist() == [w // 4 + 1 for w in widths]
    x = ((lines / 255.0 - 0.5) / 0.5).astype(np.float32)
    for i, w in enumerate(widths):
        x[i, :, w:] = 0
    want = reader.debug_stage(x, 9, widths)
    for i, n in enumerate(lengths.tolist()):
        # the two paths may take different forms of the recurrence; their states are the same bit for bit
        assert np.array_equal(states[i, :n].cpu().numpy(), want[i, :n]) and (states[i, n:] == 0).all()
    W, b = (torch.from_numpy(np.asarray(synth_en["rnn.1.embedding." + n])).cuda() for n in ("weight", "bias"))
    logits = reader.linear(states, W, bias=b)
    full = reader.debug_stage(x, 10, widths)
    for i, n in enumerate(lengths.tolist()):
        assert np.abs(logits[i, :n].cpu().numpy() - full[i, :n]).max() < 1e-3     # the same classifier, in fp32 both times
    assert torch.equal(reader.line_states(d)[0][0], states[0]) and reader.line_states(d)[1].tolist() == [51] * 5
    # ordered against the current stream: the lines are written on it just before, and read by the next kernel just after
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        late = torch.zeros_like(d)
        torch.cuda._sleep(20_000_000)
        late.copy_(d)
        got = reader.line_states(late, widths)[0] + 0
    s.synchronize()
    assert torch.equal(got, states)


@pytest.mark.parametrize("dt, q8", [("fp32", False), ("bf16", False), ("bf16", True)])
def test_line_attention_over_a_batch_of_lines(reader, dt, q8):
    """norm -> q -> attention over the recogniser's states -> out + residual, against the same in 64 bits step by step."""
    from ocr_amd.crnn.attention import LineAttention
    g = gen(20)
    heads, d, kvh, dim = 8, 32, 4, 320
    w = layer_weights(g, dim, heads, d, kvh, dt, q8)
    layer = LineAttention(reader, w, heads, kvh)
    rs = np.random.RandomState(6)
    lines = torch.from_numpy(rs.randint(0, 256, size=(6, 32, 160)).astype(np.uint8)).cuda()
    widths = [160, 40, 99, 8, 160, 64]
    states, lengths = reader.line_states(lines, widths)
    memory, page = layer.memory(states, lengths), layer.page_memory(states, lengths)
    kv, err = R.linear(states.to(DT[dt]), w["kv.weight"], out_dtype=DT[dt])
    R.check(torch.stack((memory.k, memory.v), 2), kv.view(6, 41, 2, kvh, d), err.view(6, 41, 2, kvh, d))
    assert page.k.shape == (1, 6 * 41, kvh, d) and int(page.mask.sum()) == int(lengths.sum())
    for mem, n, t in ((memory, 6, 1), (memory, 6, 9), (page, 1, 1), (page, 1, 12)):
        x, r = randn(g, n, t, dim, dt=dt), randn(g, n, t, dim, dt=dt)
        got = layer(x, mem, residual=r)
        # each step from what the step before left, so that each is held to its own bound
        y, scale, total = reader.rms_norm(x, w["norm.weight"], residual=r, out_dtype=torch.float8_e4m3fn if q8 else None)
        want, err = R.linear(y, w["q.weight"], w["q.bias"], out_dtype=DT[dt], x_scale=scale, w_scale=w.get("q.scale"))
        q = reader.linear(y, w["q.weight"], bias=w["q.bias"], x_scale=scale, w_scale=w.get("q.scale")).view(n, t, heads, d)
        R.check(q, want.view(q.shape), err.view(q.shape))
        a = reader.cross_attention(q, mem.k, mem.v, mem.lengths, mem.mask)
        R.check(a, *R.attention(q, mem.k, mem.v, mem.lengths, mem.mask))
        want, err = R.linear(a.view(n * t, -1), w["out.weight"], w["out.bias"], total.view(n * t, -1), out_dtype=DT[dt])
        R.check(got.view(n * t, -1), want, err)
        assert torch.equal(layer(x, mem), layer(x + 0, mem))


def test_line_attention_captured_and_replayed(reader):
    """A decoding step and a page query in two graphs, replayed in turn with eager work between; long memories split over
    workgroups use a workspace of each graph's own."""
    from ocr_amd.crnn.attention import LineAttention
    g = gen(21)
    w = layer_weights(g, 256, 4, 64, 4, "bf16")
    layer = LineAttention(reader, w, 4)
    states = torch.tanh(randn(g, 300, 71, 512))
    lengths = torch.randint(0, 72, (300,), generator=g, device="cuda", dtype=torch.int32)
    lines, page = layer.memory(states, lengths), layer.page_memory(states, lengths)
    xs = [randn(g, n, 1, 256, dt="bf16") for n in (300, 1)]
    reader.stream_ptr(0)
    graphs, outs = [], []
    for x, mem in zip(xs, (lines, page)):
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            layer(x, mem)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(x, mem)
        graphs.append(graph)
        outs.append(out)
    for turn in range(4):
        for x in xs:
            x.copy_(randn(g, *x.shape))
        for i in (0, 1, 1, 0) if turn % 2 else (1, 0):
            graphs[i].replay()
        busy = layer(xs[0] + 1, lines)
        torch.cuda.synchronize()
        for x, mem, out in zip(xs, (lines, page), outs):
            assert torch.equal(out, layer(x, mem)) and float(out.float().abs().max()) > 0
        assert torch.isfinite(busy.float()).all()


def test_operators_on_another_stream_and_from_two_threads(crnn):
    g = gen(22)
    x, w = randn(g, 600, 512, dt="bf16"), randn(g, 512, 512, dt="bf16")
    q, k, v = qkv(g, 1, 1, 9000, 4, 4, 64, "bf16")
    gain = randn(g, 512)
    want = (crnn.linear(x, w), crnn.rms_norm(x, gain, out_dtype=torch.float8_e4m3fn).y.float(), crnn.cross_attention(q, k, v))
    torch.cuda.synchronize()
    bad = []

    def work():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(40):
                got = (crnn.linear(x, w), crnn.rms_norm(x, gain, out_dtype=torch.float8_e4m3fn).y.float(), crnn.cross_attention(q, k, v))
                s.synchronize()
                bad.extend(i for i in range(3) if not torch.equal(got[i], want[i]))
    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_refusals_with_tensors(crnn):
    g = gen(23)
    x, w = randn(g, 4, 64), randn(g, 8, 64)
    q = randn(g, 2, 3, 4, 32)
    for call in (lambda: crnn.linear(x, w.bfloat16()), lambda: crnn.linear(x, w[:, :60]), lambda: crnn.linear(x.half(), w.half()), lambda: crnn.linear(x, w, act="tanh"),
                 lambda: crnn.linear(x, w, bias=randn(g, 9)), lambda: crnn.linear(x, w, bias=randn(g, 8).bfloat16()), lambda: crnn.linear(x, w, residual=randn(g, 4, 9)),
                 lambda: crnn.linear(x, w, out_dtype=torch.float16), lambda: crnn.linear(x, w, x_scale=randn(g, 4)), lambda: crnn.linear(x.t(), w),
                 lambda: crnn.linear(x, w, out=x[:, :8]), lambda: crnn.linear(x, w.requires_grad_()), lambda: crnn.rms_norm(x, randn(g, 63)),
                 lambda: crnn.rms_norm(x, randn(g, 64), out_dtype=torch.bfloat16), lambda: crnn.rms_norm(x, randn(g, 64), eps=-1.0),
                 lambda: crnn.rms_norm(x, randn(g, 64), sum_out=x), lambda: crnn.rms_norm(x, randn(g, 64), residual=x[:, :63]),
                 lambda: crnn.cross_attention(q, q.bfloat16(), q.bfloat16()), lambda: crnn.cross_attention(q, q[:, :, :3], q[:, :, :3]),
                 lambda: crnn.cross_attention(q, q, q[:, :2]), lambda: crnn.cross_attention(q, q, q, lengths=torch.zeros(2, device="cuda")),
                 lambda: crnn.cross_attention(q, q, q, mask=torch.ones(2, 4, device="cuda", dtype=torch.bool)), lambda: crnn.cross_attention(q, q, q, out=q),
                 lambda: crnn.cross_attention(randn(g, 1, 1, 1, 129), randn(g, 1, 1, 1, 129), randn(g, 1, 1, 1, 129)),
                 lambda: crnn.line_states(torch.zeros(2, 31, 64, dtype=torch.uint8, device="cuda"))):
        with pytest.raises(ValueError):
            call()
    from ocr_amd.crnn import _capi
    with pytest.raises(_capi.CrnnError):      # no weights loaded
        crnn.line_states(torch.zeros(2, 32, 64, dtype=torch.uint8, device="cuda"))
    with torch.no_grad():
        assert crnn.linear(x, w).shape == (4, 8)
