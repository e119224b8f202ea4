"""Plain 64-bit forms of the sequence operators, each with the error its 32-bit form may have: (value, bound).

A float32 operation is off by at most 2^-24 of its result; matrix instructions may add their products in any order and cut
instead of rounding, so 2^-23 is counted for each addition.  A rounding to bfloat16 is off by 2^-8 of the value, one to
e4m3 by 2^-4 of the value or half its smallest step, 2^-10.

The 8-bit matrix instructions align the products of a group (at most 8 neighbours) to the largest one's exponent and keep 13
bits below it: each product loses less than 2^-13 of the largest in its group.  They serve bfloat16 results; float32 ones
are summed exactly in bfloat16."""
import math

import torch

ROUND = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
TINY = 1e-37          # results below the normal numbers


def act64(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "leaky":
        return torch.where(z > 0, z, 0.2 * z)
    if act == "gelu":
        return 0.5 * z * torch.erfc(-z / math.sqrt(2.0))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def linear(x, w, bias=None, residual=None, act="none", x_scale=None, w_scale=None, out_dtype=torch.float32):
    k = w.shape[1]
    xd, wd = x.double().cpu().reshape(-1, k), w.double().cpu()
    if x_scale is not None:
        xd = xd * x_scale.double().cpu().reshape(-1, 1)
    if w_scale is not None:
        wd = wd * w_scale.double().cpu()[:, None]
    z, size = xd @ wd.t(), xd.abs() @ wd.abs().t()
    if bias is not None:
        z, size = z + bias.double().cpu(), size + bias.double().cpu().abs()
    y = act64(z, act)
    # k products and additions, the scales and the bias; the slope of gelu is at most 1.13, of silu 1.1; the activation itself
    # is good to 2^-21 of max(|z|, 1) (erf to 2^-22 absolutely)
    err = 1.2 * (k + 8) * 2.0 ** -23 * size
    if x.dtype is torch.float8_e4m3fn and out_dtype is torch.bfloat16:
        # |x w| of a group is at most (max |x|)(max |w|) in it
        pad = (-k) % 8
        xg, wg = (torch.nn.functional.pad(t.abs(), (0, pad)).view(t.shape[0], -1, 8).amax(2) for t in (xd, wd))
        err = err + 1.2 * 8 * 2.0 ** -13 * (xg @ wg.t())
    if act in ("gelu", "silu"):
        err = err + 2.0 ** -21 * z.abs()
    if residual is not None:
        r = residual.double().cpu().reshape(y.shape)
        y = y + r
        err = err + 2.0 ** -23 * (y.abs() + r.abs())
    err = err * 1.01 + ROUND[out_dtype] * y.abs() + TINY
    return y, err


def rms_norm(x, gain, residual=None, eps=1e-6):
    """(t, y, relative error of y in 32 bits)."""
    t = x.double().cpu()
    if residual is not None:
        t = t + residual.double().cpu()
    n = t.shape[-1]
    y = t / (t.square().mean(-1, keepdim=True) + eps).sqrt() * gain.double().cpu()
    # each square is off by 3 roundings of 2^-24 (the sum's rounding counts twice), the sum of n by n more, half of that in
    # the root, which with the division, the products and t itself adds 6
    return t, y, (0.5 * (n + 3) + 8) * 2.0 ** -24


def attention(q, k, v, lengths=None, mask=None, scale=None):
    dt = q.dtype
    b, t, heads, d = q.shape
    s, kvh = k.shape[1], k.shape[2]
    scale = d ** -0.5 if scale is None else scale
    out, err = torch.zeros(b, t, heads, d, dtype=torch.float64), torch.zeros(b, t, heads, d, dtype=torch.float64)
    for i in range(b):
        n = s if lengths is None else max(0, min(s, int(lengths[i])))
        at = torch.arange(n)
        if mask is not None:
            at = at[mask[i].cpu()[:n].bool()]
        if len(at) == 0:
            continue
        for h in range(heads):
            g = h // (heads // kvh)
            qi = q[i, :, h].double().cpu()
            ki, vi = k[i, :, g][at.to(k.device)].double().cpu(), v[i, :, g][at.to(v.device)].double().cpu()
            z = qi @ ki.t() * scale
            p = torch.softmax(z, 1)
            out[i, :, h] = p @ vi
            # a score: d products and additions, the scale, and its difference from the maximum (|z| each) -> the same
            # absolute error in the exponent, for p and, as a mean, for their sum; 4 for the exponential and the running scale
            dz = (d + 4) * 2.0 ** -23 * (qi.abs() @ ki.abs().t() * abs(scale)) + 2.0 ** -22 * (z.abs() + z.abs().amax(1, keepdim=True))
            rel = dz + (p * dz).sum(1, keepdim=True) + (2 * len(at) + 16) * 2.0 ** -23
            if dt is torch.bfloat16:
                rel = rel + 2.0 ** -8           # p in bfloat16 for the second product
            err[i, :, h] = (p * rel) @ vi.abs()
    return out, 1.01 * err + ROUND[dt] * out.abs() + TINY


def check(got, want, err, what=""):
    got = got.double().cpu().reshape(want.shape)
    assert torch.isfinite(got).all(), what
    over = (got - want).abs() - err
    assert over.max() <= 0, "%s: off by %.3g where %.3g is allowed" % (what, float((got - want).abs().flatten()[over.argmax()]), float(err.flatten()[over.argmax()]))
