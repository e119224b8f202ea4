"""Numbers of the sequence operators, each held to a bound derived for the one thing that it looks at."""
import numpy as np
import pytest
import torch

from tests import seq_reference as R
from tests.test_hip_seq_ops import DT, gen, randn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def crnn():
    from ocr_amd.crnn.network_hip import CRNN
    return CRNN(32, 1, 65, 256, device=0)


@pytest.mark.parametrize("n", [512, 1000, 4096, 9000])
def test_rms_norm_8_bit_values_are_the_quotient(crnn, n):
    """y / scale rounded to e4m3, not y times the scale's inverse: quotients at and beside the middle between two e4m3 values."""
    x = torch.ones(2, n, device="cuda")                                   # eps 0: y is the gain itself
    x[1] = -4
    for c in range(1, 512, 8):
        c |= 1 if c < 256 else 7
        mid = torch.arange(17, 32, 2, dtype=torch.float64) / 16
        y = torch.cat([mid * 2.0 ** e for e in range(-7, 8)]) * (c / 64.0)
        gain = torch.cat([y.float(), torch.nextafter(y.float(), torch.full_like(y, 1e9).float()), torch.nextafter(y.float(), torch.zeros_like(y).float())])
        gain = gain.repeat(n // gain.numel() + 1)[:n]
        gain[n - 2], gain[n - 1] = -0.0, 448 * (c / 64.0)
        got = crnn.rms_norm(x, gain.cuda(), eps=0.0, out_dtype=DT["e4m3"])
        assert (got.scale == c / 64.0).all()
        want = (gain / np.float32(c / 64.0)).to(DT["e4m3"]).view(torch.uint8)       # (IEEE division, on the host)
        assert torch.equal(got.y[0].view(torch.uint8).cpu(), want) and torch.equal(got.y[1].view(torch.uint8).cpu(), want ^ 0x80), c


def test_rms_norm_8_bit_values_are_the_quotient_of_random_rows(crnn):
    g = gen(31)
    for m, n in ((6000, 2048), (900, 5000), (100, 20000)):
        x, gain = randn(g, m, n), randn(g, n)
        y, got = crnn.rms_norm(x, gain).y, crnn.rms_norm(x, gain, out_dtype=DT["e4m3"])
        assert torch.equal(got.scale.cpu(), y.abs().amax(1).cpu() / 448)
        assert torch.equal(got.y.view(torch.uint8).cpu(), (y.cpu() / got.scale.cpu()[:, None]).to(DT["e4m3"]).view(torch.uint8))


@pytest.mark.parametrize("n", [512, 5000, 9000])
def test_rms_norm_8_bit_values_of_infinite_and_tiny_rows(crnn, n):
    """Infinite factors and values at the smallest scale go through the quotient as through a division."""
    x, gain = torch.ones(4, n, device="cuda"), torch.ones(n, device="cuda")
    x[1, 3] = float("inf")
    x[2] = 0
    gain[5] = float("inf")
    got = crnn.rms_norm(x, gain, eps=0.5, out_dtype=DT["e4m3"])
    y = crnn.rms_norm(x, gain, eps=0.5).y.cpu()
    want = (y / got.scale.cpu()[:, None]).to(DT["e4m3"]).float()
    torch.testing.assert_close(got.y.float().cpu(), want, rtol=0, atol=0, equal_nan=True)
    gain[5] = 1e-38
    x[0], x[1, 3] = 1e-37, 1
    got, y = crnn.rms_norm(x, gain * 1e-35, eps=1.0, out_dtype=DT["e4m3"]), crnn.rms_norm(x, gain * 1e-35, eps=1.0).y.cpu().double()
    c = got.scale.cpu().double()[:, None]
    assert float(c[0]) == 2.0 ** -126 and float(c[1]) < 1.5 * 2.0 ** -126
    assert ((got.y.float().cpu().double() * c - y).abs() <= 2.0 ** -4 * y.abs() + 2.0 ** -10 * c).all()


# (m, n): a tile of each shape, and with them each kernel of the products in three parts
@pytest.mark.parametrize("m, n", [(1, 40), (16, 40), (17, 40), (200, 300), (1500, 700), (3000, 1030), (4100, 1100)])
@pytest.mark.parametrize("k", [1, 3, 4, 8])
def test_linear_fp32_products_one_by_one(crnn, m, n, k):
    """One product per result, operands of full mantissas and one sign.  Rounded to the 8 bits of bfloat16 a value is off by 2^-8 of
    its power of two, 2^e: so |m| <= 2^-8 2^e, and l, half a step of a number below that, |l| <= 2^-9 2^-8 2^e; what is left
    after it fits l's 8 bits.  Left out are m l, l m and l l: (2 2^-25 + 2^-34) of the product.  The sum's last addition counts
    2^-23 of the result (the smaller operand is cut at half a step of the larger one, 2^-24 of it, and the sum rounded, 2^-24), the five
    before it as much of partial sums that are at most 2 2^-8 of the product."""
    g = gen(m + k)
    rel = 2.0 ** -24 + 2.0 ** -34 + 2.0 ** -23 * (1 + 5 * 2.0 ** -7)
    hard = lambda t: (1 + torch.randint(0, 128, t.shape, generator=g, device="cuda").float() / 128 - 2.0 ** -23).clamp(min=1)
    for kind in ("hard", "random"):
        x, w = torch.zeros(m, k, device="cuda"), torch.zeros(n, k, device="cuda")
        a, b = torch.rand(m, generator=g, device="cuda") + 0.5, torch.rand(n, generator=g, device="cuda") + 0.5
        if kind == "hard":
            a, b = hard(a), hard(b)
            a[::3] = b[::3] = 1 + 2.0 ** -7 - 2.0 ** -23
        x[:, k // 2], w[:, k // 2] = a, b
        want = a.double()[:, None] * b.double()
        off = ((crnn.linear(x, w).double() - want) / want).abs().max()
        assert off <= rel, (kind, float(off) * 2 ** 24)


@pytest.mark.parametrize("m, n", [(17, 40), (1500, 700), (4100, 1100)])
@pytest.mark.parametrize("k", [3, 8])
def test_linear_fp32_every_nan_stays(crnn, m, n, k):
    """NaN of any payload, also those that rounding their bits would carry out of the exponent."""
    g = gen(m)
    x, w = randn(g, m, k), randn(g, n, k)
    clean = crnn.linear(x, w)
    for bits in (0x7FFFFFFF, -1, 0x7F800001, 0x7FFF7FFF, -0x7FFFFF, 0x7FC00000):
        xn, wn = x.clone(), w.clone()
        xn[m - 1, 1], wn[5, k - 1] = (torch.tensor(bits, dtype=torch.int32).view(torch.float32),) * 2
        got = crnn.linear(xn, wn)
        assert torch.isnan(got[m - 1]).all() and torch.isnan(got[:, 5]).all(), hex(bits)
        got[:, 5] = clean[:, 5]
        assert torch.equal(got[:m - 1], clean[:m - 1])


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("n", [8193, 1 << 17, (1 << 20) + 3, 1 << 24, (1 << 27) + 1])
def test_rms_norm_of_a_long_row(crnn, n, dt):
    """One value all along, so that sums that lose what they add show it; the bound does not grow with n."""
    x = torch.full((1, n), 0.3, device="cuda").to(DT[dt])
    v = float(x[0, 0])
    x[0, n // 2] = 4 * v
    gain = torch.ones(n, device="cuda")
    r = ((v * v * (n - 1) + 16 * v * v) / n + 1e-6) ** -0.5
    # in 32 bits: the sum, n, their quotient and eps once each, halved by the root, then the root, its inverse and two products
    rel = (4 / 2 + 4) * 2.0 ** -24 + R.ROUND[DT[dt]]
    y = crnn.rms_norm(x, gain).y
    for at, t in ((0, v), (n // 2, 4 * v), (n - 1, v)):
        assert abs(float(y[0, at]) - t * r) <= rel * t * r, (at, float(y[0, at]), t * r)
    y[0, n // 2] = y[0, 0]
    assert (y == y[0, 0]).all()
    got = crnn.rms_norm(x, gain, out_dtype=DT["e4m3"])
    # the largest value times 1 / 448, two roundings more
    assert abs(float(got.scale[0]) * 448 - 4 * v * r) <= ((4 / 2 + 6) * 2.0 ** -24) * 4 * v * r


@pytest.mark.parametrize("k", [1, 8])
def test_linear_one_row_of_very_many_columns(crnn, k):
    """On both sides of 2^26 columns, where a wave for each column would take a launch of 2^32 threads."""
    for n in ((1 << 26) - 4, (1 << 26) - 3, (1 << 26) - 1, (1 << 26) + 5):
        w = torch.zeros(n, k, dtype=torch.bfloat16, device="cuda")
        w[:, k // 2] = torch.arange(n, device="cuda") % 251
        x = torch.ones(1, k, dtype=torch.bfloat16, device="cuda")
        assert torch.equal(crnn.linear(x, w)[0], w[:, k // 2])


@pytest.mark.parametrize("m, k, n", [(1, 1, 60000), (1, 8, 60000), (8, 8, 60000), (40, 8, 2000), (300, 8, 2000), (300, 3, 2000)])
def test_gelu_over_its_range(crnn, m, k, n):
    """x (1 + erf(x / sqrt 2)) / 2 at arguments that arrive exactly (the bias of a product of zeros).  Phi(-|x|), which is at most
    1/2, by a form that is off by 0.75e-7 itself; in units of 2^-24: 1.3 for that, of the evaluation 0.2 for the exponent's
    argument and 1 for the exponential, 3 roundings of t for up to 1.73 of p, 2 for the polynomial, 0.5 for the product with |x|,
    and of the result 1."""
    rel = (1.3 + 0.2 + 1 + 3 * 1.73 + 2 + 0.5 + 1) * 2.0 ** -24
    z = torch.cat([torch.linspace(-14, 14, n - n // 2), torch.logspace(-30, 1, n // 2 - n // 4), -torch.logspace(-30, 1, n // 4)])
    w = torch.zeros(n, k, device="cuda")
    got = crnn.linear(torch.zeros(m, k, device="cuda"), w, bias=z.cuda(), act="gelu").double().cpu()
    want = R.act64(z.double(), "gelu")
    assert ((got - want).abs() <= rel * z.double().abs() + R.TINY).all(), float(((got - want).abs() / z.double().abs().clamp(min=1e-30)).max() * 2 ** 24)


@pytest.mark.parametrize("m, k, n", [(3, 4096, 500), (9, 4096, 500), (48, 8192, 200), (300, 2048, 300), (800, 4096, 1100), (5000, 2048, 1100), (300, 2049, 300)])
def test_linear_8_bits_one_missing_value_shows(crnn, m, k, n):
    """Operands of +-1 (and scales of 1): every product and sum is a whole number, exact in each of the kernels."""
    g = gen(k)
    x, w = ((torch.rand(r, k, generator=g, device="cuda") < 0.5).float() * 2 - 1 for r in (m, n))
    want = (x @ w.t()).round()
    got = crnn.linear(x.to(DT["e4m3"]), w.to(DT["e4m3"]))
    assert torch.equal(got, want.to(torch.bfloat16))
    small = want.abs() <= 256                                            # (whole numbers that bfloat16 holds)
    assert small.float().mean() > 0.9 and torch.equal(got[small].float(), want[small])


@pytest.mark.parametrize("m, k, n", [(9, 4096, 500), (48, 8192, 200), (300, 2048, 300), (800, 4096, 1100), (5000, 2048, 1100), (300, 2049, 300)])
def test_linear_8_bits_error_of_many_results(crnn, m, k, n):
    """Root mean square and mean of the error over all results.  A product loses less than 2^-13 of the largest of its eight, g,
    here taken as spread evenly over that: 2^-13 g / sqrt 3 a product, of any sign, sqrt(k) of that in a sum; beside the rounding
    to bfloat16, whose own size the 64-bit results give.  A tenth more for chance; the mean of N errors lies within 5 / sqrt N of 0."""
    g = gen(k + 1)
    x, w = randn(g, m, k).to(DT["e4m3"]), randn(g, n, k).to(DT["e4m3"])
    exact = x.double() @ w.double().t().contiguous()
    off = crnn.linear(x, w).double() - exact
    pad = (-k) % 8
    top = [torch.nn.functional.pad(t.float().abs(), (0, pad)).view(t.shape[0], -1, 8).amax(2).square().mean() for t in (x, w)]
    lost = (k * float(top[0] * top[1]) / 3) ** 0.5 * 2.0 ** -13
    own = exact.to(torch.bfloat16).double() - exact
    rms = lambda t: float(t.square().mean() ** 0.5)
    print("%d x %d x %d: rms %.4g, rounding alone %.4g, allowed for the instructions %.4g; mean %.3g of %.3g" % (m, k, n, rms(off), rms(own), lost, float(off.mean()), rms(exact)))
    assert rms(off) <= 1.1 * (rms(own) ** 2 + lost ** 2) ** 0.5
    assert abs(float(off.mean())) <= 5 * rms(off) / (m * n) ** 0.5


@pytest.mark.parametrize("m, k, n", [(9, 4096, 500), (48, 8192, 200), (300, 2048, 300), (800, 4096, 1100), (300, 2049, 300)])
def test_linear_8_bits_operands_of_one_sign(crnn, m, k, n):
    """What the instructions cut off products of one sign adds up: less than 2^-13 of the largest of eight, g, a product."""
    g = gen(k + 2)
    x, w = randn(g, m, k).abs().to(DT["e4m3"]), randn(g, n, k).abs().to(DT["e4m3"])
    exact = x.double() @ w.double().t().contiguous()
    off = crnn.linear(x, w).double() - exact
    pad = (-k) % 8
    xg, wg = (torch.nn.functional.pad(t.double(), (0, pad)).view(t.shape[0], -1, 8).amax(2) for t in (x, w))
    lost = 8 * 2.0 ** -13 * (xg @ wg.t().contiguous())
    own = exact.to(torch.bfloat16).double() - exact
    print("%d x %d x %d: mean error %.3g of %.4g, allowed %.3g; rms %.4g, rounding alone %.4g" % (m, k, n, float(off.mean()), float(exact.mean()), float(lost.mean()), float(off.square().mean() ** 0.5), float(own.square().mean() ** 0.5)))
    # (the last term: 2^-23 for each of the sums' additions, and a result that crosses the middle of two values moves a whole step)
    assert (off.abs() <= lost + (k + 8) * 2.0 ** -23 * exact + 2.0 ** -8 * exact * (1 + 2.0 ** -8)).all()
    assert abs(float((off - own).mean())) <= float(lost.mean()) + (k + 8) * 2.0 ** -23 * float(exact.mean()) + 5 * float(own.square().mean() ** 0.5) * (2 / (m * n)) ** 0.5
