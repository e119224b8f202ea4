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
