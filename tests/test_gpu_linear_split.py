"""The float32 product on split operands (Linear with an epilogue): its error over K, for every width of tile, and over the range of the type.

Relative error of the sums, root mean square over normal terms: an operand is held to 2^-22 and the product of two low parts is left out (2^-21 together), and a
chain of sixteen instructions may truncate by 2^-23 of its sum each time: at most 2^-21 + 16 * 2^-23 = 2.4e-6.  A product that lost one of its small parts
is off by 1e-4."""
import math

import pytest
import torch

from test_gpu_float_ops import E32, _check, _linear64

pytestmark = pytest.mark.gpu
RMS = 2.0 ** -21 + 16 * 2.0 ** -23


def _operands(dev, m, k, o, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed + m + k + o)
    return torch.randn((m, k), device=dev, generator=g, dtype=torch.float64), torch.randn((o, k), device=dev, generator=g, dtype=torch.float64)


def _rms(y, x, w):
    z = x.double() @ w.double().t()
    return float((y.double() - z).norm() / z.norm())


@pytest.mark.parametrize("m,o", [(13, 5000), (32, 3000), (64, 3000), (200, 3000), (40, 2000), (700, 1500)])  # tiles of 16, 32, 64 and 128 rows, alone and shared
@pytest.mark.parametrize("k", [100, 1283, 2048, 4096])
def test_error_over_k(ops, dev, m, o, k):
    x, w = (t.float() for t in _operands(dev, m, k, o))
    y = ops.Linear(x, w, residual=torch.zeros((m, o), device=dev))
    assert _rms(y, x, w) <= RMS
    _check(y, *_linear64(x, w, None, None, None, False))


@pytest.mark.parametrize("m,k,o", [(40, 64, 3000), (300, 256, 1500)])
@pytest.mark.parametrize("e", [-150, -126, -125, -124, -122, -118, -114, -100, -60, 60, 100, 112, 115, 116, 117, 119])
@pytest.mark.parametrize("small", ["x", "w"])
def test_error_over_the_range_of_the_type(ops, dev, m, k, o, e, small):
    """One operand about 2^e, the other about 2^-e (2^120 at most).  Subnormal values are held to a unit or two of 2^-149."""
    x, w = _operands(dev, m, k, o, e)
    other = max(-120, min(-e, 120))
    x, w = (x * 2.0 ** e, w * 2.0 ** other) if small == "x" else (x * 2.0 ** other, w * 2.0 ** e)
    x, w = x.float(), w.float()
    y = ops.Linear(x, w, residual=torch.zeros((m, o), device=dev))
    want, bound = _linear64(x, w, None, None, None, False)
    _check(y, want, bound + 2.0 ** -147 * (x.double().abs().sum(dim=1)[:, None] + w.double().abs().sum(dim=1)[None]))
    if e >= -122:
        assert _rms(y, x, w) <= RMS


@pytest.mark.parametrize("m,o", [(40, 3000), (300, 1500)])
def test_the_largest_values(ops, dev, m, o):
    """Every value of the last binade, up to the largest of all, times values that keep the sums in range; infinities and NaN beside them."""
    k = 96
    x, w = (t.float() for t in _operands(dev, m, k, o))
    big = torch.finfo(torch.float32).max
    x = torch.where(x.abs() > 0.2, torch.sign(x) * big * (1 - torch.rand(x.shape, device=dev, generator=torch.Generator(device=dev).manual_seed(1)) / 3), x)
    x[:, 0], x[:, 1] = big, -big
    w = w / 256
    y = ops.Linear(x, w, residual=torch.zeros((m, o), device=dev))
    want, bound = _linear64(x, w, None, None, None, False)
    _check(y, want, bound)
    assert _rms(y.double() / big, x.double() / big, w) <= RMS
    x[3, 5], x[4, 6], x[5, 7] = float("inf"), float("nan"), float("-inf")
    z = ops.Linear(x, w, residual=torch.zeros((m, o), device=dev))
    keep = [i for i in range(m) if i not in (3, 4, 5)]
    assert torch.equal(z[keep], y[keep]) and torch.isnan(z[4]).all()
    assert torch.equal(z[3], torch.copysign(torch.full_like(z[3], float("inf")), w[:, 5])) and torch.equal(z[5], torch.copysign(torch.full_like(z[5], float("inf")), -w[:, 7]))


def test_exact_products_of_eleven_bits(ops, dev):
    """Whole numbers of up to eleven bits are their own high parts: their products and sums are exact."""
    g = torch.Generator(device=dev).manual_seed(3)
    x, w = (torch.randint(-2047, 2048, s, device=dev, generator=g).float() for s in ((300, 4), (1500, 4)))
    assert torch.equal(ops.Linear(x, w, activation="Relu").double(), (x.double() @ w.double().t()).clamp(min=0))
    assert E32 == 2.0 ** -23
