"""LayerNormalization and its gradient over rows shorter than sixteen bytes, several of which lie in one access: alone in their memory, and as the last
rows of a buffer whose other values must not count."""
import pytest
import torch

from test_gpu_float_ops import TYPES, _check_grad, _check_norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", list(range(1, 10)) + [15, 17])
@pytest.mark.parametrize("rows", [1, 2, 3, 5, 7, 8, 9, 31, 1001])
def test_short_rows(ops, dev, dtype, d, rows):
    if d > 1:  # (the deviations of a row of one value are zero)
        _check_norm(ops, dev, rows, d, dtype, torch.float32)
    _check_grad(ops, dev, rows, d, dtype, torch.float32)
    # the same rows with NaN behind them: the same bits
    g = torch.Generator(device=dev).manual_seed(rows + d)
    x, dy = (torch.randn((rows, d), device=dev, generator=g).to(dtype) for _ in range(2))
    s = torch.randn(d, device=dev, generator=g)
    y, mean, inv = ops.LayerNormalization(x, s, stats=True)
    want = (y, *ops.LayerNormalizationGrad(dy, x, s, mean, inv))
    wx, wd = (torch.cat([t.reshape(-1), t.new_full((64,), float("nan"))])[:rows * d].view(rows, d) for t in (x, dy))
    got = (ops.LayerNormalization(wx, s), *ops.LayerNormalizationGrad(wd, wx, s, mean, inv))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
