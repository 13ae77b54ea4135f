"""TokenLogProbs where the alternatives' buffers fill up to the end of a row: rows that ascend, so that every access offers all its values, at every length
and place of a 16-byte piece, so that the values in front of the first and behind the last whole piece are offered behind a buffer of every level."""
import math

import pytest
import torch

from test_gpu_float_ops import E32, EF

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [3, 1300])  # a block a row, a warp a row
@pytest.mark.parametrize("k", [1, 20, 32])
def test_ascending_rows_of_every_length(ops, dev, dtype, rows, k):
    vec = 128 // torch.finfo(dtype).bits
    body = 32 * vec * 4 * 5  # five rounds of a warp's accesses
    for v in list(range(body - vec, body + vec, 3)) + [k, 32 + k, 32 * vec + 1, 32 * vec * 2 + vec - 1]:
        for shift in (0, 1, vec - 1):
            buf = torch.zeros((rows, v + vec), device=dev, dtype=dtype)
            x = buf[:, shift:shift + v]
            x.copy_((torch.arange(v, device=dev, dtype=torch.float32) / 64 - 8).to(dtype).expand(rows, v))  # (16 bits: equal neighbours too)
            tok = torch.arange(rows, device=dev) % v
            _, _, _, top_lp, top = ops.TokenLogProbs(x, tok, k)
            order = torch.sort(x[0], descending=True, stable=True)[1][:k]
            assert torch.equal(top, order.expand(rows, k)), (v, shift)
            # Rows that start at other places of a piece sum in another order: the sum of v exponentials is off by v 2^-23 + 2^-20, so its logarithm by as much.
            want = torch.log_softmax(x[0].double(), dim=0)[order]
            assert ((top_lp.double() - want).abs() <= v * E32 + EF + 8 * E32 * (2 * want.abs() + math.log(v) + 1)).all(), (v, shift)
