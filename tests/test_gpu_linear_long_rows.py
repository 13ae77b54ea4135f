"""Linear over rows of more than 2^31 bytes, and over more than 2^30 rows: what lies past them counts."""
import pytest
import torch

from test_gpu_float_ops import _check, _linear64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,o", [(1, 2), (5, 1)])
def test_the_end_of_a_row_past_2_31_bytes(ops, dev, dtype, m, o):
    k, n = ((1 << 30) if dtype != torch.float32 else (1 << 29)) + 264, 200  # zeros, but for the first and the last 200 values
    g = torch.Generator(device=dev).manual_seed(m)
    x, w = torch.zeros((m, k), dtype=dtype, device=dev), torch.zeros((o, k), dtype=dtype, device=dev)
    for t in (x, w):
        t[:, :n] = torch.randn((t.shape[0], n), device=dev, generator=g).to(dtype)
        t[:, -n:] = torch.randn((t.shape[0], n), device=dev, generator=g).to(dtype)
    y = ops.Linear(x, w, activation="Relu")
    both = lambda t: torch.cat([t[:, :n], t[:, -n:]], dim=1)  # noqa: E731
    want, bound = _linear64(both(x), both(w), None, "Relu", None, False)  # (the other terms are zero, whatever their order)
    _check(y, want, bound)
    ops.device_status()


@pytest.mark.parametrize("bias", [False, True])
def test_more_rows_than_one_launch_takes(ops, dev, bias):
    n = (1 << 30) + 300
    g = torch.Generator(device=dev).manual_seed(7)
    few, b = torch.randn((9, 8), device=dev, generator=g).bfloat16(), torch.randn(n, device=dev, generator=g).bfloat16() if bias else None
    many = torch.zeros((n, 8), dtype=torch.bfloat16, device=dev)
    many[:400], many[-400:] = (torch.randn((400, 8), device=dev, generator=g).bfloat16() for _ in range(2))
    y = ops.Linear(few, many, b, activation="Relu")
    for part in (slice(0, 400), slice(n - 400, n)):
        want, bound = _linear64(few, many[part], b[part] if bias else None, "Relu", None, False)
        _check(y[:, part], want, bound)
    del y
    y = ops.Linear(many, few, b[:9] if bias else None, activation="Relu")
    for part in (slice(0, 400), slice(n - 400, n)):
        want, bound = _linear64(many[part], few, b[:9] if bias else None, "Relu", None, False)
        _check(y[part], want, bound)
    ops.device_status()
