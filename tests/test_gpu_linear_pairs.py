"""Linear on CTA pairs, the kernel of large 16-bit products: every activation, bias and residual order, residuals and outputs on 16-byte rows (through
TMA) and off them (copied), more blocks than pairs, more K blocks than stages, against the formula in 64 bits; and the same bits from every call.

The tolerances are those of test_gpu_float_ops.py: one rounding of the result, and n 2^-23 of the sum of the terms' magnitudes for a sum of n terms."""
import ctypes
import math

import pytest
import torch

from test_gpu_float_ops import ACTS, _check, _linear64

pytestmark = pytest.mark.gpu

HALVES = [torch.float16, torch.bfloat16]
# m, k, o: one K block; few blocks of many K blocks; ragged in every extent; several blocks a pair
PAIRS = [(8192, 64, 1024), (2000, 1024, 2048), (2000, 1024, 2055), (3000, 520, 3001), (2048, 1024, 1500), (2048, 2048, 2047), (4100, 1024, 4097), (1024, 4096, 4096)]


def _takes_pairs(ops, x, w, y, r):
    from chainer_compiler_b200 import _lib
    code = {torch.float16: _lib.FLOAT16, torch.bfloat16: _lib.BFLOAT16}[x.dtype]
    p = _lib.LinearParams(x=x.data_ptr(), ldx=x.stride(0), w=w.data_ptr(), ldw=w.stride(0), dtype=code, y=y.data_ptr(), ldy=y.stride(0), M=x.shape[0], O=w.shape[0], K=x.shape[1],
                          residual=r.data_ptr() if r is not None else None, ldr=r.stride(0) if r is not None else 0)
    kernel = ctypes.c_int32(-1)
    _lib.check(_lib.lib().chxq_linear_kernel(ctypes.byref(p), ctypes.byref(kernel)))
    return kernel.value == _lib.LINEAR_PAIRS


def _operands(dev, m, k, o, dtype, residual, bias, pitch=0, rpitch=0, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed + m * 7 + k * 3 + o)
    x = torch.randn((m, k + pitch), device=dev, generator=g).to(dtype)[:, :k]
    w = (torch.randn((o, k + pitch), device=dev, generator=g) / math.sqrt(k)).to(dtype)[:, :k]
    b = {"none": None, "own": torch.randn(o, device=dev, generator=g).to(dtype), "float32": torch.randn(o, device=dev, generator=g)}[bias]
    r = torch.randn((m, o + rpitch), device=dev, generator=g).to(dtype)[:, :o] if residual else None
    return x, w, b, r


def _run(ops, dev, m, k, o, dtype, act, residual, bias, pitch=0, rpitch=0, repeat=2):
    x, w, b, r = _operands(dev, m, k, o, dtype, residual, bias, pitch, rpitch)
    call = lambda: ops.Linear(x, w, b, activation=act, residual=r, residual_first=residual == "first")  # noqa: E731
    y = call()
    assert _takes_pairs(ops, x, w, y, r)
    want, bound = _linear64(x, w, b, act, r, residual == "first")
    _check(y, want, bound, "Linear on pairs %s" % ((m, k, o, dtype, act, residual, bias, pitch, rpitch),))
    for _ in range(repeat):
        assert torch.equal(call(), y)
    ops.device_status()


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("residual", [None, "last", "first"])
@pytest.mark.parametrize("m,k,o", PAIRS)
def test_extents(ops, dev, dtype, residual, m, k, o):
    _run(ops, dev, m, k, o, dtype, "Gelu" if residual else None, residual, "own")


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("residual", [None, "last", "first"])
@pytest.mark.parametrize("o", [2048, 2055])
def test_epilogues(ops, dev, dtype, act, residual, o):
    _run(ops, dev, 2000, 1024, o, dtype, act, residual, "float32" if act else "none", repeat=1)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("residual", ["last", "first"])
@pytest.mark.parametrize("rpitch", [1, 7, 8])
def test_residuals_cut_out_of_wider_buffers(ops, dev, dtype, residual, rpitch):
    """The output's rows start on 16-byte boundaries; the residual's do not where the pitch is odd."""
    _run(ops, dev, 4100, 512, 4096, dtype, "Relu", residual, "own", rpitch=rpitch, repeat=4)


@pytest.mark.parametrize("dtype", HALVES)
def test_a_residual_that_starts_off_a_boundary(ops, dev, dtype):
    m, k, o = 3000, 512, 2560
    x, w, b, _ = _operands(dev, m, k, o, dtype, None, "own")
    r = torch.randn(m * o + 3, device=dev, generator=torch.Generator(device=dev).manual_seed(2)).to(dtype)[3:].view(m, o)
    y = ops.Linear(x, w, b, activation="Tanh", residual=r)
    assert _takes_pairs(ops, x, w, y, r)
    want, bound = _linear64(x, w, b, "Tanh", r, False)
    _check(y, want, bound)
    assert all(torch.equal(ops.Linear(x, w, b, activation="Tanh", residual=r), y) for _ in range(4))


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("pitch", [1, 8])
def test_operands_cut_out_of_wider_buffers(ops, dev, dtype, pitch):
    _run(ops, dev, 2048, 1024, 2047, dtype, "Swish", "last", "own", pitch=pitch)


def test_special_values(ops, dev):
    m, o = 2300, 2055
    for dtype in HALVES:
        x = torch.zeros((m, 1024), dtype=dtype, device=dev)
        w = torch.zeros((o, 1024), dtype=dtype, device=dev)
        w[:, 0] = 1
        x[:, 0] = torch.tensor([float("nan"), float("inf"), -300.0, 300.0], dtype=dtype, device=dev)[torch.arange(m, device=dev) % 4]
        zero = torch.zeros((m, o), dtype=dtype, device=dev)
        for act in ACTS:
            y = ops.Linear(x, w, activation=act, residual=zero).float()
            assert _takes_pairs(ops, x, w, zero, zero)
            want = [float("inf"), {None: -300.0, "Tanh": -1.0}.get(act, 0.0), 300.0]
            if act in ("Sigmoid", "Tanh"):
                want[0] = want[2] = 1.0
            assert torch.isnan(y[::4]).all(), act
            for i in (1, 2, 3):
                assert (y[i::4] == want[i - 1]).all(), (act, i)


def test_the_output_in_the_residuals_memory(pkg, dev):
    """The C ABI lets y be the residual's memory, on 16-byte rows and off them."""
    from chainer_compiler_b200 import _lib
    for o in (2048, 2055):
        m, k = 2000, 512
        x, w, b, r = _operands(dev, m, k, o, torch.bfloat16, "last", "own")
        want, bound = _linear64(x, w, b, None, r, False)
        p = _lib.LinearParams(x=x.data_ptr(), ldx=k, w=w.data_ptr(), ldw=k, dtype=_lib.BFLOAT16, bias=b.data_ptr(), bias_dtype=_lib.BFLOAT16, residual=r.data_ptr(), ldr=o,
                              M=m, O=o, K=k, y=r.data_ptr(), ldy=o)
        _lib.check(pkg.lib().chxq_linear(ctypes.byref(p), None, 0, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
        _check(r, want, bound)
