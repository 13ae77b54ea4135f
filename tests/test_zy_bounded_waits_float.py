"""The bounded device-side waits of Linear's tensor-core kernels and of LayerNormalizationGrad's ring, made to run out in the allowed way: a hook leaves
one load out, so that its stage never fills; with the wait limit shortened to 5 ms the waits behind it expire, every role leaves its loop, and the kernel
returns by itself.  Nothing traps, faults or spins on: the status word reports the timeout, and the next ordinary call has the bits of the one before."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu


def _expire(pkg, ops, skip, call):
    from chainer_compiler_b200 import _lib
    L = pkg.lib()
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    want = [t.clone() for t in call()]
    ops.device_status()
    try:
        _lib.check(L.chxq_tc_test_hooks(5_000_000, skip))
        call()
        rc = L.chxq_device_status(stream)  # synchronizes; the kernel has returned by itself
        assert rc == _lib.ERR_DEVICE_TIMEOUT, rc
        assert L.chxq_device_status(stream) == _lib.OK  # reading the status cleared it
    finally:
        _lib.check(L.chxq_tc_test_hooks(2_000_000_000, -1))
    got = call()
    ops.device_status()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def _linear(ops, dev, m, k, o, dtype, residual):
    g = torch.Generator(device=dev).manual_seed(m + k + o)
    x, w = (torch.randn(s, device=dev, generator=g).to(dtype) for s in ((m, k), (o, k)))
    r = torch.randn((m, o), device=dev, generator=g).to(dtype) if residual else None
    return lambda: [ops.Linear(x, w, activation="Swish", residual=r)]


@pytest.mark.parametrize("m,k,o,skip", [(2500, 264, 1500, 1), (12, 1024, 3000, 0), (40, 512, 1000, 3), (140, 2048, 1000, 31)])  # a CTA a tile, and clusters that share one
def test_tiles_of_16_bits(pkg, ops, dev, m, k, o, skip):
    _expire(pkg, ops, skip, _linear(ops, dev, m, k, o, torch.bfloat16, True))


@pytest.mark.parametrize("m,k,o,skip", [(2048, 512, 2048, 5), (300, 256, 1500, 0), (20, 2048, 2500, 63), (40, 640, 3000, 7)])
def test_tiles_of_float32(pkg, ops, dev, m, k, o, skip):
    _expire(pkg, ops, skip, _linear(ops, dev, m, k, o, torch.float32, True))


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("m,k,o,skip", [(2000, 1024, 2048, 0), (2000, 1024, 2055, 9), (4100, 512, 4097, 7)])  # with TMA's output and residual, and without
def test_pairs(pkg, ops, dev, m, k, o, skip, residual):
    _expire(pkg, ops, skip, _linear(ops, dev, m, k, o, torch.float16, residual))


@pytest.mark.parametrize("rows,d,dtype,skip", [(2405, 4096, torch.bfloat16, 0), (2405, 1283, torch.float16, 2), (1203, 8192, torch.float32, 7), (1203, 16384, torch.float32, 5),
                                               (1203, 16384, torch.bfloat16, 3), (803, 28000, torch.bfloat16, 9), (803, 12001, torch.float16, 0)])  # blocks, and clusters
def test_ring_of_the_gradient(pkg, ops, dev, rows, d, dtype, skip):
    g = torch.Generator(device=dev).manual_seed(rows + d)
    x, dy = (torch.randn((rows, d), device=dev, generator=g).to(dtype) for _ in range(2))
    s = torch.randn(d, device=dev, generator=g)
    _, mean, inv = ops.LayerNormalization(x, s, stats=True)
    _expire(pkg, ops, skip, lambda: ops.LayerNormalizationGrad(dy, x, s, mean, inv))
