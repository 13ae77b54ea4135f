"""Which kernel a Linear takes (host side, no GPU): the sizes of test_gpu_linear_pairs.py are those of the CTA pairs, and every other kernel is within
reach of sizes that test_gpu_float_ops.py has."""
import ctypes

import pytest

from test_gpu_linear_pairs import PAIRS


def route(pkg, m, k, o, dtype="bfloat16", **kw):
    from chainer_compiler_b200 import _lib
    code = {"float32": _lib.FLOAT32, "float16": _lib.FLOAT16, "bfloat16": _lib.BFLOAT16}[dtype]
    d = dict(x=256, ldx=k, w=256, ldw=k, dtype=code, y=256, ldy=o, M=m, O=o, K=k)
    d.update(kw)
    p, kernel = _lib.LinearParams(**d), ctypes.c_int32(-1)
    rc = pkg.lib().chxq_linear_kernel(ctypes.byref(p), ctypes.byref(kernel))
    return kernel.value if rc == 0 else -rc


@pytest.mark.parametrize("m,k,o", PAIRS)
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_the_sizes_of_the_pair_tests_run_on_pairs(pkg, m, k, o, dtype):
    from chainer_compiler_b200 import _lib
    assert route(pkg, m, k, o, dtype) == _lib.LINEAR_PAIRS
    assert route(pkg, m, k, o, dtype, ldx=k + 3, ldw=k + 5, ldy=o + 1) == _lib.LINEAR_PAIRS


def test_the_other_kernels(pkg):
    from chainer_compiler_b200 import _lib
    for dtype in ("float16", "bfloat16"):
        assert route(pkg, 1, 1024, 4096, dtype) == route(pkg, 64, 2000, 64, dtype) == _lib.LINEAR_ROWS
        assert route(pkg, 1, 8192, 8192, dtype) == route(pkg, 20, 96, 2500, dtype) == route(pkg, 140, 96, 600, dtype) == route(pkg, 512, 4096, 4096, dtype) == _lib.LINEAR_TILES
    assert route(pkg, 8, 4096, 4096, "float32") == _lib.LINEAR_ROWS
    assert route(pkg, 256, 2048, 1000, "float32") == route(pkg, 2048, 2048, 2048, "float32") == _lib.LINEAR_TILES_F32
    assert route(pkg, 0, 8, 8) == route(pkg, 8, 0, 8) == route(pkg, 8, 8, 0) == _lib.LINEAR_NO_PRODUCT


@pytest.mark.parametrize("dtype,size", [("float16", 2), ("bfloat16", 2), ("float32", 4)])
def test_rows_whose_bytes_pass_the_coordinates_of_tma(pkg, dtype, size):
    """(TMA's coordinates are 32 signed bits; the kernels that use it count bytes along a row.)"""
    from chainer_compiler_b200 import _lib
    for m, o in ((1, 1), (1, 2), (5, 1), (9, 3), (40, 40), (200, 700)):
        for k in ((1 << 31) // size - 64, (1 << 31) // size + 8, (1 << 30) + 264):
            assert route(pkg, m, k, o, dtype) == _lib.LINEAR_ROWS
    if size == 2:
        assert route(pkg, 1, 1 << 28, 8, dtype) == _lib.LINEAR_TILES


def test_rows_off_16_byte_boundaries(pkg):
    """Read value by value: as long as all blocks of eight rows of x together read no more than 2^22 weights, and always for four rows."""
    from chainer_compiler_b200 import _lib
    for dtype in ("float16", "bfloat16"):
        for m, k, o in ((4, 8001, 4096), (8, 1001, 4096), (8, 4001, 1000), (16, 1001, 1000), (64, 8001, 64)):
            assert route(pkg, m, k, o, dtype) == _lib.LINEAR_ROWS
        for m, k, o in ((8, 8001, 1000), (16, 4001, 1000), (64, 8001, 256), (64, 2001, 1000)):
            assert route(pkg, m, k, o, dtype) == _lib.LINEAR_TILES


def test_refusals(pkg):
    from chainer_compiler_b200 import _lib
    bad = -_lib.ERR_INVALID_ARGUMENT
    assert route(pkg, -1, 8, 8) == bad and route(pkg, 4, 8, 8, ldx=7) == bad and route(pkg, 4, 8, 8, dtype="float16", activation=9) == bad
    assert pkg.lib().chxq_linear_kernel(None, None) == _lib.ERR_INVALID_ARGUMENT
