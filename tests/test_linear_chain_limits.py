"""Limits of the float32 product without an epilogue (host side, no GPU)."""


def test_rows_too_long_to_count_are_refused(pkg):
    """(Addresses here are never read: the call ends in the check of its arguments.)"""
    from chainer_compiler_b200 import _lib
    for k in (2 ** 31 - 1, 2 ** 31 - 32, 2 ** 31 - 1024):
        assert pkg.lib().chxq_linear_f32(64, 64, None, 1, k, 1, 64, None) == _lib.ERR_INVALID_ARGUMENT
        assert b"too long" in pkg.lib().chxq_last_error()
    for n, k, o in ((0, 8, 8), (8, 0, 8), (8, 8, 0), (-1, 8, 8)):
        assert pkg.lib().chxq_linear_f32(64, 64, None, n, k, o, 64, None) == _lib.ERR_INVALID_ARGUMENT
