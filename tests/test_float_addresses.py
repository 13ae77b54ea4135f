"""Addresses that are no multiple of their values' size would fault on the device: the C entries of the float operators refuse them (host side, no GPU;
no address here is read)."""
import ctypes

import pytest


def _call(pkg, entry, **kw):
    from chainer_compiler_b200 import _lib
    L, f32 = pkg.lib(), _lib.FLOAT32
    a = dict(x=64, w=64, y=64, b=64, r=64, mean=64, inv=64, dy=64, dx=64, dscale=64, dbias=64, ws=64, tok=64, lp=64, ent=64, lse=64, top=64, toptok=64, dtype=f32, affine=f32,
             tok_dtype=_lib.INT64)
    a.update(kw)
    if entry == "linear":
        p = _lib.LinearParams(x=a["x"], ldx=8, w=a["w"], ldw=8, dtype=a["dtype"], activation=1, bias=a["b"], bias_dtype=a["affine"], residual=a["r"], ldr=8, M=3, O=8, K=8, y=a["y"], ldy=8)
        return L.chxq_linear(ctypes.byref(p), None, 0, None)
    if entry == "linear_f32":
        return L.chxq_linear_f32(a["x"], a["w"], a["b"], 3, 8, 8, a["y"], None)
    if entry == "norm":
        return L.chxq_layernorm(a["x"], 8, a["dtype"], a["w"], a["b"], a["affine"], 3, 8, 1e-5, a["y"], a["mean"], a["inv"], None)
    if entry == "norm_grad":
        return L.chxq_layernorm_grad(a["dy"], 8, a["x"], 8, a["dtype"], a["w"], a["affine"], a["mean"], a["inv"], 3, 8, a["dx"], a["dscale"], a["dbias"], a["ws"],
                                     L.chxq_layernorm_grad_workspace(3, 8), None)
    if entry == "logprobs":
        return L.chxq_token_logprobs(a["x"], 8, a["dtype"], a["tok"], a["tok_dtype"], 3, 8, 2, 0, 0, a["lp"], a["ent"], a["lse"], a["top"], a["toptok"], None)
    return L.chxq_token_logprobs_grad(a["lp"], a["dy"], a["x"], 8, a["dtype"], a["tok"], a["tok_dtype"], a["lse"], a["ent"], 3, 8, 0, 0, a["dx"], None)


@pytest.mark.parametrize("entry,names", [("linear", "x w y b r"), ("linear_f32", "x w y b"), ("norm", "x w b y mean inv"), ("norm_grad", "dy x w mean inv dx dscale dbias ws"),
                                         ("logprobs", "x tok lp ent lse top toptok"), ("logprobs_grad", "lp dy x tok lse ent dx")])
def test_addresses_between_values_are_refused(pkg, entry, names):
    from chainer_compiler_b200 import _lib
    for name in names.split():
        for off in (1, 2, 3) + ((4,) if name in ("tok", "toptok") else ()):
            assert _call(pkg, entry, **{name: 64 + off}) == _lib.ERR_INVALID_ARGUMENT, (name, off)
            assert b"multiple" in pkg.lib().chxq_last_error()
        if name in ("x", "y", "r", "w", "dx") and entry != "linear_f32":
            more = dict(dtype=_lib.BFLOAT16, affine=_lib.BFLOAT16)
            assert _call(pkg, entry, **{name: 65}, **more) == _lib.ERR_INVALID_ARGUMENT and b"multiple" in pkg.lib().chxq_last_error()
