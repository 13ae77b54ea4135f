"""The float operators on a host without a GPU: refusals of the op bodies and of the C ABI, which come before any device is touched."""
import ctypes

import pytest
import torch


def test_float_ops_refuse_cpu_tensors(ops):
    x, w, v, t = torch.zeros(2, 4), torch.zeros(3, 4), torch.zeros(4), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: ops.Linear(x, w, activation="Relu"), lambda: ops.LayerNormalization(x, v),
                 lambda: ops.LayerNormalizationGrad(x, x, v, torch.zeros(2), torch.zeros(2)), lambda: ops.TokenLogProbs(x, t),
                 lambda: ops.TokenLogProbsGrad(torch.zeros(2), None, x, t, torch.zeros(2))):
        with pytest.raises(ops.ChxqError):
            call()
    with pytest.raises(TypeError):
        ops.LayerNormalization([[1.0]], v)


@pytest.mark.parametrize("name", ["relu", "Softmax", 3, ["Relu"]])
def test_unknown_activations_are_refused(ops, name):
    with pytest.raises(ops.ChxqError, match="unknown activation"):
        ops.Linear(torch.zeros(2, 4), torch.zeros(3, 4), activation=name)


def _params(**kw):
    from chainer_compiler_b200 import _lib
    d = dict(x=64, ldx=32, w=64, ldw=32, dtype=_lib.BFLOAT16, y=64, ldy=16, M=4, O=16, K=32)
    d.update(kw)
    return _lib.LinearParams(**d)


@pytest.mark.parametrize("change", [dict(dtype=9), dict(M=-1), dict(K=-2), dict(O=1 << 31), dict(x=None), dict(y=None), dict(ldx=31), dict(ldw=8), dict(ldy=15),
                                    dict(bias=64, bias_dtype=7), dict(activation=7), dict(activation=-1), dict(residual=64, ldr=15)])
def test_linear_refuses_bad_parameters(pkg, change):
    """(Addresses here are never read: every one of these calls ends in the check of its arguments.)"""
    from chainer_compiler_b200 import _lib
    p = _params(**change)
    assert pkg.lib().chxq_linear(ctypes.byref(p), None, 0, None) == _lib.ERR_INVALID_ARGUMENT
    assert pkg.lib().chxq_linear(None, None, 0, None) == _lib.ERR_INVALID_ARGUMENT


def test_linear_without_outputs_does_nothing(pkg):
    for kw in (dict(M=0), dict(O=0)):
        p = _params(x=None, w=None, y=None, **kw)
        assert pkg.lib().chxq_linear(ctypes.byref(p), None, 0, None) == 0 and pkg.lib().chxq_linear_workspace(ctypes.byref(p)) == 0


def test_norm_and_logprob_refusals(pkg):
    from chainer_compiler_b200 import _lib
    L, bad = pkg.lib(), _lib.ERR_INVALID_ARGUMENT
    f32, f16, bf16 = _lib.FLOAT32, _lib.FLOAT16, _lib.BFLOAT16
    norm = lambda x=64, ld=8, dt=f32, scale=64, adt=f32, rows=3, d=8, y=64: L.chxq_layernorm(x, ld, dt, scale, None, adt, rows, d, 1e-5, y, None, None, None)  # noqa: E731
    assert norm(dt=3) == bad and norm(dt=f16, adt=bf16) == bad and norm(d=0) == bad and norm(rows=-1) == bad and norm(ld=7) == bad and norm(x=None) == bad
    assert norm(scale=None) == bad and norm(y=None) == bad and norm(rows=0, x=None, y=None) == 0
    need = L.chxq_layernorm_grad_workspace(3, 8)
    grad = lambda nbytes, rows=3, d=8, ws=64, x=64, ld=8, mean=64: L.chxq_layernorm_grad(64, 8, x, ld, f32, 64, f32, mean, 64, rows, d, 64, 64, 64, ws, nbytes, None)  # noqa: E731
    assert need > 0 and grad(need - 1) == _lib.ERR_WORKSPACE and grad(need, ws=None) == _lib.ERR_WORKSPACE
    assert grad(need, d=0) == bad and grad(need, x=None) == bad and grad(need, ld=7) == bad and grad(need, mean=None) == bad
    lp = lambda top=0, v=8, ld=8, dt=f32, tdt=_lib.INT64, rows=3, tok=64, tops=64: L.chxq_token_logprobs(64, ld, dt, tok, tdt, rows, v, top, 0, 0, 64, 64, 64, tops, tops, None)  # noqa: E731
    assert lp(top=9) == bad and lp(top=33, v=64, ld=64) == bad and lp(top=-1) == bad and lp(v=0) == bad and lp(ld=7) == bad and lp(dt=6) == bad
    assert lp(tdt=f32) == bad and lp(tok=None) == bad and lp(top=1, tops=None) == bad and lp(rows=0, tok=None) == 0
    lpg = lambda v=8, dent=None, ent=None, lse=64, out=64: L.chxq_token_logprobs_grad(64, dent, 64, 8, f32, 64, _lib.INT64, lse, ent, 3, v, 0, 0, out, None)  # noqa: E731
    assert lpg(dent=64) == bad and lpg(lse=None) == bad and lpg(out=None) == bad and lpg(v=9) == bad
