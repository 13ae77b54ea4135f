"""Float ONNX graphs through run_onnx: every Linear, LayerNormalization and loss of a block against its formula in 64 bits on the values it read, the same
graph captured and replayed, gradient nodes, broadcast Adds, and the most probable classes on the command line."""
import json

import numpy as np
import pytest
import torch

import __graft_entry__ as entry
from test_gpu_float_ops import E32, EF, _check, _linear64, _norm64, _tiny, _u

pytestmark = pytest.mark.gpu
B, S, D, F, V = 3, 7, 48, 96, 33


@pytest.fixture(scope="module")
def mods():
    entry.load_package()
    from chainer_compiler_b200 import onnx_io, ops, run_onnx
    return onnx_io, ops, run_onnx


def _block(onnx_io, dtype):
    rng = np.random.default_rng(1)
    N = lambda op, i, o, **a: onnx_io.Node(op, i, o, a)  # noqa: E731
    r = lambda *s: (rng.standard_normal(s) * 0.3).astype(dtype)  # noqa: E731
    inits = {"s1": r(D) + dtype(1), "c1": r(D), "w1": r(D, F), "b1": r(F), "w2": r(F, D), "b2": r(D), "s2": r(D) + dtype(1), "c2": r(D), "w3": r(D, V), "b3": r(1, V),
             "rows": np.array([-1, D], np.int64), "flat": np.array([-1], np.int64)}
    nodes = [N("LayerNormalization", ["x", "s1", "c1"], ["n1"], epsilon=1e-5), N("MatMul", ["n1", "w1"], ["p1"]), N("Add", ["p1", "b1"], ["q1"]), N("Gelu", ["q1"], ["a1"]),
             N("MatMul", ["a1", "w2"], ["p2"]), N("Add", ["p2", "b2"], ["q2"]), N("Add", ["q2", "x"], ["h"]),
             N("LayerNormalization", ["h", "s2", "c2"], ["n2", "mean", "inv"], axis=2, epsilon=1e-3), N("Reshape", ["n2", "rows"], ["f"]),
             N("Gemm", ["f", "w3", "b3"], ["logits"]), N("SoftmaxCrossEntropyLoss", ["logits", "labels"], ["loss"], ignore_index=-1)]
    return onnx_io.Model(nodes, inits, ["x", "labels"], ["h", "mean", "inv", "logits", "loss"])


def _inputs(dtype, seed):
    rng = np.random.default_rng(seed)
    labels = rng.integers(0, V, B * S)
    labels[::5] = -1
    return {"x": rng.standard_normal((B, S, D)).astype(dtype), "labels": labels}


def _check_trace(prog, ex, trace, eps):
    value = lambda k: trace[k] if k in trace else ex.consts[k]  # noqa: E731
    for i in prog.insts:
        x = [value(k) if k else None for k in i.inputs]
        y = trace[i.outputs[0]]
        if i.op == "Linear":
            b, r = x[2], x[3]
            rows = x[0].reshape(-1, x[0].shape[-1])
            want, bound = _linear64(rows, x[1], None if b is None else b.reshape(-1), i.attrs["activation"], None if r is None else r.reshape(rows.shape[0], -1), i.attrs["residual_first"])
            _check(y.reshape(want.shape), want, bound, repr(i))
        elif i.op == "LayerNormalization":
            v, d = x[0], x[0].shape[-1]
            wy, wm, wi = _norm64(v, x[1], x[2], eps[i.outputs[0]])
            dm = (d + 2) * E32 * v.double().abs().mean(dim=-1, keepdim=True)
            dev = dm + E32 * (v.double().abs().amax(dim=-1, keepdim=True) + wm.abs())
            rel = ((d + 6) * E32 + (dm ** 2 + 2 * dev / wi) * wi ** 2)
            xh = (v.double() - wm) * wi
            _check(y, wy, x[1].double().abs() * (dev * wi + xh.abs() * (rel + EF)) + EF * wy.abs() + E32 * x[2].double().abs() + _u(y.dtype) * 1.001 * wy.abs() + _tiny(y.dtype), repr(i))
            if len(i.outputs) > 1:
                assert trace[i.outputs[1]].shape == v.shape[:-1] + (1,) and trace[i.outputs[1]].dtype == torch.float32
                _check(trace[i.outputs[1]], wm, dm, "mean")
                _check(trace[i.outputs[2]], wi, wi * (rel + EF), "inv_std_dev")
        elif i.op == "SoftmaxCrossEntropyLoss":
            keep = x[1] >= 0
            lp = torch.log_softmax(x[0].double(), dim=1)[keep].gather(1, x[1][keep][:, None])
            # a row: the sum of its exponentials, its logarithm, two subtractions; then the mean over the rows
            row = (x[0].shape[1] + 8) * E32 + EF + 4 * E32 * (x[0].double().abs().amax() + lp.abs().amax())
            want = -lp.mean()
            _check(y, want, row + (len(lp) + 2) * E32 * want.abs() + _u(y.dtype) * 1.001 * want.abs(), "loss")


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_block_of_a_float_graph(mods, dtype):
    onnx_io, _, run_onnx = mods
    model = onnx_io.parse_model(onnx_io.serialize_model(_block(onnx_io, dtype)))
    eps = {"n1": 1e-5, "n2": 1e-3}
    prog = run_onnx.compile_model(model)
    assert [i.op for i in prog.insts] == ["LayerNormalization", "Linear", "Linear", "LayerNormalization", "Reshape", "Linear", "SoftmaxCrossEntropyLoss"]
    ex = run_onnx.Executor(prog, "cuda:0")
    for seed in (0, 1):
        ins = {k: ex.stage(v) for k, v in _inputs(dtype, seed).items()}
        trace = dict(ins)
        ex.run(ins, trace=trace)
        _check_trace(prog, ex, trace, eps)
    plain = run_onnx.compile_model(model, peephole=False)
    ep = run_onnx.Executor(plain, "cuda:0")
    trace = dict(ins)
    ep.run(ins, trace=trace)
    _check_trace(plain, ep, trace, eps)
    # captured, beside the same program run eagerly: same sizes, same bits
    assert ex.is_static()
    ex.capture(_inputs(dtype, 0))
    for seed in (2, 3, 2):
        got = {k: v.clone() for k, v in ex.replay(_inputs(dtype, seed))}
        want = dict(ep.run(_inputs(dtype, seed)) and run_onnx.Executor(prog, "cuda:0").run(_inputs(dtype, seed)))
        assert all(torch.equal(got[k], want[k]) for k in want)


def test_adds_that_broadcast(mods):
    onnx_io, _, run_onnx = mods
    rng = np.random.default_rng(3)
    w, b = rng.standard_normal((6, 4)).astype(np.float32), rng.standard_normal((1, 4)).astype(np.float32)
    N = onnx_io.Node
    for nodes, f in (([N("MatMul", ["x", "w"], ["p"], {}), N("Add", ["p", "r"], ["q"], {}), N("Tanh", ["q"], ["y"], {})], lambda x, r: torch.tanh(x @ torch.from_numpy(w).double() + r)),
                     ([N("MatMul", ["x", "w"], ["p"], {}), N("Relu", ["p"], ["q"], {}), N("Add", ["r", "q"], ["y"], {})], lambda x, r: torch.relu(x @ torch.from_numpy(w).double()) + r),
                     ([N("MatMul", ["x", "w"], ["p"], {}), N("Add", ["p", "b"], ["s"], {}), N("Add", ["s", "r"], ["y"], {})],
                      lambda x, r: x @ torch.from_numpy(w).double() + torch.from_numpy(b).double() + r)):
        prog = run_onnx.compile_model(onnx_io.Model(nodes, {"w": w, "b": b}, ["x", "r"], ["y"]))
        assert [i.op for i in prog.insts] == ["Linear"]
        ex = run_onnx.Executor(prog, "cuda:0")
        for xs, rs in (((5, 6), (5, 4)), ((5, 6), (4,)), ((5, 6), (1, 1)), ((5, 6), (2, 5, 4)), ((6,), (3, 4)), ((6,), (4,)), ((2, 3, 6), (3, 1))):
            x, r = rng.standard_normal(xs).astype(np.float32), rng.standard_normal(rs).astype(np.float32)
            want = f(torch.from_numpy(x).double(), torch.from_numpy(r).double())
            (_, y), = ex.run({"x": x, "r": r})
            mag = torch.from_numpy(np.abs(x)).double() @ torch.from_numpy(np.abs(w)).double() + 4 + torch.from_numpy(np.abs(r)).double()
            assert y.shape == want.shape
            _check(y.cpu(), want, 16 * E32 * mag + EF, (xs, rs))


def test_scale_and_bias_that_broadcast(mods):
    onnx_io, ops, run_onnx = mods
    rng = np.random.default_rng(6)
    x, r = rng.standard_normal((3, 5, 8)).astype(np.float32), lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    for axis, ss, bs in ((-1, (8,), (1, 1, 8)), (1, (8,), (5, 1)), (1, (1, 5, 8), (1,)), (2, (1, 8), ())):
        s, b = r(*ss), r(*bs)
        model = onnx_io.Model([onnx_io.Node("LayerNormalization", ["x", "s", "b"], ["y"], {"axis": axis})], {"s": s, "b": b}, ["x"], ["y"])
        (_, y), = run_onnx.Executor(run_onnx.compile_model(model), "cuda:0").run({"x": x})
        shape = x.shape[axis:]
        full = [torch.from_numpy(np.broadcast_to(v.reshape(v.shape[max(0, v.ndim - len(shape)):]), shape).copy()).cuda() for v in (s, b)]
        assert torch.equal(y, ops.LayerNormalization(torch.from_numpy(x).cuda(), full[0], full[1], axis=axis))


def test_gradient_nodes_run_on_the_operators(mods):
    onnx_io, ops, run_onnx = mods
    rng = np.random.default_rng(4)
    s = rng.standard_normal(40).astype(np.float32)
    N = onnx_io.Node
    nodes = [N("LayerNormalization", ["x", "s", ""], ["n", "mean", "inv"], {}), N("TokenLogProbs", ["n", "tok"], ["lp", "ent", "lse", "tl", "tt"], {"num_top": 3, "ignore_index": 2}),
             N("TokenLogProbsGrad", ["g", "", "n", "tok", "lse"], ["dn"], {"ignore_index": 2}), N("LayerNormalizationGrad", ["dn", "x", "s", "mean", "inv"], ["dx", "ds", "db"], {})]
    outs = ["lp", "ent", "tl", "tt", "dn", "dx", "ds", "db"]
    ex = run_onnx.Executor(run_onnx.compile_model(onnx_io.parse_model(onnx_io.serialize_model(onnx_io.Model(nodes, {"s": s}, ["x", "tok", "g"], outs)))), "cuda:0")
    x, tok, g = rng.standard_normal((9, 40)).astype(np.float32), rng.integers(0, 40, 9), rng.standard_normal(9).astype(np.float32)
    tok[3] = 2
    got = dict(ex.run({"x": x, "tok": tok, "g": g}))
    dx, dt, dg, ds = (torch.from_numpy(v).cuda() for v in (x, tok, g, s))
    n, mean, inv = ops.LayerNormalization(dx, ds, stats=True)
    lp, ent, lse, tl, tt = ops.TokenLogProbs(n, dt, 3, 2)
    dn = ops.TokenLogProbsGrad(dg, None, n, dt, lse, None, 2)
    want = dict(zip(outs, (lp, ent, tl, tt, dn) + tuple(ops.LayerNormalizationGrad(dn, dx, ds, mean, inv))))
    assert all(torch.equal(got[k], want[k]) for k in outs) and float(got["lp"][3]) == 0


def test_most_probable_classes_on_the_command_line(mods, tmp_path, capsys):
    onnx_io, _, run_onnx = mods
    rng = np.random.default_rng(5)
    w, b, x = rng.standard_normal((24, 10)).astype(np.float32), rng.standard_normal(10).astype(np.float32), rng.standard_normal((4, 24)).astype(np.float32)
    N = onnx_io.Node
    model = onnx_io.Model([N("MatMul", ["x", "w"], ["p"], {}), N("Add", ["p", "b"], ["y"], {})], {"w": w, "b": b}, ["x"], ["y"])
    y = x.astype(np.float64) @ w + b
    d, report = str(tmp_path / "t"), str(tmp_path / "r.json")
    onnx_io.write_test_dir(d, model, [({"x": x}, [("y", y.astype(np.float32))])])
    assert run_onnx.run_onnx([d, "--top", "3", "-I", "3", "--cuda_graph", "--report_json", report, "--atol", "1e-5"]) == 0
    rep = json.load(open(report))
    top = rep["outputs"][0]["top"]
    logp = y - np.log(np.exp(y).sum(axis=1, keepdims=True))
    order = np.argsort(-logp, axis=1, kind="stable")[:, :3]
    assert rep["cuda_graph"] and np.array_equal(order, top["indices"])
    assert np.allclose(np.take_along_axis(logp, order, 1), top["logprobs"], rtol=0, atol=1e-4) and np.allclose(logp.max(axis=1), top["expected"], rtol=0, atol=1e-4)
    assert "row 3" in capsys.readouterr().out
    assert run_onnx.run_onnx([d, "--top", "32", "-q", "--no_peephole", "--atol", "1e-5"]) == 0  # no more than there are
