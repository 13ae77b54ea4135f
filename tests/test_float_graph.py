"""Float products of an ONNX graph as Linear instructions (CPU): what the pass takes into the epilogue, what it leaves, and that the export gives the
nodes back."""
import numpy as np
import pytest

import __graft_entry__ as entry


@pytest.fixture(scope="module")
def mods():
    entry.load_package()
    from chainer_compiler_b200 import onnx_io, run_onnx
    return onnx_io, run_onnx


def _model(onnx_io, nodes, outputs=("y",), inputs=("x", "r"), dtype=np.float32, **more):
    rng = np.random.default_rng(0)
    inits = {"w": rng.standard_normal((6, 4)).astype(dtype), "wt": rng.standard_normal((4, 6)).astype(dtype), "b": rng.standard_normal(4).astype(dtype),
             "b2": rng.standard_normal((1, 4)).astype(dtype), "m": rng.standard_normal((3, 4)).astype(dtype), "s": rng.standard_normal(1).astype(dtype)}
    inits.update(more)
    used = {i for n in nodes for i in n[1]}
    return onnx_io.Model([onnx_io.Node(op, list(i), list(o), a) for op, i, o, a in nodes], {k: v for k, v in inits.items() if k in used}, list(inputs), list(outputs))


MM = ("MatMul", ["x", "w"], ["p"], {})


@pytest.mark.parametrize("nodes,want", [
    ([MM], ("", None, "", False)),
    ([MM, ("Add", ["p", "b"], ["q"], {})], ("b", None, "", False)),
    ([MM, ("Add", ["b2", "p"], ["q"], {}), ("Relu", ["q"], ["u"], {})], ("b2", "Relu", "", False)),
    ([MM, ("Add", ["p", "b"], ["q"], {}), ("Gelu", ["q"], ["u"], {"approximate": "tanh"}), ("Add", ["r", "u"], ["v"], {})], ("b", "GeluTanh", "r", False)),
    ([MM, ("Add", ["p", "r"], ["q"], {}), ("Tanh", ["q"], ["u"], {})], ("", "Tanh", "r", True)),
    ([MM, ("Sigmoid", ["p"], ["g"], {}), ("Mul", ["g", "p"], ["u"], {}), ("Add", ["u", "r"], ["v"], {})], ("", "Swish", "r", False)),
    ([MM, ("Sigmoid", ["p"], ["u"], {})], ("", "Sigmoid", "", False)),
    ([("Gemm", ["x", "w", "b"], ["p"], {}), ("Gelu", ["p"], ["u"], {})], ("b", "Gelu", "", False)),
])
def test_what_a_linear_takes(mods, nodes, want):
    onnx_io, run_onnx = mods
    last = nodes[-1][2][0]
    model = _model(onnx_io, nodes, outputs=(last,))
    prog = run_onnx.compile_model(model)
    (i,) = prog.insts
    assert i.op == "Linear" and i.outputs == [last] and i.inputs[0] == "x"
    assert (i.inputs[2], i.attrs["activation"], i.inputs[3], i.attrs["residual_first"]) == want
    w = prog.constants[i.inputs[1]]
    assert np.array_equal(w, model.initializers["w"].T) and w.flags.c_contiguous and "w" not in prog.constants
    assert run_onnx.infer_dtypes(prog)[last] == "float32"
    out = run_onnx.program_to_onnx(prog)
    assert [repr(n) for n in out.nodes] == [repr(n) for n in model.nodes] and set(out.initializers) == set(model.initializers)
    assert all(np.array_equal(out.initializers[k], v) for k, v in model.initializers.items())
    plain = run_onnx.compile_model(model, peephole=False)  # the product alone
    assert [p.op for p in plain.insts] == ["Linear"] + [n[0] for n in nodes[1:]] and plain.insts[0].inputs[3] == "" and plain.insts[0].attrs["activation"] is None
    assert [p.op for p in run_onnx.compile_model(model, float_linear=False).insts] == [n[0] for n in nodes]


@pytest.mark.parametrize("nodes,outputs,ops", [
    ([MM, ("Add", ["p", "m"], ["q"], {})], ["q"], ["Linear", "Add"]),  # a constant matrix, and one value
    ([MM, ("Add", ["p", "s"], ["q"], {})], ["q"], ["Linear", "Add"]),
    ([MM, ("Add", ["p", "b"], ["q"], {}), ("Relu", ["q"], ["u"], {})], ["q", "u"], ["Linear", "Relu"]),  # read elsewhere
    ([MM, ("Relu", ["p"], ["u"], {}), ("Tanh", ["p"], ["v"], {})], ["u", "v"], ["Linear", "Relu", "Tanh"]),
    ([MM, ("Add", ["p", "p"], ["q"], {})], ["q"], ["Linear", "Add"]),
    ([MM, ("Sigmoid", ["p"], ["g"], {}), ("Mul", ["g", "p"], ["u"], {})], ["g", "u"], ["Linear", "Sigmoid", "Mul"]),
    ([("MatMul", ["x", "r"], ["p"], {})], ["p"], ["MatMul"]),  # two computed operands
    ([("MatMul", ["w", "x"], ["p"], {})], ["p"], ["MatMul"]),
    ([("Gemm", ["x", "wt", "b"], ["p"], {"transB": 1}), ("Relu", ["p"], ["u"], {})], ["u"], ["Gemm", "Relu"]),  # runs as before
    ([("Gemm", ["x", "w", "b"], ["p"], {"alpha": 0.5})], ["p"], ["Gemm"]),
    ([("Gemm", ["x", "w", "s"], ["p"], {})], ["p"], ["Gemm"]),
    ([("Gemm", ["x", "w", "b"], ["p"], {"transA": 1})], ["p"], ["Gemm"]),
    # two products into one Add: one of them takes it, the other is its residual
    ([MM, ("MatMul", ["r", "w"], ["q"], {}), ("Add", ["p", "q"], ["u"], {})], ["u"], ["Linear", "Linear"]),
])
def test_what_a_linear_leaves(mods, nodes, outputs, ops):
    onnx_io, run_onnx = mods
    model = _model(onnx_io, nodes, outputs=outputs)
    prog = run_onnx.compile_model(model)
    assert [i.op for i in prog.insts] == ops
    made = set(prog.inputs) | set(prog.constants) | {""}
    for i in prog.insts:  # in an order that can run
        assert all(v in made for v in i.inputs)
        made.update(i.outputs)
    assert set(outputs) <= made


def test_sixteen_bit_gemm_and_quantized_graphs(mods):
    onnx_io, run_onnx = mods
    model = _model(onnx_io, [("Gemm", ["x", "wt", "b"], ["p"], {"transB": 1}), ("Relu", ["p"], ["u"], {})], outputs=["u"], dtype=np.float16)
    prog = run_onnx.compile_model(model)
    assert [i.op for i in prog.insts] == ["Linear"] and np.array_equal(prog.constants[prog.insts[0].inputs[1]], model.initializers["wt"])
    assert [repr(n) for n in run_onnx.program_to_onnx(prog).nodes] == [repr(n) for n in model.nodes]
    model = _model(onnx_io, [MM, ("Add", ["p", "b"], ["q"], {})], outputs=["q"])
    assert [i.op for i in run_onnx.compile_model(model, quantize=True).insts][-2:] == ["Mul", "Add"]


def test_one_matrix_read_both_ways(mods):
    onnx_io, run_onnx = mods
    rng = np.random.default_rng(1)
    w = rng.standard_normal((4, 4)).astype(np.float16)
    model = onnx_io.Model([onnx_io.Node("MatMul", ["x", "w"], ["p"], {}), onnx_io.Node("Gemm", ["p", "w"], ["q"], {"transB": 1}), onnx_io.Node("MatMul", ["q", "w"], ["y"], {})],
                          {"w": w}, ["x"], ["y"])
    prog = run_onnx.compile_model(model)
    assert [i.op for i in prog.insts] == ["Linear"] * 3
    for i, want in zip(prog.insts, (w.T, w, w.T)):
        assert np.array_equal(prog.constants[i.inputs[1]], want)
    out = run_onnx.program_to_onnx(prog)
    assert [repr(n) for n in out.nodes] == [repr(n) for n in model.nodes] and np.array_equal(out.initializers["w"], w)


def test_types_of_the_new_nodes(mods):
    onnx_io, run_onnx = mods
    nodes = [("LayerNormalization", ["x", "s4", "b4"], ["n", "mean", "inv"], {"axis": -1}), ("TokenLogProbs", ["n", "tok"], ["lp", "ent", "lse", "tl", "tt"], {"num_top": 2}),
             ("TokenLogProbsGrad", ["g", "", "n", "tok", "lse"], ["dn"], {}), ("LayerNormalizationGrad", ["dn", "x", "s4", "mean", "inv"], ["dx", "ds", "db"], {})]
    model = _model(onnx_io, nodes, outputs=["dx"], inputs=("x", "tok", "g"), s4=np.ones(4, np.float16), b4=np.zeros(4, np.float16))
    prog = run_onnx.compile_model(model)
    assert [i.op for i in prog.insts] == [n[0] for n in nodes]
    dt = run_onnx.infer_dtypes(prog)
    assert [dt[k] for k in ("n", "mean", "inv", "lp", "tl", "tt", "dn", "dx", "ds")] == ["float32", "float32", "float32", "float32", "float32", "int64", "float32", "float32", "float16"]


def test_top_is_checked_before_anything_runs(mods):
    _, run_onnx = mods
    for k in ("-1", "33"):
        with pytest.raises(SystemExit):
            run_onnx.run_onnx(["nowhere", "--top", k])
