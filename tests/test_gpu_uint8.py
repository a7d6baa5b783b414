"""Bytes and truth values on the device: what the operators around pools of 8 bits make of uint8 tensors, against ATen."""

import pytest
import torch

import quant_ref as Q
import serving_ref as R
from conftest import gpu_available
from test_gpu_serving import _meta, _rand, _run

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a ROCm GPU")]

DT = {"uint8": torch.uint8, "bool": torch.bool, "int32": torch.int32, "int64": torch.int64, "float32": torch.float32,
      "bfloat16": torch.bfloat16}


def _bytes(seed, *shape):
    return torch.randint(0, 256, shape, generator=torch.Generator().manual_seed(seed), dtype=torch.uint8)


def _graph(steps, inputs):
    """``steps``: (op, names of operands, attributes, name of the result); the last result is the graph's output."""
    from irgen.builder import IRBuilder

    b = IRBuilder("Bytes")
    env = {n: b.input(n, list(t.shape), str(t.dtype).replace("torch.", "")) for n, t in inputs.items()}
    for op, names, attrs, out in steps:
        env[out] = b.op(op, [env[n] for n in names], attrs)
    b.output(env[steps[-1][3]])
    return b.to_dict()


X, Y = _bytes(1, 6, 2, 37), _bytes(2, 6, 2, 37)
CHAINS = {
    "clone": ([("aten.clone.default", ["x"], {}, "z")], lambda x, y: x.clone()),
    "add": ([("aten.add.Tensor", ["x", "y"], {}, "z")], lambda x, y: x + y),
    "add a number": ([("aten.add.Tensor", ["x"], {"other": 7}, "z")], lambda x, y: x + 7),
    "sub": ([("aten.sub.Tensor", ["x", "y"], {"alpha": 3}, "z")], lambda x, y: torch.sub(x, y, alpha=3)),
    "mul": ([("aten.mul.Tensor", ["x", "y"], {}, "z")], lambda x, y: x * y),
    "neg": ([("aten.neg.default", ["x"], {}, "z")], lambda x, y: -x),
    "maximum": ([("aten.maximum.default", ["x", "y"], {}, "z")], lambda x, y: torch.maximum(x, y)),
    # every step's result is a byte, also inside a chain
    "sum as a number": ([("aten.add.Tensor", ["x", "y"], {}, "s"), ("aten.to.dtype", ["s"], {"dtype": "float32"}, "z")],
                        lambda x, y: (x + y).float()),
    "product's sum": ([("aten.mul.Tensor", ["x", "y"], {}, "s"), ("aten.to.dtype", ["s"], {"dtype": "int32"}, "t"),
                       ("aten.add.Tensor", ["t"], {"other": 1000}, "z")], lambda x, y: (x * y).int() + 1000),
    "truth as a number": ([("aten.to.dtype", ["x"], {"dtype": "bool"}, "s"), ("aten.to.dtype", ["s"], {"dtype": "int64"}, "t"),
                           ("aten.add.Tensor", ["t", "t"], {}, "z")], lambda x, y: x.bool().long() * 2),
    "truth": ([("aten.to.dtype", ["x"], {"dtype": "bool"}, "z")], lambda x, y: x.bool()),
    "truth's byte": ([("aten.to.dtype", ["x"], {"dtype": "bool"}, "s"), ("aten.to.dtype", ["s"], {"dtype": "uint8"}, "z")],
                     lambda x, y: x.bool().to(torch.uint8)),
}


@pytest.mark.parametrize("name", list(CHAINS))
def test_chains_of_bytes(backend, name):
    steps, want = CHAINS[name]
    x = X.clone()
    x[0, 0, :3] = 0
    used = {"x": x, "y": Y}
    used = {n: t for n, t in used.items() if any(n in s[1] for s in steps)}
    got, = _run(_graph(steps, used), backend, used)
    w = want(x, Y)
    assert got.dtype == w.dtype and torch.equal(got, w)


@pytest.mark.parametrize("src,dst,values", [
    ("int64", "uint8", [0, 1, 127, 255, 256, 300, 511]), ("int32", "uint8", [3, 256, 1000]), ("float32", "uint8", [0.0, 0.9, 1.5, 254.7]),
    ("bfloat16", "uint8", [0.0, 3.0, 200.0]), ("float32", "bool", [0.0, -0.0, 0.25, -0.5, 1e-30, float("nan"), float("inf")]),
    ("int64", "bool", [0, 256, -1, 1 << 40]), ("bool", "uint8", [True, False]), ("uint8", "float32", [0, 200, 255])])
def test_casts_to_and_from_bytes(backend, src, dst, values):
    x = torch.tensor(values).to(DT[src])
    got, = _run(_graph([("aten.to.dtype", ["x"], {"dtype": dst}, "z")], {"x": x}), backend, {"x": x})
    assert torch.equal(got, x.to(DT[dst]))


def test_truth_values_add_to_truth_values(backend):
    x, y = X > 100, Y > 100
    for op, want in (("aten.add.Tensor", x + y), ("aten.mul.Tensor", x * y)):
        got, = _run(_graph([(op, ["x", "y"], {}, "z")], {"x": x, "y": y}), backend, {"x": x, "y": y})
        assert got.dtype == torch.bool and torch.equal(got, want)


@pytest.mark.parametrize("dtype,value", [("uint8", 127), ("uint8", 255), ("uint8", 0), ("bool", True), ("bool", False), ("bool", 0.5),
                                         ("int32", 16777217), ("int32", -5), ("int64", 16777217), ("float32", 1.5)])
def test_tensors_of_one_number(backend, dtype, value):
    from irgen.builder import IRBuilder

    b = IRBuilder("Full")
    x = b.input("x", [1], "float32")
    b.output(b.op("aten.full.default", [], {"size": [5, 7], "fill_value": value, "dtype": dtype}), b.op("aten.neg.default", [x]))
    got, _ = _run(b.to_dict(), backend, {"x": torch.ones(1)})
    want = torch.full((5, 7), value, dtype=DT[dtype])
    assert got.dtype == want.dtype and torch.equal(got, want)


def test_attention_over_a_clone_and_powers_of_one_number(backend):
    """A module that clones its k pages and makes its values' powers with torch.full, exported as one device program."""
    from hip_compiler import is_hip_op_supported
    from irgen.exporter import extract_ir
    from npu_compiler import partition

    class Step(torch.nn.Module):
        def forward(self, q, kp, vp, ks, table, start, kv):
            vs = torch.full((9, 2, 16), 121, dtype=torch.uint8)
            return torch.ops.serving.paged_quant_attention(q, kp.clone(), vp, ks, vs, table, start, kv, 0.125)

    bt = R.batch([5, 1, 0], [60, 17, 3], 16, pad=2, seed=4, spare=2)
    assert bt["pages"] == 9
    kp, vp, ks, vs = Q.pools8(bt, 2, 16, 64, stale=False)
    vs = torch.full_like(vs, 121)
    q = _rand(9, bt["rows"], 4, 64, dtype="bfloat16")
    args = (q, kp, vp, ks, *_meta(bt).values())
    ir = extract_ir(Step(), args, "step")
    assert [s.target for s in partition(ir, is_hip_op_supported).steps] == ["npu"]
    got, = _run(ir, backend, {i["name"]: a for i, a in zip(ir["graph_inputs"], args)})
    out, mag, big = Q.attention64(q, (kp, vp, ks, vs), bt, 16, 0.125)
    assert ((got.double() - out).abs() <= R.attention_tol("bfloat16", 64, 60, out, mag, big)).all()
