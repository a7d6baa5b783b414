"""The serving operators' definitions (CPU) against plain 64-bit forms, their refusals, and their path through the
IR: builder, exporter, partitioner, compiler and CPU fallback."""

import numpy as np
import pytest
import torch

import serving_ref as R
from hip_compiler import compile_subgraph, is_hip_op_supported
from irgen.builder import IRBuilder
from irgen.exporter import extract_ir
from irgen.serving import build_paged_append_ir, build_paged_attention_ir, build_sample_ir
from npu_compiler import partition
from npu_runtime import DAGExecutor
from npu_runtime.serving_ops import paged_append, paged_attention, sample

# new tokens, cache lengths: one token, several sequences with idle ones among them, none at all
BATCHES = [([1], [1]), ([1, 0, 3, 1], [17, 5, 3, 40]), ([0, 0], [0, 9]), ([7, 2], [7, 34])]


def _inv(r):
    return 1.0 / 1e4 ** (torch.arange(r).float() / max(r, 1))


@pytest.mark.parametrize("news,kvs", BATCHES)
@pytest.mark.parametrize("layout,page,r", [("hnd", 16, 8), ("nhd", 5, 3), ("hnd", 1, 0)])
def test_paged_append_rotates_and_writes_only_its_places(news, kvs, layout, page, r):
    bt = R.batch(news, kvs, page, pad=2, lead=1)
    kp, vp = R.pools(bt, 2, page, 16, "float32", layout)
    q, k, v = (torch.randn(bt["rows"], h, 16, generator=torch.Generator().manual_seed(h)) for h in (6, 2, 2))
    got = paged_append(q, k, v, kp, vp, bt["block_table"], bt["q_start"], bt["kv_len"], _inv(r), 1.5, layout)
    ref = R.append64(q, k, v, kp, vp, bt, _inv(r), page, layout, 1.5)
    for g, x in zip(got, ref):   # three roundings of terms up to 1.5 * 2 * max|x|
        assert np.abs(g.double().numpy() - x).max() <= 4 * 2.0 ** -24 * 1.5 * 2 * 5


@pytest.mark.parametrize("news,kvs", BATCHES)
@pytest.mark.parametrize("layout,page", [("hnd", 16), ("nhd", 5)])
def test_paged_attention_is_causal_over_the_pages_and_reads_no_stale_place(news, kvs, layout, page):
    bt = R.batch(news, kvs, page, pad=2, lead=1)
    kp, vp = R.pools(bt, 2, page, 16, "float32", layout, stale=float("nan"))
    q = torch.randn(bt["rows"], 6, 16, generator=torch.Generator().manual_seed(3))
    got = paged_attention(q, kp, vp, bt["block_table"], bt["q_start"], bt["kv_len"], 0.3, layout)
    out, mag, big = R.attention64(q, kp, vp, bt, page, 0.3, layout)
    assert ((got.double() - out).abs() <= R.attention_tol("float32", 16, max(kvs + [1]), out, mag, big)).all()


def test_places_that_do_not_exist_are_closed():
    bt = R.batch([2, 3], [20, 9], 4, pad=1)
    bt["block_table"][0, 1], bt["block_table"][0, 4] = 99, -5     # positions 4-7 and 16-19
    bt["kv_len"][1] = 2                                           # its first new row sits at position -1
    kp, vp = R.pools(bt, 1, 4, 8, "float32", stale=float("nan"))
    q, k, v = (torch.randn(bt["rows"], h, 8) for h in (2, 1, 1))
    meta = (bt["block_table"], bt["q_start"], bt["kv_len"])
    got = paged_append(q, k, v, kp, vp, *meta, _inv(4))
    ref = R.append64(q, k, v, kp, vp, bt, _inv(4), 4)
    for g, x in zip(got, ref):
        assert np.allclose(g.numpy(), x, atol=1e-5, equal_nan=True)
    out = paged_attention(q, got[1], got[2], *meta, 1.0)
    want, mag, big = R.attention64(q, got[1], got[2], bt, 4, 1.0)
    assert (want[2] == 0).all() and (out[2] == 0).all()           # position -1: no open position
    assert ((out.double() - want).abs() <= R.attention_tol("float32", 8, 20, want, mag, big)).all()


def _params(B, seed, T=(0.0, 0.5, 1.0, 2.0), k=(0, 1, 3, 10, 10 ** 6), p=(1.0, 0.9, 0.3, 0.0, 2.0), m=(0.0, 0.1, 0.9, 1.0)):
    r = np.random.default_rng(seed)
    f = lambda a: torch.tensor(r.choice(np.array(a, np.float32), B))
    return f(T), torch.tensor(r.choice(np.array(k, np.int32), B)), f(p), f(m), torch.tensor(r.random(B, np.float32))


@pytest.mark.parametrize("V,dtype", [(1, "float32"), (7, "bfloat16"), (300, "float32"), (1001, "float16")])
def test_sample_against_a_ranked_walk(V, dtype):
    x = (2.5 * torch.randn(40, V, generator=torch.Generator().manual_seed(V))).to(R.DT[dtype])
    par = _params(40, V)
    assert torch.equal(sample(x, *par), R.sample64(x, *par))


def test_sample_of_special_rows():
    inf, nan = float("inf"), float("nan")
    x = torch.tensor([[-inf, nan, -inf, nan], [nan, 1.0, 1.0, -inf], [inf, 0.0, inf, nan], [-0.0, 0.0, -1.0, 0.0],
                      [2.0, 2.0, 2.0, 2.0], [3.0, -3.4e38, 3.4e38, 0.0]])
    one = torch.ones(6)
    off = torch.zeros(6, dtype=torch.int32)
    at = lambda u, **kw: sample(x, kw.get("T", one), kw.get("k", off), kw.get("p", one), kw.get("m", 0 * one), u * one).tolist()
    assert at(0.0) == [0, 1, 0, 0, 0, 2]
    assert at(0.999) == [0, 2, 2, 3, 3, 2]
    assert at(1.0) == [0, 2, 2, 3, 3, 2]                 # no running sum passes: the last of positive weight
    assert at(0.999, T=0 * one) == [0, 1, 0, 0, 0, 2]    # greedy: -0 equals 0, the lowest index
    assert at(0.999, k=off + 2) == [0, 2, 2, 1, 1, 2]    # ties at the k-th: the lower indices stay
    assert at(0.999, p=0.5 * one) == [0, 1, 0, 1, 1, 2]  # 1 of 2, 2 of 4 equal weights reach a half
    assert at(0.999, p=nan * one, m=nan * one) == [0, 2, 2, 3, 3, 2]
    assert at(nan) == at(-1.0) == at(0.0)
    assert at(0.6, T=inf * one) == [0, 2, 2, 2, 2, 2]


def _meta(**over):
    t = {"q": torch.zeros(3, 4, 16), "k_pages": torch.zeros(5, 2, 8, 16), "v_pages": torch.zeros(5, 2, 8, 16),
         "block_table": torch.zeros(2, 3, dtype=torch.int32), "q_start": torch.zeros(3, dtype=torch.int32),
         "kv_len": torch.zeros(2, dtype=torch.int32)}
    t.update(over)
    return t


@pytest.mark.parametrize("over,what", [
    ({"q": torch.zeros(3, 64)}, "q must be"), ({"q": torch.zeros(3, 3, 16)}, "do not divide"),
    ({"q": torch.zeros(3, 4, 8)}, "head_dim"), ({"q": torch.zeros(3, 4, 16).half()}, "one floating type"),
    ({"v_pages": torch.zeros(5, 2, 4, 16)}, "one 4-dimensional shape"), ({"kv_len": torch.zeros(2)}, "must be int32"),
    ({"q_start": torch.zeros(2, dtype=torch.int32)}, r"q_start \[B \+ 1\]"),
    ({"block_table": torch.zeros(2, 3, dtype=torch.int64)}, "must be int32")])
def test_paged_operands_that_do_not_fit_are_refused(over, what):
    t = _meta(**over)
    for device in ("cpu", "meta"):
        args = [t[k].to(device) for k in ("q", "k_pages", "v_pages", "block_table", "q_start", "kv_len")]
        with pytest.raises(ValueError, match=what):
            torch.ops.serving.paged_attention(*args, 1.0)
        kv = torch.zeros(3, 2, 16, device=device)
        with pytest.raises(ValueError, match=what):
            torch.ops.serving.paged_append(args[0], kv, kv, *args[1:], torch.zeros(8, device=device))


def test_other_refusals():
    t = _meta()
    rest = [t[k] for k in ("k_pages", "v_pages", "block_table", "q_start", "kv_len")]
    kv = torch.zeros(3, 2, 16)
    with pytest.raises(ValueError, match="not one of"):
        torch.ops.serving.paged_attention(t["q"], *rest, 1.0, page_layout="dnh")
    with pytest.raises(ValueError, match="inv_freq"):
        torch.ops.serving.paged_append(t["q"], kv, kv, *rest, torch.zeros(9))
    with pytest.raises(ValueError, match="v must be"):
        torch.ops.serving.paged_append(t["q"], kv, kv[:, :1], *rest, torch.zeros(8))
    with pytest.raises(ValueError, match="non-decreasing"):
        torch.ops.serving.paged_attention(t["q"], *rest[:3], torch.tensor([0, 2, 1], dtype=torch.int32), rest[4], 1.0)
    x, f, i = torch.zeros(2, 9), torch.zeros(2), torch.zeros(2, dtype=torch.int32)
    for bad, what in (((torch.zeros(2, 0), f, i, f, f, f), "vocab > 0"), ((x, f, f, f, f, f), "top_k must be int32"),
                      ((x, f[:1], i, f, f, f), "temperature must be"), ((x, f, i, f, f, f.double()), "u must be float32")):
        with pytest.raises(ValueError, match=what):
            torch.ops.serving.sample(*bad)


def test_the_ops_are_device_ops_and_update_pools_in_place():
    ir = build_paged_append_ir(9, 2, 12, 16, 4, 12, 2, 128)
    assert all(is_hip_op_supported(n["op_type"], n["attrs"]) for n in ir["nodes"])
    prog = compile_subgraph(ir)
    assert sorted(prog.stats["mutated_inputs"]) == ["k_pages", "v_pages"] and len(prog.steps) == 1
    copied = compile_subgraph(ir, inplace_inputs=False)
    assert not copied.stats["mutated_inputs"] and len(copied.steps) == 3
    assert compile_subgraph(build_sample_ir(3, 1000)).steps[-1].kind == "sample"
    with pytest.raises(NotImplementedError, match="vocabulary"):
        compile_subgraph(build_sample_ir(1, 1 << 22))
    with pytest.raises(NotImplementedError, match="head_dim"):
        compile_subgraph(build_paged_attention_ir(1, 1, 4, 16, 4, 2, 1, 512))
    for ir in (build_sample_ir(0, 100), build_paged_attention_ir(0, 1, 4, 16, 4, 2, 1, 64)):   # no rows
        assert all(s.kind == "copy" for s in compile_subgraph(ir).steps)


def test_a_whole_step_runs_in_the_cpu_fallback():
    bt = R.batch([2, 1], [9, 4], 4)
    b = IRBuilder("Step")
    from irgen.serving import batch_inputs, paged_append as append, paged_attention as attend, sampling_inputs

    q, k, v = (b.input(n, [3, h, 8], "float32") for n, h in (("q", 4), ("k", 2), ("v", 2)))
    kp, vp = (b.input(n, [bt["pages"], 2, 4, 8], "float32") for n in ("k_pages", "v_pages"))
    batch = batch_inputs(b, 2, bt["block_table"].shape[1])
    qr, kp2, vp2 = append(b, q, k, v, kp, vp, batch, b.input("inv_freq", [4], "float32"))
    o = attend(b, qr, kp2, vp2, batch, 0.5)
    logits = b.op("aten.reshape.default", [o], {"shape": [3, 32]})
    b.output(kp2, b.op("serving.sample.default", [logits, *sampling_inputs(b, 3)]))
    ir = b.to_dict()
    x = {"q": torch.randn(3, 4, 8), "k": torch.randn(3, 2, 8), "v": torch.randn(3, 2, 8), "inv_freq": _inv(4),
         **dict(zip(("k_pages", "v_pages"), R.pools(bt, 2, 4, 8, "float32"))),
         **{n: bt[n] for n in ("block_table", "q_start", "kv_len")}, "temperature": torch.ones(3),
         "top_k": torch.zeros(3, dtype=torch.int32), "top_p": torch.ones(3), "min_p": torch.zeros(3), "u": torch.rand(3)}
    ex = DAGExecutor(partition(ir, lambda op, attrs=None: False), None)
    ex.load_weights({})
    out = ex.execute({n: t.numpy() for n, t in x.items()})
    meta = [x[n] for n in ("block_table", "q_start", "kv_len")]
    a = paged_append(x["q"], x["k"], x["v"], x["k_pages"], x["v_pages"], *meta, x["inv_freq"])
    want = sample(paged_attention(a[0], a[1], a[2], *meta, 0.5).reshape(3, 32),
                  *(x[n] for n in ("temperature", "top_k", "top_p", "min_p", "u")))
    assert np.array_equal(out[ir["graph_outputs"][0]["name"]], a[1].numpy())
    assert np.array_equal(out[ir["graph_outputs"][1]["name"]], want.numpy())


def test_modules_that_call_the_ops_export():
    class M(torch.nn.Module):
        def forward(self, q, k, v, kp, vp, table, start, kv, inv, u):
            q, kp, vp = torch.ops.serving.paged_append(q, k, v, kp, vp, table, start, kv, inv, page_layout="nhd")
            o = torch.ops.serving.paged_attention(q, kp, vp, table, start, kv, 0.25, page_layout="nhd")
            z = torch.zeros_like(u)
            return torch.ops.serving.sample(o.flatten(1), z + 1, z.to(torch.int32), z + 0.9, z, u), kp, vp

    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    args = (torch.zeros(5, 4, 16), torch.zeros(5, 2, 16), torch.zeros(5, 2, 16), torch.zeros(6, 8, 2, 16),
            torch.zeros(6, 8, 2, 16), i32(2, 3), i32(3), i32(2), torch.zeros(8), torch.zeros(5))
    ir = extract_ir(M(), args, "step")
    ops = [n["op_type"] for n in ir["nodes"]]
    assert [o for o in ops if o.startswith("serving.")] == [
        "serving.paged_append.default", "serving.paged_attention.default", "serving.sample.default"]
    app = next(n for n in ir["nodes"] if "append" in n["op_type"])
    assert app["attrs"]["page_layout"] == "nhd" and len(app["outputs"]) == 3
