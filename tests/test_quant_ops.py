"""The definitions (CPU) of the appends that norm heads or quantise them and of attention over pages of 8 bits, against 64-bit
forms; their refusals; their path through builder, exporter, compiler, fallback and generator."""

import numpy as np
import pytest
import torch

import quant_ref as Q
import serving_ref as R
import test_paged_generation as M
from hip_compiler import compile_subgraph, is_hip_op_supported
from irgen.exporter import extract_ir
from irgen.qwen import QwenConfig, build_paged_ir
from irgen.serving import build_paged_append_ir, build_paged_attention_ir
from npu_compiler import partition
from npu_runtime import DAGExecutor
from npu_runtime import serving_ops as S

BATCHES = [([1], [1]), ([1, 0, 3, 1], [17, 5, 3, 40]), ([0, 0], [0, 9]), ([7, 2], [7, 34])]
FORMS = [(True, False), (False, True), (True, True)]


def inv(r, theta=1e4):
    return 1.0 / theta ** (torch.arange(r).float() / max(r, 1))


def rand(seed, *shape, dtype="float32"):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(R.DT[dtype])


def call(norm, quant, q, k, v, weights, eps, pools, bt, inv_freq, scaling, layout):
    name = "paged_" + ("norm_" if norm else "") + ("quant_" if quant else "") + "append"
    return getattr(torch.ops.serving, name)(
        q, k, v, *(weights if norm else ()), *pools, bt["block_table"], bt["q_start"], bt["kv_len"], inv_freq,
        *((eps,) if norm else ()), scaling, layout)


def check(got, pools, q, k, v, bt, r, page, D, dtype, layout, scaling, weights, eps):
    rows, at = Q.append64(q, k, v, bt, r, page, scaling, weights, eps)
    Q.check_rows(got[0], rows, dtype, D)
    for i in range(2):
        if len(pools) == 4:
            Q.check_places8(got[1 + i], got[3 + i], pools[i], pools[2 + i], at, i, D, layout)
        else:
            Q.check_places16(got[1 + i], pools[i], at, i, dtype, D, layout)


@pytest.mark.parametrize("news,kvs", BATCHES)
@pytest.mark.parametrize("layout,page,r,dtype", [("hnd", 16, 8, "float32"), ("nhd", 5, 3, "bfloat16"), ("hnd", 1, 0, "float16")])
@pytest.mark.parametrize("norm,quant", FORMS)
def test_appends(norm, quant, layout, page, r, dtype, news, kvs):
    bt = R.batch(news, kvs, page, pad=2, lead=1)
    pools = Q.pools8(bt, 2, page, 16, layout) if quant else tuple(R.pools(bt, 2, page, 16, dtype, layout))
    q, k, v = (rand(h, bt["rows"], h, 16, dtype=dtype) for h in (6, 2, 2))
    weights = (1 + 0.2 * rand(1, 16), 1 + 0.2 * rand(2, 16))
    weights = tuple(w.to(R.DT[dtype]) for w in weights) if norm else None
    got = call(norm, quant, q, k, v, weights, 1e-5, pools, bt, inv(r), 1.5, layout)
    check(got, pools, q, k, v, bt, inv(r), page, 16, dtype, layout, 1.5, weights, 1e-5)


def test_powers_are_the_smallest_that_hold_a_head():
    tops = torch.tensor([448.0, 448.00003, 447.99997, 224.0, 224.00002, 1.75, 1.7500001, 0.0, 1e-45, 2.0 ** -92, 1.76 * 2.0 ** -92,
                         3.4028235e38, 1.0, float("inf"), float("nan")])
    x = torch.zeros(15, 4)
    x[:, 2] = tops
    x[:, 0] = torch.where(tops.isfinite(), -tops / 3, torch.tensor(-2.0))
    b, s = S.quantise(x)
    e = s.int() - 127
    assert e.tolist() == [0, 1, 0, -1, 0, -8, -7, -100, -100, -100, -99, 120, -8, -7, -7]   # (448 2^-100 = 1.75 2^-92)
    y = b.view(torch.float8_e4m3fn).double() * 2.0 ** e[:, None].double()
    fin = x.double()
    half = torch.maximum(Q.E4M3 * fin.abs(), 2.0 ** (e[:, None].double() - 10))
    ok = (y - fin).abs() <= half
    assert ok[:13].all() and ok[13:, [0, 1, 3]].all() and y[13:, 2].isnan().all()
    # the bytes' numbers round to nearest, ties to even
    t = torch.tensor([[448.0, 17, 18, 19, 21, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10]])
    assert S.quantise(t)[0].view(torch.float8_e4m3fn).float().tolist() == [[448.0, 16, 18, 20, 20, 2.0 ** -9, 0.0, 2.0 ** -8]]


@pytest.mark.parametrize("news,kvs", BATCHES)
@pytest.mark.parametrize("layout,page,dtype", [("hnd", 16, "float32"), ("nhd", 5, "bfloat16")])
def test_attention_reads_the_numbers_and_no_stale_place(news, kvs, layout, page, dtype):
    bt = R.batch(news, kvs, page, pad=2, lead=1)
    pools = Q.pools8(bt, 2, page, 16, layout)
    q = rand(3, bt["rows"], 6, 16, dtype=dtype)
    got = S.paged_quant_attention(q, *pools, bt["block_table"], bt["q_start"], bt["kv_len"], 0.3, layout)
    out, mag, big = Q.attention64(q, pools, bt, page, 0.3, layout)
    assert ((got.double() - out).abs() <= R.attention_tol(dtype, 16, max(kvs + [1]), out, mag, big)).all()


def _operands(**over):
    u8, i32 = torch.uint8, torch.int32
    t = {"q": torch.zeros(3, 4, 16), "k": torch.zeros(3, 2, 16), "v": torch.zeros(3, 2, 16), "q_weight": torch.ones(16),
         "k_weight": torch.ones(16), "k_pages": torch.zeros(5, 2, 8, 16, dtype=u8), "v_pages": torch.zeros(5, 2, 8, 16, dtype=u8),
         "k_scales": torch.zeros(5, 2, 8, dtype=u8), "v_scales": torch.zeros(5, 2, 8, dtype=u8),
         "block_table": torch.zeros(2, 3, dtype=i32), "q_start": torch.zeros(3, dtype=i32), "kv_len": torch.zeros(2, dtype=i32),
         "inv_freq": torch.zeros(8)}
    t.update(over)
    return t


CACHE = ("k_pages", "v_pages", "k_scales", "v_scales", "block_table", "q_start", "kv_len")


@pytest.mark.parametrize("over,what", [
    ({"k_pages": torch.zeros(5, 2, 8, 16)}, "k_pages must be uint8"), ({"v_pages": torch.zeros(5, 2, 8, 16).to(torch.int8)}, "v_pages must be uint8"),
    ({"k_scales": torch.zeros(5, 2, 8)}, "k_scales must be uint8"), ({"v_scales": torch.zeros(5, 8, 2, dtype=torch.uint8)}, "v_scales must be"),
    ({"q": torch.zeros(3, 4, 16, dtype=torch.float64)}, "q must be bfloat16"), ({"q": torch.zeros(3, 3, 16)}, "do not divide"),
    ({"kv_len": torch.zeros(2)}, "must be int32"), ({"k_pages": torch.zeros(5, 2, 8, 8, dtype=torch.uint8)}, "one 4-dimensional shape")])
def test_operands_that_do_not_fit_are_refused(over, what):
    t = _operands(**over)
    for device in ("cpu", "meta"):
        x = {k: v.to(device) for k, v in t.items()}
        cache = [x[k] for k in CACHE]
        with pytest.raises(ValueError, match=what):
            torch.ops.serving.paged_quant_attention(x["q"], *cache, 1.0)
        with pytest.raises(ValueError, match=what):
            torch.ops.serving.paged_quant_append(x["q"], x["k"], x["v"], *cache, x["inv_freq"])
        with pytest.raises(ValueError, match=what):
            torch.ops.serving.paged_norm_quant_append(x["q"], x["k"], x["v"], x["q_weight"], x["k_weight"], *cache, x["inv_freq"], 1e-6)


def test_other_refusals():
    t = _operands()
    qkv, cache = [t[k] for k in "qkv"], [t[k] for k in CACHE]
    pools = [torch.zeros(5, 2, 8, 16)] * 2
    append = torch.ops.serving.paged_norm_append
    rest = [*pools, *cache[4:], t["inv_freq"]]
    for weights, eps, what in (((torch.ones(8), t["k_weight"]), 1e-6, "q_weight must be"),
                               ((t["q_weight"], t["k_weight"].half()), 1e-6, "k_weight must be"),
                               ((t["q_weight"], t["k_weight"]), -1.0, "eps")):
        with pytest.raises(ValueError, match=what):
            append(*qkv, *weights, *rest, eps)
    with pytest.raises(ValueError, match="one floating type"):
        append(*qkv, t["q_weight"], t["k_weight"], *cache[:2], *rest[2:], 1e-6)
    with pytest.raises(ValueError, match="not one of"):
        torch.ops.serving.paged_quant_attention(t["q"], *cache, 1.0, page_layout="dnh")
    with pytest.raises(ValueError, match="is not one of"):
        build_paged_attention_ir(1, 1, 4, 16, 4, 2, 1, 64, cache="int8")
    with pytest.raises(ValueError, match="is not one of"):
        build_paged_ir(4, 1, 4, 16, 4, QwenConfig(layers=1), cache="int8")
    with pytest.raises(NotImplementedError, match="head_dim"):
        compile_subgraph(build_paged_attention_ir(1, 1, 4, 16, 4, 2, 1, 512, cache="float8_e4m3fn"))


@pytest.mark.parametrize("norm,quant", FORMS)
def test_the_ops_are_device_ops_and_update_pools_in_place(norm, quant):
    kw = dict(norm_eps=1e-6 if norm else None, cache="float8_e4m3fn" if quant else None)
    ir = build_paged_append_ir(9, 2, 12, 16, 4, 12, 2, 128, **kw)
    assert all(is_hip_op_supported(n["op_type"], n["attrs"]) for n in ir["nodes"])
    prog = compile_subgraph(ir)
    pools = ["k_pages", "k_scales", "v_pages", "v_scales"] if quant else ["k_pages", "v_pages"]
    assert sorted(prog.stats["mutated_inputs"]) == pools and len(prog.steps) == 1
    copied = compile_subgraph(ir, inplace_inputs=False)
    assert not copied.stats["mutated_inputs"] and len(copied.steps) == 1 + len(pools)
    for args in ((0, 1, 4, 16, 4, 2, 1, 64), (3, 1, 4, 16, 4, 2, 1, 64)):
        steps = compile_subgraph(build_paged_attention_ir(*args, cache="float8_e4m3fn")).steps
        assert [s.kind for s in steps if s.kind != "copy"] == (["paged_attention"] * 2 if args[0] else [])


def _kernel(**kw):
    sizes = dict(tokens=9, seqs=2, pages=12, page_size=16, table_pages=4, heads=12, kv_heads=2, head_dim=128, cache="float8_e4m3fn")
    return compile_subgraph(build_paged_append_ir(**{**sizes, **kw})).steps[-1].kernel


def test_which_kernel_takes_an_append():
    assert _kernel() == "k_paged_quant_append_bf16_row"
    assert _kernel(tokens=2000, dtype="float16", norm_eps=0.0) == "k_paged_norm_quant_append_f16"
    assert _kernel(cache=None, norm_eps=0.0) == "k_paged_norm_append_bf16_row"
    assert _kernel(cache=None) == "k_paged_append_bf16_row"
    for odd in ({"dtype": "float32"}, {"head_dim": 72}, {"head_dim": 272}, {"rotary_dim": 24}):
        assert _kernel(**odd) == "k_paged_quant_append_any", odd


def test_modules_that_call_the_ops_export_and_run_on_the_host():
    class Step(torch.nn.Module):
        def forward(self, q, k, v, wq, wk, kp, vp, ks, vs, table, start, kv, inv_freq):
            q, kp, vp, ks, vs = torch.ops.serving.paged_norm_quant_append(q, k, v, wq, wk, kp, vp, ks, vs, table, start, kv,
                                                                          inv_freq, 1e-5, page_layout="nhd")
            return torch.ops.serving.paged_quant_attention(q, kp, vp, ks, vs, table, start, kv, 0.25, page_layout="nhd"), kp, vp, ks, vs

    bt = R.batch([5, 1, 0], [40, 17, 3], 8, pad=2, seed=4)
    args = (rand(1, bt["rows"], 4, 16), rand(2, bt["rows"], 2, 16), rand(3, bt["rows"], 2, 16), 1 + 0.1 * rand(4, 16),
            1 + 0.1 * rand(5, 16), *Q.pools8(bt, 2, 8, 16, "nhd", stale=False),
            *(bt[n] for n in ("block_table", "q_start", "kv_len")), inv(8))
    want = Step()(*(a.clone() for a in args))
    ir = extract_ir(Step(), args, "step")
    assert [n["op_type"] for n in ir["nodes"] if n["op_type"].startswith("serving.")] == [
        "serving.paged_norm_quant_append.default", "serving.paged_quant_attention.default"]
    dag = DAGExecutor(partition(ir, lambda *a, **k: False), None)
    dag.load_weights({})
    got = dag.execute({i["name"]: a.numpy() for i, a in zip(ir["graph_inputs"], args)})
    for o, w in zip(ir["graph_outputs"], want):
        assert np.array_equal(got[o["name"]], w.numpy())


# ---------------------------------------------------------------- the step graph and its generator

def generator(cfg, rows, slots, pages, page_size, table_pages, backend=None, decode=True, layout="hnd", weights=None, **kw):
    from npu_runtime.paged_generation import PagedGenerator

    irs = [build_paged_ir(n, slots, pages, page_size, table_pages, cfg, layout, **kw) for n in ((rows, slots) if decode else (rows,))]
    if weights is None:
        weights = M.make_weights(irs[0], cfg)
    dags = [M.executor(ir, weights, backend) for ir in irs]
    return PagedGenerator(dags[0], irs[0], *((dags[1], irs[1]) if decode else ()), backend=backend), weights


@pytest.mark.parametrize("layout,norm", [("hnd", False), ("nhd", True)])
def test_generation_over_pages_of_8_bits(layout, norm):
    """The same tokens whatever the batch and the chunks: what a position's cache holds depends on its own token alone (up
    to 32-bit sums: 1e-5 of a border between two tokens, or between two steps of e4m3, would be the exception)."""
    from npu_runtime.paged_generation import SamplingParams

    kw = dict(cache="float8_e4m3fn", qk_norm=norm, layout=layout)
    gen, w = generator(M.CFG, rows=16, slots=4, pages=9, page_size=8, table_pages=5, **kw)
    ps = M.prompts(M.CFG, [1, 23, 5, 30, 8, 17, 2])
    greedy = SamplingParams(temperature=0.0)
    got = gen.generate(ps, 6, greedy)
    assert [len(t) for t in got] == [6] * 7
    alone, _ = generator(M.CFG, rows=5, slots=1, pages=5, page_size=8, table_pages=5, decode=False, weights=w, **kw)
    assert alone.generate(ps, 6, greedy) == got
    assert gen.generate(ps, 6, greedy) == got


def test_normed_heads_of_the_step_graph_follow_the_ops():
    """Weights of ones and heads of root mean square 1: the normed graph is the plain one."""
    ir = build_paged_ir(8, 2, 6, 8, 4, M.CFG, qk_norm=True)
    names = {w["name"]: w["shape"] for w in ir["weights"]}
    for li in range(M.CFG.layers):
        assert names[f"model.layers.{li}.self_attn.q_norm.weight"] == [64] == names[f"model.layers.{li}.self_attn.k_norm.weight"]
    ops = [n["op_type"] for n in ir["nodes"] if "append" in n["op_type"]]
    assert ops == ["serving.paged_norm_append.default"] * M.CFG.layers
    both = build_paged_ir(8, 2, 6, 8, 4, M.CFG, qk_norm=True, cache="float8_e4m3fn")
    assert [i["name"] for i in both["graph_inputs"]][-4:] == ["k_pages_1", "v_pages_1", "k_scales_1", "v_scales_1"]
    assert len(both["graph_outputs"]) == 1 + 4 * M.CFG.layers


def test_the_step_graph_is_one_program_that_survives_its_file(tmp_path):
    from hip_compiler.program_io import load_program, save_program

    ir = build_paged_ir(40, 6, 40, 16, 12, QwenConfig(layers=1), qk_norm=True, cache="float8_e4m3fn")
    assert [p.target for p in partition(ir, is_hip_op_supported).steps] == ["npu"]
    prog = compile_subgraph(ir)
    assert sorted(prog.stats["mutated_inputs"]) == ["k_pages_0", "k_scales_0", "v_pages_0", "v_scales_0"]
    save_program(prog, tmp_path / "step.hipbin")
    assert load_program(tmp_path / "step.hipbin") == prog


def test_graphs_of_different_caches_are_refused():
    from npu_runtime.paged_generation import PagedGenerator

    shape = dict(seqs=2, pages=4, page_size=8, table_pages=2, cfg=M.CFG)
    step, decode = build_paged_ir(6, cache="float8_e4m3fn", **shape), build_paged_ir(2, **shape)
    with pytest.raises(ValueError, match="slots and pools"):
        PagedGenerator(object(), step, object(), decode)
