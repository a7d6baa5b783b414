"""The serving operators as a server uses them: the paged step graph and its generator on the device."""

import pytest

import test_paged_generation as M
from conftest import gpu_available
from irgen.qwen import QwenConfig

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs the GPU")]


# Rounding of the activations: some 12 a layer and 4 after them, each of a relative half step, add up like independent
# ones to sqrt(28) half steps of a logit's spread; a token is off by more than four times that of two logits once in 10^4.
@pytest.mark.parametrize("dtype,D,layout,half", [("bfloat16", 128, "hnd", 2 ** -8), ("float16", 64, "nhd", 2 ** -11)])
def test_generation_of_a_batch(backend, dtype, D, layout, half):
    from npu_runtime.paged_generation import SamplingParams

    cfg = QwenConfig(hidden=512, intermediate=1024, layers=2, heads=4, kv_heads=2, head_dim=D, vocab=8192, dtype=dtype)
    gen, w = M.generator(cfg, rows=40, slots=6, pages=40, page_size=16, table_pages=12, backend=backend, layout=layout)
    ps = M.prompts(cfg, [1, 70, 33, 5, 150, 2, 40, 16])
    print(f"[case] {dtype} head_dim {D} {layout}: 8 prompts, 9 tokens each", flush=True)
    got = gen.generate(ps, 9, SamplingParams(temperature=0.0))
    for p, new in zip(ps, got):
        assert len(new) == 9
        spread = float(M.logits64(cfg, w, p + new[:-1])[len(p) - 1:].std())
        M.assert_likeliest(cfg, w, p, new, 4 * 2 ** 0.5 * 28 ** 0.5 * half * spread)
    # the same calls again, over pools that hold the last run's tokens
    assert gen.generate(ps, 9, SamplingParams(temperature=0.0)) == got
    par = SamplingParams(temperature=1.1, top_k=40, top_p=0.9, min_p=0.01, seed=11)
    assert gen.generate(ps, 9, par) == gen.generate(ps, 9, par)
    # top_k 1 is the likeliest token whatever else
    assert gen.generate(ps, 9, SamplingParams(temperature=1.5, top_k=1, top_p=0.3)) == got


def test_pools_that_are_not_updated_in_place(backend):
    """A step graph that reads a pool a second time gets a copy of it written: the generator carries it over."""
    from irgen.qwen import build_paged_ir
    from npu_runtime.paged_generation import PagedGenerator, SamplingParams

    cfg = QwenConfig(hidden=256, intermediate=512, layers=1, heads=4, kv_heads=2, head_dim=64, vocab=4096)
    ir = build_paged_ir(24, 3, 20, 16, 6, cfg)
    w = M.make_weights(ir, cfg)
    ps, greedy = M.prompts(cfg, [5, 40, 1]), SamplingParams(temperature=0.0)
    want = PagedGenerator(M.executor(ir, w, backend), ir, backend=backend).generate(ps, 6, greedy)
    pool = next(i for i in ir["graph_inputs"] if i["name"] == "k_pages_0")
    ir["nodes"].append({"name": "twice", "op_type": "aten.add.Tensor", "inputs": [pool, pool], "attrs": {},
                        "outputs": [{**pool, "name": "twice", "producer_node": "twice", "producer_output_idx": 0}]})
    ir["graph_outputs"].append({**pool, "name": "twice"})
    gen = PagedGenerator(M.executor(ir, w, backend), ir, backend=backend)
    assert gen.generate(ps, 6, greedy) == want and gen._moved == {24: [("k_pages_0", ir["graph_outputs"][1]["name"])]}
