"""Paged step graph and generator on the CPU fallback, against an uncached model in 32 bits and against themselves."""

import numpy as np
import pytest
import torch

from irgen.qwen import QwenConfig, build_paged_ir, inv_freq
from irgen.workloads import make_weights

CFG = QwenConfig(hidden=256, intermediate=512, layers=2, heads=4, kv_heads=2, head_dim=64, vocab=1000,
                 rope_theta=1e4, dtype="float32")


def executor(ir, weights, backend=None):
    from npu_compiler import partition
    from npu_runtime import DAGExecutor

    if backend is None:
        dag = DAGExecutor(partition(ir, lambda *a, **k: False), None)
    else:
        from hip_compiler import compile_subgraph, is_hip_op_supported

        dag = DAGExecutor(partition(ir, is_hip_op_supported), backend, compile_fn=compile_subgraph)
    dag.load_weights(weights)
    return dag


def generator(cfg, rows, slots, pages, page_size, table_pages, backend=None, decode=True, layout="hnd", weights=None):
    from npu_runtime.paged_generation import PagedGenerator

    irs = [build_paged_ir(n, slots, pages, page_size, table_pages, cfg, layout) for n in ((rows, slots) if decode else (rows,))]
    weights = make_weights(irs[0], cfg) if weights is None else weights
    dags = [executor(ir, weights, backend) for ir in irs]
    return PagedGenerator(dags[0], irs[0], *((dags[1], irs[1]) if decode else ()), backend=backend), weights


def prompts(cfg, lengths, seed=3):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, cfg.vocab, (n,), generator=g).tolist() for n in lengths]


def logits64(cfg, weights, tokens):
    """Logits [T, vocab] of the whole sequence without a cache, in 64 bits."""
    def get(name):
        w = weights[name]
        w = w if isinstance(w, torch.Tensor) else torch.from_numpy(np.asarray(w))
        return w.cpu().double()

    def norm(x, name):
        return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + cfg.eps) * get(name)

    T, D = len(tokens), cfg.head_dim
    ang = torch.arange(T).double()[:, None] * inv_freq(cfg).double()[None]
    cos, sin = torch.cat([ang.cos()] * 2, -1)[:, None], torch.cat([ang.sin()] * 2, -1)[:, None]
    turn = lambda t: torch.cat([-t[..., D // 2:], t[..., :D // 2]], -1)   # noqa: E731
    rope = lambda t: t * cos + turn(t) * sin   # noqa: E731
    x = get("model.embed_tokens.weight")[torch.tensor(tokens)]
    mask = torch.full((T, T), float("-inf")).double().triu(1)
    for li in range(cfg.layers):
        pre = f"model.layers.{li}."
        h = norm(x, pre + "input_layernorm.weight")
        q, k, v = (h @ get(f"{pre}self_attn.{n}_proj.weight").T + get(f"{pre}self_attn.{n}_proj.bias") for n in "qkv")
        q, k, v = rope(q.view(T, -1, D)), rope(k.view(T, -1, D)), v.view(T, -1, D)
        k, v = (t.repeat_interleave(cfg.heads // cfg.kv_heads, 1) for t in (k, v))
        s = torch.einsum("ihd,jhd->hij", q, k) * D ** -0.5 + mask
        o = torch.einsum("hij,jhd->ihd", s.softmax(-1), v).reshape(T, -1)
        x = x + o @ get(pre + "self_attn.o_proj.weight").T
        h = norm(x, pre + "post_attention_layernorm.weight")
        g, u = h @ get(pre + "mlp.gate_proj.weight").T, h @ get(pre + "mlp.up_proj.weight").T
        x = x + (torch.nn.functional.silu(g) * u) @ get(pre + "mlp.down_proj.weight").T
    return norm(x, "model.norm.weight") @ get("model.embed_tokens.weight").T


def assert_likeliest(cfg, weights, prompt, new, slack):
    """Each token is the likeliest after those before it, or within ``slack`` of it."""
    l = logits64(cfg, weights, prompt + new[:-1])[len(prompt) - 1:]
    for i, t in enumerate(new):
        assert l[i].max() - l[i, t] <= slack, f"token {i}: {t}, {l[i].max() - l[i, t]} below the best"


@pytest.mark.parametrize("layout", ["hnd", "nhd"])
def test_likeliest_tokens_follow_an_uncached_model(layout):
    """Seven prompts through four slots: chunked prompts, steps of both kinds, pages given back and taken again.
    float32 against float64: logits of a few units after 2 layers of sums of 256 to 512 products are off by some 1e-5."""
    from npu_runtime.paged_generation import SamplingParams

    gen, w = generator(CFG, rows=16, slots=4, pages=9, page_size=8, table_pages=5, layout=layout)
    ps = prompts(CFG, [1, 23, 5, 30, 8, 17, 2])
    got = gen.generate(ps, 6, SamplingParams(temperature=0.0))
    for p, new in zip(ps, got):
        assert len(new) == 6
        assert_likeliest(CFG, w, p, new, 1e-3)
    eos = got[1][3]
    cut = gen.generate(ps, 6, SamplingParams(temperature=0.0), eos_token_id=eos)
    assert cut == [t[:t.index(eos)] if eos in t else t for t in got]


def test_sampled_tokens_do_not_depend_on_the_batch():
    """The same request alone, in another batch, by chunks of another size: the same uniform numbers, so the same tokens
    (a border between two tokens within the model's rounding, 1e-5 of the sum, would be the exception)."""
    from npu_runtime.paged_generation import SamplingParams

    ps = prompts(CFG, [13, 4, 29])
    par = [SamplingParams(0.8, 50, 0.9, 0.0, 5), SamplingParams(1.2, 0, 1.0, 0.02, 6), SamplingParams(1.0, 3, 0.5, 0.0, 7)]
    gen, w = generator(CFG, rows=16, slots=4, pages=20, page_size=8, table_pages=5)
    got = gen.generate(ps, 5, par)
    small, _ = generator(CFG, rows=5, slots=1, pages=5, page_size=8, table_pages=5, decode=False, weights=w)
    assert small.generate(ps, 5, par) == got
    assert gen.generate(ps, 5, par) == got
    assert gen.generate(ps[:1], 5, par[:1]) == got[:1]


def test_refusals():
    from npu_runtime.paged_generation import PagedGenerator

    gen, w = generator(CFG, rows=8, slots=2, pages=3, page_size=4, table_pages=4)
    assert gen.generate([], 4) == []
    for bad in (lambda: gen.generate([[]], 4), lambda: gen.generate([[1] * 10], 4), lambda: gen.generate([[1]], 0),
                lambda: gen.generate([[1]], 2, [])):
        with pytest.raises(ValueError):
            bad()
    ir = build_paged_ir(8, 2, 3, 4, 4, CFG)
    other = build_paged_ir(8, 2, 5, 4, 4, CFG)
    few = build_paged_ir(1, 2, 3, 4, 4, CFG)
    with pytest.raises(ValueError, match="pools"):
        PagedGenerator(None, ir, object(), other)
    with pytest.raises(ValueError, match="row"):
        PagedGenerator(None, few)
    from irgen.qwen import build_decode_ir
    with pytest.raises(ValueError, match="paged"):
        PagedGenerator(None, build_decode_ir(16, CFG))


def test_the_step_graph_is_one_program():
    """No part of it falls back to the host."""
    from hip_compiler import is_hip_op_supported
    from npu_compiler import partition

    plan = partition(build_paged_ir(40, 6, 40, 16, 12, QwenConfig(layers=2)), is_hip_op_supported)
    assert [p.target for p in plan.steps] == ["npu"]


def test_the_program_survives_its_file(tmp_path):
    from hip_compiler import compile_subgraph
    from hip_compiler.program_io import load_program, save_program

    prog = compile_subgraph(build_paged_ir(40, 6, 40, 16, 12, QwenConfig(layers=1)))
    save_program(prog, tmp_path / "step.hipbin")
    assert load_program(tmp_path / "step.hipbin") == prog
