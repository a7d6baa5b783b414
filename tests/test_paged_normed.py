"""The step graph of a model that norms its heads, over pages of the model's type and of 8 bits, with and without q, k and v
biases, against an uncached model in 64 bits that norms, rotates, and rounds its cache by itself."""

from dataclasses import replace

import numpy as np
import pytest
import torch

import quant_ref as Q
import test_paged_generation as M
from irgen.qwen import build_paged_ir, inv_freq
from npu_runtime.paged_generation import PagedGenerator, SamplingParams

GREEDY = SamplingParams(temperature=0.0)
CFG = replace(M.CFG, tie_embeddings=False)   # (with the embedding as its own head a model mostly repeats its input)


def weights_of(ir, cfg):
    """``make_weights`` with norms of heads that differ from 1, from each other and from layer to layer, and attention that weighs
    four times as much in a layer's sum."""
    w = M.make_weights(ir, cfg)
    g = torch.Generator().manual_seed(7)
    for name in sorted(w):
        if name.endswith(("q_norm.weight", "k_norm.weight")):
            w[name] = (1 + 0.5 * torch.randn(w[name].shape, generator=g)).to(w[name].dtype)
        if name.endswith("o_proj.weight"):
            w[name] = 4 * w[name]
    return w


def generator(cfg, rows, slots, pages, page_size, table_pages, backend=None, layout="hnd", **kw):
    irs = [build_paged_ir(n, slots, pages, page_size, table_pages, cfg, layout, qk_norm=True, **kw) for n in (rows, slots)]
    w = weights_of(irs[0], cfg)
    dags = [M.executor(ir, w, backend) for ir in irs]
    return PagedGenerator(dags[0], irs[0], dags[1], irs[1], backend=backend), w


def held(x):
    """Heads [T, heads, D] as e4m3 numbers times a power of two each hold them: the smallest power >= 2^-100 under which the
    largest magnitude is at most 448."""
    x = x.numpy()
    s = 2.0 ** np.maximum(np.ceil(np.log2(np.abs(x).max(-1, keepdims=True) / 448)), -100)
    return torch.from_numpy((x / s).astype(np.float32)).to(torch.float8_e4m3fn).double() * torch.from_numpy(s)


def logits64(cfg, weights, tokens, quant, norms="qk", eps=None):
    """Logits [T, vocab] of the whole sequence, in 64 bits. ``norms``: whose weights q and k take."""
    get = lambda name: weights[name].cpu().double()   # noqa: E731
    eps = cfg.eps if eps is None else eps

    def norm(x, name):
        return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + cfg.eps) * get(name)

    T, D = len(tokens), cfg.head_dim
    inv = inv_freq(cfg).double().numpy()
    x = get("model.embed_tokens.weight")[torch.tensor(tokens)]
    mask = torch.full((T, T), float("-inf")).double().triu(1)
    for li in range(cfg.layers):
        pre = f"model.layers.{li}."
        h = norm(x, pre + "input_layernorm.weight")
        q, k, v = (h @ get(f"{pre}self_attn.{n}_proj.weight").T +
                   (get(f"{pre}self_attn.{n}_proj.bias") if f"{pre}self_attn.{n}_proj.bias" in weights else 0) for n in "qkv")
        q, k = (torch.from_numpy(Q.normed(t.view(T, -1, D), get(f"{pre}self_attn.{n}_norm.weight"), eps)) for t, n in zip((q, k), norms))
        q, k = (torch.stack([torch.from_numpy(Q.turned(t[p].numpy(), p, inv, 1.0)[0]) for p in range(T)]) for t in (q, k))
        v = v.view(T, -1, D)
        k, v = (held(t) if quant else t for t in (k, v))
        k, v = (t.repeat_interleave(cfg.heads // cfg.kv_heads, 1) for t in (k, v))
        s = torch.einsum("ihd,jhd->hij", q, k) * D ** -0.5 + mask
        x = x + torch.einsum("hij,jhd->ihd", s.softmax(-1), v).reshape(T, -1) @ get(pre + "self_attn.o_proj.weight").T
        h = norm(x, pre + "post_attention_layernorm.weight")
        g, u = h @ get(pre + "mlp.gate_proj.weight").T, h @ get(pre + "mlp.up_proj.weight").T
        x = x + (torch.nn.functional.silu(g) * u) @ get(pre + "mlp.down_proj.weight").T
    return norm(x, "model.norm.weight") @ get("lm_head.weight").T


def furthest(cfg, weights, prompt, new, quant, **kw):
    """How far below the likeliest a token is, at most."""
    l = logits64(cfg, weights, prompt + new[:-1], quant, **kw)[len(prompt) - 1:]
    return max(float(l[i].max() - l[i, t]) for i, t in enumerate(new))


@pytest.mark.parametrize("cache", [None, "float8_e4m3fn"])
@pytest.mark.parametrize("layout,bias", [("hnd", True), ("nhd", False)])
def test_likeliest_tokens_follow_an_uncached_model(layout, bias, cache):
    """float32 against float64: logits of a few units after 2 layers of sums of 256 to 512 products are off by some 1e-5 (a number
    within that of a border between two steps of e4m3, which takes the other one, would be the exception). With the two norms'
    weights exchanged, or an epsilon of 0.5, the tokens are others'."""
    gen, w = generator(CFG, rows=16, slots=4, pages=9, page_size=8, table_pages=5, layout=layout, cache=cache, qkv_bias=bias)
    assert any(n.endswith("q_proj.bias") for n in w) == bias
    ps = M.prompts(CFG, [1, 23, 5, 30, 8, 17, 2])
    got = gen.generate(ps, 6, GREEDY)
    quant = cache is not None
    assert max(furthest(CFG, w, p, new, quant) for p, new in zip(ps, got)) <= 1e-3
    assert max(furthest(CFG, w, p, new, quant, norms="kq") for p, new in zip(ps, got)) > 1e-2
    assert max(furthest(CFG, w, p, new, quant, eps=0.5) for p, new in zip(ps, got)) > 1e-2


def test_a_graph_without_biases_has_none():
    ir = build_paged_ir(8, 2, 6, 8, 4, M.CFG, qk_norm=True, qkv_bias=False)
    assert not [x["name"] for x in ir["weights"] if x["name"].endswith("bias")]
    assert [x["name"] for x in build_paged_ir(8, 2, 6, 8, 4, M.CFG)["weights"] if x["name"].endswith("bias")]
