"""Generation with models that norm their heads on the device: over pages of the model's type and of 8 bits, with and without biases."""

import pytest

import test_paged_generation as M
import test_paged_normed as P
from conftest import gpu_available
from irgen.qwen import QwenConfig

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs the GPU")]


@pytest.mark.parametrize("cache", [None, "float8_e4m3fn"])
@pytest.mark.parametrize("layout,bias", [("hnd", True), ("nhd", False)])
def test_likeliest_tokens_in_32_bits_are_the_hosts(backend, layout, bias, cache):
    """The uncached model's tokens to 1e-3, as on the host, and the host's own tokens: sums in another order are off by some 1e-5
    (what lies within that of a border between tokens, or steps of e4m3, would be the exception)."""
    shape = dict(rows=16, slots=4, pages=9, page_size=8, table_pages=5, layout=layout, cache=cache, qkv_bias=bias)
    gen, w = P.generator(P.CFG, **shape, backend=backend)
    ps = M.prompts(P.CFG, [1, 23, 5, 30, 8, 17, 2])
    print(f"[case] float32 {layout} {cache} biases {bias}", flush=True)
    got = gen.generate(ps, 6, P.GREEDY)
    assert max(P.furthest(P.CFG, w, p, new, cache is not None) for p, new in zip(ps, got)) <= 1e-3
    assert got == P.generator(P.CFG, **shape)[0].generate(ps, 6, P.GREEDY)


# Roundings of the activations as counted for the plain step graph: some 12 a layer and 4 after them, here 14 a layer with the
# rotated heads', of a relative half step each; over 8 bits each layer's keys and values take another of at most 2^-4 each.
# They add up like independent ones, to the root of their squares' sum times a logit's spread; a token is off by more than
# four times that of two logits once in 10^4.
@pytest.mark.parametrize("cache", [None, "float8_e4m3fn"])
@pytest.mark.parametrize("dtype,D,layout,half", [("bfloat16", 128, "hnd", 2 ** -8), ("float16", 64, "nhd", 2 ** -11)])
def test_likeliest_tokens_in_16_bits(backend, dtype, D, layout, half, cache):
    cfg = QwenConfig(hidden=512, intermediate=1024, layers=2, heads=4, kv_heads=2, head_dim=D, vocab=8192, dtype=dtype, tie_embeddings=False)
    gen, w = P.generator(cfg, rows=40, slots=6, pages=40, page_size=16, table_pages=12, backend=backend, layout=layout, cache=cache,
                         qkv_bias=False)
    ps = M.prompts(cfg, [1, 70, 33, 5, 150, 2, 40, 16])
    print(f"[case] {dtype} head_dim {D} {layout} {cache}", flush=True)
    got = gen.generate(ps, 9, P.GREEDY)
    off = (32 * half ** 2 + (4 * 2.0 ** -8 if cache else 0)) ** 0.5
    for p, new in zip(ps, got):
        assert len(new) == 9
        spread = float(P.logits64(cfg, w, p + new[:-1], cache is not None)[len(p) - 1:].std())
        assert P.furthest(cfg, w, p, new, cache is not None) <= 4 * 2 ** 0.5 * off * spread
