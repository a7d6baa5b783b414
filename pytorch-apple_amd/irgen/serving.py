"""IR builders of the serving operators (``npu_runtime.serving_ops``): one-operator graphs, and the nodes that
model graphs are built of.

Graph inputs carry the operators' argument names; the graph outputs are, in order, the operator's results
(``paged_append``: rotated q, k pages, v pages; pages of 8 bits: k scales, v scales behind them). No counterpart in the reference.
"""

from __future__ import annotations

from irgen.builder import IRBuilder, T


def pool_shape(pages: int, page_size: int, kv_heads: int, head_dim: int, layout: str = "hnd") -> list[int]:
    return [pages, kv_heads, page_size, head_dim] if layout == "hnd" else [pages, page_size, kv_heads, head_dim]


def batch_inputs(b: IRBuilder, seqs: int, table_pages: int) -> tuple[T, T, T]:
    """(block_table, q_start, kv_len) graph inputs of a batch of ``seqs`` sequences."""
    return (b.input("block_table", [seqs, table_pages], "int32"), b.input("q_start", [seqs + 1], "int32"),
            b.input("kv_len", [seqs], "int32"))


def paged_append(b: IRBuilder, q: T, k: T, v: T, k_pages: T, v_pages: T, batch: tuple[T, T, T], inv_freq: T,
                 layout: str = "hnd", attention_scaling: float = 1.0) -> tuple[T, T, T]:
    out = b.op("serving.paged_append.default", [q, k, v, k_pages, v_pages, *batch, inv_freq],
               {"attention_scaling": attention_scaling, "page_layout": layout}, n_out=3)
    return b.getitem(out, 0), b.getitem(out, 1), b.getitem(out, 2)


def paged_norm_append(b: IRBuilder, q: T, k: T, v: T, weights: tuple[T, T], eps: float, k_pages: T, v_pages: T,
                      batch: tuple[T, T, T], inv_freq: T, layout: str = "hnd",
                      attention_scaling: float = 1.0) -> tuple[T, T, T]:
    """``paged_append`` with each head of q and k normed first, by ``weights`` (of q, of k)."""
    out = b.op("serving.paged_norm_append.default", [q, k, v, *weights, k_pages, v_pages, *batch, inv_freq],
               {"eps": eps, "attention_scaling": attention_scaling, "page_layout": layout}, n_out=3)
    return tuple(b.getitem(out, i) for i in range(3))


def paged_quant_append(b: IRBuilder, q: T, k: T, v: T, pools: tuple[T, T, T, T], batch: tuple[T, T, T], inv_freq: T,
                       layout: str = "hnd", attention_scaling: float = 1.0, weights: tuple[T, T] | None = None,
                       eps: float = 0.0) -> tuple[T, T, T, T, T]:
    """Append to ``pools`` (k pages, v pages, k scales, v scales) of 8 bits; with ``weights`` each head of q and k is normed
    first. (rotated q, then the pools)"""
    attrs = {"attention_scaling": attention_scaling, "page_layout": layout}
    if weights is None:
        out = b.op("serving.paged_quant_append.default", [q, k, v, *pools, *batch, inv_freq], attrs, n_out=5)
    else:
        out = b.op("serving.paged_norm_quant_append.default", [q, k, v, *weights, *pools, *batch, inv_freq],
                   {"eps": eps, **attrs}, n_out=5)
    return tuple(b.getitem(out, i) for i in range(5))


def paged_attention(b: IRBuilder, q: T, k_pages: T, v_pages: T, batch: tuple[T, T, T], scale: float,
                    layout: str = "hnd") -> T:
    return b.op("serving.paged_attention.default", [q, k_pages, v_pages, *batch], {"scale": scale, "page_layout": layout})


def paged_quant_attention(b: IRBuilder, q: T, pools: tuple[T, T, T, T], batch: tuple[T, T, T], scale: float,
                          layout: str = "hnd") -> T:
    """Attention over ``pools`` (k pages, v pages, k scales, v scales) of 8 bits."""
    return b.op("serving.paged_quant_attention.default", [q, *pools, *batch], {"scale": scale, "page_layout": layout})


CACHES = (None, "float8_e4m3fn")


def cache_inputs(b: IRBuilder, pages: int, page_size: int, kv_heads: int, head_dim: int, layout: str, dtype: str,
                 cache: str | None = None, suffix: str = "") -> tuple[T, ...]:
    """Graph inputs of a K/V cache: k pages and v pages of ``dtype``, or with ``cache`` "float8_e4m3fn" of 8 bits, and then
    their scales too."""
    if cache not in CACHES:
        raise ValueError(f"cache {cache!r} is not one of {CACHES}")
    shape = pool_shape(pages, page_size, kv_heads, head_dim, layout)
    out = tuple(b.input(n + suffix, shape, "uint8" if cache else dtype) for n in ("k_pages", "v_pages"))
    if cache:
        out += tuple(b.input(n + suffix, [pages, kv_heads, page_size], "uint8") for n in ("k_scales", "v_scales"))
    return out


def build_paged_append_ir(tokens: int, seqs: int, pages: int, page_size: int, table_pages: int, heads: int,
                          kv_heads: int, head_dim: int, dtype: str = "bfloat16", layout: str = "hnd",
                          rotary_dim: int | None = None, attention_scaling: float = 1.0, norm_eps: float | None = None,
                          cache: str | None = None) -> dict:
    """q [tokens, heads, head_dim] and k rotated, k and v written into the pages (in place on a device). With ``norm_eps``
    each head of q and k is normed first (inputs ``q_weight``, ``k_weight``); ``cache`` "float8_e4m3fn": pages of 8 bits
    (inputs and outputs ``k_scales``, ``v_scales``)."""
    b = IRBuilder("PagedAppend")
    q = b.input("q", [tokens, heads, head_dim], dtype)
    k = b.input("k", [tokens, kv_heads, head_dim], dtype)
    v = b.input("v", [tokens, kv_heads, head_dim], dtype)
    weights = None if norm_eps is None else tuple(b.input(n, [head_dim], dtype) for n in ("q_weight", "k_weight"))
    pools = cache_inputs(b, pages, page_size, kv_heads, head_dim, layout, dtype, cache)
    batch = batch_inputs(b, seqs, table_pages)
    inv = b.input("inv_freq", [(head_dim if rotary_dim is None else rotary_dim) // 2], "float32")
    b.output(*append(b, q, k, v, pools, batch, inv, layout, attention_scaling, weights, norm_eps))
    return b.to_dict()


def append(b: IRBuilder, q: T, k: T, v: T, pools: tuple[T, ...], batch: tuple[T, T, T], inv_freq: T, layout: str = "hnd",
           attention_scaling: float = 1.0, weights: tuple[T, T] | None = None, eps: float | None = None) -> tuple[T, ...]:
    """The append that ``pools`` (of ``cache_inputs``) and ``weights`` ask for: (rotated q, then the pools)."""
    if len(pools) == 4:
        return paged_quant_append(b, q, k, v, pools, batch, inv_freq, layout, attention_scaling, weights, eps)
    if weights is not None:
        return paged_norm_append(b, q, k, v, weights, eps, *pools, batch, inv_freq, layout, attention_scaling)
    return paged_append(b, q, k, v, *pools, batch, inv_freq, layout, attention_scaling)


def attention(b: IRBuilder, q: T, pools: tuple[T, ...], batch: tuple[T, T, T], scale: float, layout: str = "hnd") -> T:
    """The attention that reads ``pools`` (of ``cache_inputs``)."""
    if len(pools) == 4:
        return paged_quant_attention(b, q, pools, batch, scale, layout)
    return paged_attention(b, q, *pools, batch, scale, layout)


def build_paged_attention_ir(tokens: int, seqs: int, pages: int, page_size: int, table_pages: int, heads: int,
                             kv_heads: int, head_dim: int, dtype: str = "bfloat16", layout: str = "hnd",
                             scale: float | None = None, cache: str | None = None) -> dict:
    """Causal attention of q [tokens, heads, head_dim] over the pages; ``scale`` defaults to head_dim ** -0.5. ``cache``
    "float8_e4m3fn": over pages of 8 bits (inputs ``k_scales``, ``v_scales``)."""
    b = IRBuilder("PagedAttention")
    q = b.input("q", [tokens, heads, head_dim], dtype)
    pools = cache_inputs(b, pages, page_size, kv_heads, head_dim, layout, dtype, cache)
    batch = batch_inputs(b, seqs, table_pages)
    b.output(attention(b, q, pools, batch, head_dim ** -0.5 if scale is None else scale, layout))
    return b.to_dict()


def sampling_inputs(b: IRBuilder, rows: int) -> list[T]:
    return [b.input("temperature", [rows], "float32"), b.input("top_k", [rows], "int32"),
            b.input("top_p", [rows], "float32"), b.input("min_p", [rows], "float32"), b.input("u", [rows], "float32")]


def build_sample_ir(rows: int, vocab: int, dtype: str = "bfloat16") -> dict:
    """One token of each row of logits [rows, vocab], int64 [rows]."""
    b = IRBuilder("Sample")
    x = b.input("logits", [rows, vocab], dtype)
    b.output(b.op("serving.sample.default", [x, *sampling_inputs(b, rows)]))
    return b.to_dict()
