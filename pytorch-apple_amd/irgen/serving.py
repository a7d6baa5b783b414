"""IR builders of the serving operators (``npu_runtime.serving_ops``): one-operator graphs, and the nodes that
model graphs are built of.

Graph inputs carry the operators' argument names; the graph outputs are, in order, the operator's results
(``paged_append``: rotated q, k pages, v pages). No counterpart in the reference.
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


def paged_attention(b: IRBuilder, q: T, k_pages: T, v_pages: T, batch: tuple[T, T, T], scale: float,
                    layout: str = "hnd") -> T:
    return b.op("serving.paged_attention.default", [q, k_pages, v_pages, *batch], {"scale": scale, "page_layout": layout})


def _pools(b: IRBuilder, *shape) -> tuple[T, T]:
    *dims, dtype = shape
    return b.input("k_pages", pool_shape(*dims), dtype), b.input("v_pages", pool_shape(*dims), dtype)


def build_paged_append_ir(tokens: int, seqs: int, pages: int, page_size: int, table_pages: int, heads: int,
                          kv_heads: int, head_dim: int, dtype: str = "bfloat16", layout: str = "hnd",
                          rotary_dim: int | None = None, attention_scaling: float = 1.0) -> dict:
    """q [tokens, heads, head_dim] and k rotated, k and v written into the pages (in place on a device)."""
    b = IRBuilder("PagedAppend")
    q = b.input("q", [tokens, heads, head_dim], dtype)
    k = b.input("k", [tokens, kv_heads, head_dim], dtype)
    v = b.input("v", [tokens, kv_heads, head_dim], dtype)
    pools = _pools(b, pages, page_size, kv_heads, head_dim, layout, dtype)
    batch = batch_inputs(b, seqs, table_pages)
    inv = b.input("inv_freq", [(head_dim if rotary_dim is None else rotary_dim) // 2], "float32")
    b.output(*paged_append(b, q, k, v, *pools, batch, inv, layout, attention_scaling))
    return b.to_dict()


def build_paged_attention_ir(tokens: int, seqs: int, pages: int, page_size: int, table_pages: int, heads: int,
                             kv_heads: int, head_dim: int, dtype: str = "bfloat16", layout: str = "hnd",
                             scale: float | None = None) -> dict:
    """Causal attention of q [tokens, heads, head_dim] over the pages; ``scale`` defaults to head_dim ** -0.5."""
    b = IRBuilder("PagedAttention")
    q = b.input("q", [tokens, heads, head_dim], dtype)
    pools = _pools(b, pages, page_size, kv_heads, head_dim, layout, dtype)
    batch = batch_inputs(b, seqs, table_pages)
    b.output(paged_attention(b, q, *pools, batch, head_dim ** -0.5 if scale is None else scale, layout))
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
