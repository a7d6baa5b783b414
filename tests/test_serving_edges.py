"""The serving operators at the edges of what their arguments may be: definitions, refusals and lowering on the CPU."""

import pytest
import torch

import serving_ref as R
from hip_compiler import compile_subgraph
from irgen.serving import build_paged_append_ir, build_paged_attention_ir
from npu_runtime.serving_ops import paged_attention


@pytest.mark.parametrize("news,kvs,before,behind", [([4, 1, 40, 3], [30, 9, 300, 8], 2, 20), ([6], [40], 2, 0),
                                                    ([70, 0, 90], [700, 3, 91], 33, 40)])
def test_sequences_that_reach_past_the_rows(news, kvs, before, behind):
    bt = R.batch(news, kvs, 16, seed=1)
    kp, vp = R.pools(bt, 2, 16, 32, "float32", stale=float("nan"))
    q = torch.randn(bt["rows"], 4, 32, generator=torch.Generator().manual_seed(2))
    cut = slice(before, bt["rows"] - behind)
    out, mag, big = (t[cut] for t in R.attention64(q, kp, vp, bt, 16, 32 ** -0.5))
    got = paged_attention(q[cut], kp, vp, bt["block_table"], bt["q_start"] - before, bt["kv_len"], 32 ** -0.5)
    assert ((got.double() - out).abs() <= R.attention_tol("float32", 32, max(kvs), out, mag, big)).all()


@pytest.mark.parametrize("heads,page,what", [(4, 0, "no position"), (0, 8, "do not divide")])
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
def test_pages_of_no_position_and_no_heads_are_refused(heads, page, what, layout):
    """A kernel would divide by the page size, or be launched over no heads."""
    shape = (5, 2, page, 16) if layout == "hnd" else (5, page, 2, 16)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)   # noqa: E731
    for device in ("cpu", "meta"):
        q, kv, pool = (torch.zeros(s, device=device) for s in ((3, heads, 16), (3, 2, 16), shape))
        meta = [t.to(device) for t in (i32(2, 3), i32(3), i32(2))]
        with pytest.raises(ValueError, match=what):
            torch.ops.serving.paged_attention(q, pool, pool, *meta, 1.0, page_layout=layout)
        with pytest.raises(ValueError, match=what):
            torch.ops.serving.paged_append(q, kv, kv, pool, pool, *meta, torch.zeros(8, device=device), page_layout=layout)
    # (built on a graph that is in order: the builder runs the check as well)
    for build in (build_paged_append_ir, build_paged_attention_ir):
        ir = build(3, 2, 5, 8, 3, 4, 2, 16, "float32", layout)
        for t in [*ir["graph_inputs"], *(t for n in ir["nodes"] for t in [*n["inputs"], *n["outputs"]])]:
            if t["shape"][1:] == list(((5, 2, 8, 16) if layout == "hnd" else (5, 8, 2, 16))[1:]):
                t["shape"] = list(shape)
            elif t["shape"] == [3, 4, 16]:
                t["shape"] = [3, heads, 16]
        with pytest.raises(ValueError, match=what):
            compile_subgraph(ir)


def test_tables_of_positions_past_32_bits_are_refused():
    """The plain kernel's steps over the positions would pass 2^31 - 1, and begin again below 0."""
    pages = lambda M: build_paged_attention_ir(1, 1, 4, 64, M, 2, 1, 16, "float32")   # noqa: E731
    for M in (1 << 25, 1 << 26):
        with pytest.raises(NotImplementedError, match="positions of a table"):
            compile_subgraph(pages(M))
    assert compile_subgraph(pages((1 << 25) - 1)).steps[-1].kernel == "k_paged_attn_any"
    for M in (1 << 25, (1 << 25) - 1):   # (the tiled kernels' counts end before that)
        ir = build_paged_attention_ir(1, 1, 4, 64, M, 2, 1, 64)
        if M == 1 << 25:
            with pytest.raises(NotImplementedError, match="positions of a table"):
                compile_subgraph(ir)
        else:
            assert compile_subgraph(ir).steps[-1].kernel == "k_paged_attn_any"


def _sliced_pools(offset, D, dtype, N=3, page=16, pages=4):
    """Attention over pools that are ranges of one flat input, beginning ``offset`` elements into it."""
    from irgen.builder import IRBuilder
    from irgen.serving import batch_inputs, paged_attention as attend

    b = IRBuilder("Sliced")
    size = pages * 2 * page * D
    q, flat = b.input("q", [N, 4, D], dtype), b.input("flat", [offset + 2 * size], dtype)
    cut = lambda at: b.op("aten.view.default", [b.op("aten.slice.Tensor", [flat], {"dim": 0, "start": at, "end": at + size})],
                          {"size": [pages, 2, page, D]})   # noqa: E731
    batch = batch_inputs(b, 1, pages)
    b.output(attend(b, q, cut(offset), cut(offset + size), batch, D ** -0.5))
    return b.to_dict()


@pytest.mark.parametrize("offset,copies", [(0, 0), (8, 0), (4, 2), (1, 2)])
def test_pools_that_begin_between_pieces_of_an_input_are_copied(offset, copies):
    """The tiled kernels read pools in pieces of 16 bytes; the plain one by elements."""
    steps = compile_subgraph(_sliced_pools(offset, 64, "bfloat16")).steps
    assert [s.kind for s in steps].count("copy") == copies and steps[-1].kernel.startswith("k_paged_combine")
    assert [s.kind for s in compile_subgraph(_sliced_pools(offset, 80, "bfloat16")).steps] == ["paged_attention"]


def test_lengths_at_the_end_of_int32_take_no_memory():
    """A sequence is looked at as far as its table reaches."""
    bt = R.batch([2, 1], [40, 20], 16, extra_pages=0)
    kp, vp = R.pools(bt, 2, 16, 32, "float32")
    q = torch.randn(3, 4, 32, generator=torch.Generator().manual_seed(2))
    ends = torch.full((2,), torch.iinfo(torch.int32).max, dtype=torch.int32)
    bt["block_table"][1] = bt["block_table"][0]
    got = paged_attention(q, kp, vp, bt["block_table"], bt["q_start"], ends, 0.2)
    bt["kv_len"][:] = 48 + 2   # every row behind the table's 48 positions
    out, mag, big = R.attention64(q, kp, vp, bt, 16, 0.2)
    assert ((got.double() - out).abs() <= R.attention_tol("float32", 32, 48, out, mag, big)).all()


def test_rows_whose_scores_are_all_negative_infinity():
    """They have nothing to weigh, as rows without an open position; with one finite score among them it takes all."""
    q, kp, vp, meta = all_infinite("float32", 32, 16)
    got = paged_attention(q, kp, vp, *meta, 0.2)
    assert got[:2].eq(0).all() and torch.equal(got[2], vp[meta[0][0, 0], :, 2].repeat_interleave(2, 0))


def all_infinite(dtype, D, page):
    """Three rows at positions 0, 1 and 2; the keys of 0 and 1 score -inf, that of 2 does not."""
    bt = R.batch([3], [3], page)
    kp, vp = R.pools(bt, 2, page, D, dtype)
    pg = int(bt["block_table"][0, 0])
    kp[pg, :, :2, 0] = float("-inf")
    q = torch.randn(3, 4, D, generator=torch.Generator().manual_seed(2)).abs().to(R.DT[dtype])
    return q, kp, vp, [bt[n] for n in ("block_table", "q_start", "kv_len")]
