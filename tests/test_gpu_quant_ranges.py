"""Attention over pages of 8 bits where its tiles are cut into many parts, into parts that hold nothing, or are too short to be
cut, where few rows and many are joined, and over pools of more bytes than 32 bits count.

Tolerances count roundings (``serving_ref``, ``quant_ref``)."""

import pytest
import torch

import quant_ref as Q
import serving_ref as R
from conftest import gpu_available
from test_gpu_quant import E4M3FN, NAMES, _attention
from test_gpu_serving import _dag, _inv, _meta, _rand

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a ROCm GPU")]


@pytest.mark.parametrize("D,dtype,page,H", [(128, "bfloat16", 16, 4), (64, "float16", 64, 3)])
@pytest.mark.parametrize("news,kvs", [([40], [30000]), ([1], [60000]), ([300, 1], [20000, 20000])])
def test_tiles_of_hundreds_of_parts(backend, D, dtype, page, H, news, kvs):
    """One K/V head: a tile's blocks go to hundreds of workgroups or waves, and its rows are joined of as many parts."""
    _attention(backend, R.batch(news, kvs, page, seed=D), H, 1, D, dtype, page)


@pytest.mark.parametrize("D,dtype,page", [(128, "float16", 16), (64, "bfloat16", 32)])
def test_parts_that_hold_nothing(backend, D, dtype, page):
    """Tables far shorter than the lengths: blocks past a table's end are open by position and hold nothing, so whole parts
    of a tile add nothing; a sequence whose table has none at all gives zeros."""
    bt = R.batch([200, 1, 90, 60], [9000, 8000, 500, 700], page, pad=3, seed=4)
    bt["block_table"] = bt["block_table"][:, :6].contiguous()
    bt["block_table"][3] = -1
    got, _ = _attention(backend, bt, 4, 2, D, dtype, page)
    assert (got[291:] == 0).all()


@pytest.mark.parametrize("D,dtype,page", [(128, "bfloat16", 16), (64, "float16", 32)])
@pytest.mark.parametrize("seqs", [150, 400])
def test_many_short_tiles(backend, D, dtype, page, seqs):
    """More wide tiles than workgroups, or nearly as many: ranges of blocks end at tiles' ends."""
    g = torch.Generator().manual_seed(seqs)
    news = torch.randint(1, 12, (seqs,), generator=g).tolist()
    kvs = [n + k for n, k in zip(news, torch.randint(0, 400, (seqs,), generator=g).tolist())]
    _attention(backend, R.batch(news, kvs, page, pad=9, seed=1), 8, 2, D, dtype, page)


@pytest.mark.parametrize("D,dtype,page", [(128, "bfloat16", 16), (64, "float16", 32)])
@pytest.mark.parametrize("seqs", [40, 150, 400])
def test_many_short_wide_tiles(backend, D, dtype, page, seqs):
    """As above with chunks long enough that all but a few take wide tiles, of one to a few blocks."""
    g = torch.Generator().manual_seed(seqs)
    news = torch.randint(1, 50, (seqs,), generator=g).tolist()
    kvs = [n + k for n, k in zip(news, torch.randint(0, 300, (seqs,), generator=g).tolist())]
    _attention(backend, R.batch(news, kvs, page, pad=9, seed=1), 8, 2, D, dtype, page)


@pytest.mark.parametrize("D,dtype,page", [(128, "bfloat16", 16), (64, "float16", 32)])
def test_wide_tiles_over_places_that_do_not_exist(backend, D, dtype, page):
    bt = R.batch([100, 60, 20], [300, 90, 20], page, pad=4)
    bt["block_table"][0, 1], bt["block_table"][0, 5], bt["block_table"][1, 0] = 99999, -7, -1
    bt["kv_len"][2] = 7                              # its first 13 tokens sit before position 0
    got, _ = _attention(backend, bt, 4, 2, D, dtype, page)
    assert (got[160:173] == 0).all() and (got[180:] == 0).all()


@pytest.mark.parametrize("D,dtype,page", [(128, "bfloat16", 16), (64, "float16", 32)])
@pytest.mark.parametrize("starts", [[0, 50, 20, 100], [0, 100, 0, 100]])
def test_many_rows_of_starts_that_descend_give_zeros(backend, D, dtype, page, starts):
    from irgen.serving import build_paged_attention_ir

    bt = R.batch([1, 1, 1], [60, 60, 60], page)
    t = {"q": _rand(1, 101, 4, D, dtype=dtype), **dict(zip(NAMES, Q.pools8(bt, 2, page, D))), **_meta(bt),
         "q_start": torch.tensor(starts, dtype=torch.int32)}
    ir = build_paged_attention_ir(101, 3, bt["pages"], page, bt["block_table"].shape[1], 4, 2, D, dtype, cache=E4M3FN)
    bufs = {k: backend.allocate_buffer(x.cuda()) for k, x in t.items()}
    out = _dag(ir, backend).execute(bufs)[ir["graph_outputs"][0]["name"]].to_torch()
    torch.cuda.synchronize()
    assert out.eq(0).all()


@pytest.mark.parametrize("D,dtype", [(128, "bfloat16"), (64, "float16")])
@pytest.mark.parametrize("N", [63, 64, 65])
def test_joined_by_workgroups_and_by_waves(backend, D, dtype, N):
    """Rows times heads at, below and above the count up to which a workgroup joins a row; rows of no sequence around them."""
    bt = R.batch([1, 30, 1, 20], [900, 1000, 3, 20], 16, pad=N - 54, lead=2, seed=N)
    got, _ = _attention(backend, bt, 4, 2, D, dtype, 16)
    assert got.shape[0] == N and (got[:2] == 0).all() and (got[54:] == 0).all()


@pytest.mark.parametrize("news", [[1, 1], [40, 1]])
def test_pools_of_more_bytes_than_32_bits_count(backend, news):
    """The same batch in pages of a small pool and in the last of a pool of 4.3 GB: equal bits, and nothing else written."""
    from irgen.serving import build_paged_append_ir, build_paged_attention_ir

    D, page, H, KVH, kvs, dtype, P = 128, 64, 16, 8, [300, 129], "bfloat16", 66000
    bt = R.batch(news, kvs, page, seed=3)
    N, M, near = bt["rows"], bt["block_table"].shape[1], bt["pages"]
    small = [p.cuda() for p in Q.pools8(bt, KVH, page, D)]
    large = [torch.zeros(P, *p.shape[1:], dtype=torch.uint8, device="cuda") for p in small]
    for a, b in zip(small, large):
        b[P - near:] = a
    x = {n: _rand(i, N, h, D, dtype=dtype).cuda() for i, (n, h) in enumerate((("q", H), ("k", KVH), ("v", KVH)))}

    def step(pools, table, pages):
        batch = {k: t.cuda() for k, t in _meta(bt).items()} | {"block_table": table.cuda()}
        ir = build_paged_append_ir(N, 2, pages, page, M, H, KVH, D, dtype, cache=E4M3FN)
        bufs = {k: backend.allocate_buffer(t) for k, t in {**x, **dict(zip(NAMES, pools)), **batch, "inv_freq": _inv(D // 2).cuda()}.items()}
        out = _dag(ir, backend).execute(bufs)
        q, *pools = [out[o["name"]].to_torch() for o in ir["graph_outputs"]]
        ir = build_paged_attention_ir(N, 2, pages, page, M, H, KVH, D, dtype, cache=E4M3FN)
        bufs = {k: backend.allocate_buffer(t) for k, t in {"q": q, **dict(zip(NAMES, pools)), **batch}.items()}
        o = _dag(ir, backend).execute(bufs)[ir["graph_outputs"][0]["name"]].to_torch()
        torch.cuda.synchronize()
        return [q, o], pools

    table = bt["block_table"]
    ours, far = step(large, torch.where(table < 0, table, table + P - near).int(), P)
    theirs, by = step(small, table, near)
    assert all(torch.equal(a, b) for a, b in zip(ours, theirs))
    assert all(torch.equal(a[P - near:], b) and not a[:P - near].any() for a, b in zip(far, by))


@pytest.mark.parametrize("D,dtype,page", [(128, "bfloat16", 16), (64, "float16", 32), (80, "bfloat16", 16)])
@pytest.mark.parametrize("news,kvs", [([1, 3, 2], [300, 200, 9]), ([70, 1], [300, 5])])
def test_queries_that_are_no_numbers(backend, D, dtype, page, news, kvs):
    """A NaN or an infinity in a query makes its own row and head NaN (an infinity among scores of both signs); the others are
    right as ever. (Not to the bit: 32 rows of a tile with such an output are done again row by row, whose probabilities keep
    32 bits where a tile's are rounded to 16.)"""
    bt = R.batch(news, kvs, page, seed=6)
    q = _rand(9, bt["rows"], 4, D, dtype=dtype)
    q[0, 1, 3], q[2, 2, 7] = torch.nan, torch.inf
    if bt["rows"] > 60:
        q[50, 0, 5], q[69, 3, 0] = -torch.inf, torch.nan
    clean = q.isfinite().all(-1)
    pools = Q.pools8(bt, 2, page, D)
    got, _ = _attention(backend, bt, 4, 2, D, dtype, page, pools=pools, q=q, rows=clean)
    assert got[~clean].isnan().all()


def test_two_executors_on_two_streams(backend):
    """Each with its own workspaces: calls that overlap give what calls one by one give."""
    from irgen.serving import build_paged_attention_ir

    D, page, H, KVH = 128, 16, 12, 2
    runs = []
    for seed, (news, kvs) in enumerate((([1] * 8, [3000] * 8), ([300, 1], [4000, 900]))):
        bt = R.batch(news, kvs, page, seed=seed)
        t = {"q": _rand(seed, bt["rows"], H, D, dtype="bfloat16"), **dict(zip(NAMES, Q.pools8(bt, KVH, page, D))), **_meta(bt)}
        ir = build_paged_attention_ir(bt["rows"], len(news), bt["pages"], page, bt["block_table"].shape[1], H, KVH, D, cache=E4M3FN)
        bufs = {k: backend.allocate_buffer(x.cuda()) for k, x in t.items()}
        name = ir["graph_outputs"][0]["name"]
        dags = [_dag(ir, backend) for _ in range(2)]
        want = dags[0].execute(bufs)[name].to_torch().clone()
        torch.cuda.synchronize()
        runs += [(d, bufs, name, want, torch.cuda.Stream()) for d in dags]
    for _ in range(5):
        outs = []
        for d, bufs, name, _, stream in runs:
            with torch.cuda.stream(stream):
                outs.append(d.execute(bufs)[name])
        torch.cuda.synchronize()
        assert all(torch.equal(o.to_torch(), w) for o, (*_, w, _) in zip(outs, runs))
