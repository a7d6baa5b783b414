"""Paged operators where batches reach past the tensors, and where a type's range ends, on every kernel path.

Tolerances count roundings (``serving_ref``)."""

import pytest
import torch

import serving_ref as R
from conftest import gpu_available
from test_gpu_serving import _dag, _meta, _rand, _run

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a ROCm GPU")]

LIM = torch.iinfo(torch.int32)


def _calls(backend, ir, tensors, changes):
    """The output of one program on ``tensors``, then with each of ``changes`` made to its inputs."""
    bufs = {k: backend.allocate_buffer(t.cuda()) for k, t in tensors.items()}
    dag, name = _dag(ir, backend), ir["graph_outputs"][0]["name"]
    print(f"[case] {ir['model_name']} {[(i['name'], i['shape'], i['dtype']) for i in ir['graph_inputs'][:1]]}", flush=True)
    outs = []
    for change in ({}, *changes):
        for k, t in change.items():
            bufs[k].native_handle.copy_(t)
        outs.append(dag.execute(bufs)[name].to_torch().cpu().clone())
    return outs


# the paths: both tile widths of the tiled kernels, and the plain kernel
PATHS = [(128, "bfloat16", 16), (64, "float16", 32), (80, "bfloat16", 16), (64, "float32", 16)]


@pytest.mark.parametrize("D,dtype,page", PATHS)
@pytest.mark.parametrize("news,kvs,before,behind", [
    ([4, 1, 40, 3], [30, 9, 300, 8], 2, 20),     # the first sequence begins before the rows, the third ends behind them
    ([6], [6], 0, 2), ([6], [40], 2, 0), ([1, 1, 1], [5, 5, 900], 0, 1),
    ([70, 0, 90], [700, 3, 91], 33, 40),         # long chunks cut at both ends
    ([3, 5], [3, 5], 3, 4)])                     # one row of one sequence
def test_sequences_that_reach_past_the_rows(backend, D, dtype, page, news, kvs, before, behind):
    """The rows that there are, each at its own position; nothing of an earlier call shows. The reference has the
    missing rows too, and is cut."""
    from irgen.serving import build_paged_attention_ir

    H, KVH = 4, 2
    bt = R.batch(news, kvs, page, seed=D)
    kp, vp = R.pools(bt, KVH, page, D, dtype, stale=float("nan"))
    q = _rand(3, bt["rows"], H, D, dtype=dtype)
    out, mag, big = R.attention64(q, kp, vp, bt, page, D ** -0.5)
    pad = 3
    N = bt["rows"] - before - behind + (pad if behind == 0 else 0)
    here = torch.zeros(N, H, D, dtype=q.dtype)
    real = bt["rows"] - before - behind
    here[:real] = q[before:before + real]
    start = (bt["q_start"] - before).to(torch.int32)
    B = len(news)
    ir = build_paged_attention_ir(N, B, bt["pages"], page, bt["block_table"].shape[1], H, KVH, D, dtype)
    valid = {"q": 100 + here, "k_pages": kp, "v_pages": torch.full_like(vp, 100.0), **_meta(bt),
             "q_start": torch.tensor([0] + [N] * B, dtype=torch.int32), "kv_len": torch.full((B,), N, dtype=torch.int32)}
    _, got = _calls(backend, ir, valid, [{"q": here, "v_pages": vp, "q_start": start, "kv_len": bt["kv_len"]}])
    sl = slice(before, before + real)
    tol = R.attention_tol(dtype, D, max(kvs), out[sl], mag[sl], big[sl])
    worst = ((got[:real].double() - out[sl]).abs() / tol).max().item()
    assert worst <= 1.0, worst
    assert got[real:].eq(0).all()


@pytest.mark.parametrize("D,dtype,rows", [(128, "bfloat16", 0), (128, "float16", 1100), (80, "float32", 0)])
def test_appended_sequences_that_reach_past_the_rows(backend, D, dtype, rows):
    """Only the rows that there are rotate and are written, each at its own position. Tolerance as in test_paged_append."""
    from irgen.serving import build_paged_append_ir
    from test_gpu_serving import _inv

    H, KVH, page, before, behind = 4, 2, 16, 2, 20
    bt = R.batch([4, 1, 40 + rows, 3], [30, 9, 300 + rows, 8], page, seed=D)
    kp, vp = R.pools(bt, KVH, page, D, dtype)
    q, k, v = (_rand(i, bt["rows"], h, D, dtype=dtype) for i, h in enumerate((H, KVH, KVH)))
    cut = slice(before, bt["rows"] - behind)
    N = bt["rows"] - before - behind
    ir = build_paged_append_ir(N, 4, bt["pages"], page, bt["block_table"].shape[1], H, KVH, D, dtype)
    got = _run(ir, backend, {"q": q[cut], "k": k[cut], "v": v[cut], "k_pages": kp, "v_pages": vp, **_meta(bt),
                             "q_start": (bt["q_start"] - before).to(torch.int32), "inv_freq": _inv(D // 2)})
    ref = list(R.append64(q, k, v, kp, vp, bt, _inv(D // 2), page))
    ref[0] = ref[0][cut]
    places = R.places(bt, page)
    for row, b, p in places[:before] + places[bt["rows"] - behind:]:   # the missing rows' places stay as they were
        pg, off = R.slot(bt, b, p, page)
        for x, old in ((ref[1], kp), (ref[2], vp)):
            x[pg, :, off] = old[pg, :, off].double().numpy()
    for g, x in zip(got[:2], ref[:2]):
        assert (abs(g.double().numpy() - x) <= 1.001 * R.HALF_STEP[dtype] * abs(x) + 7 * 2.0 ** -24 * 16).all()
    assert (got[2].double().numpy() == ref[2]).all()


@pytest.mark.parametrize("D,dtype,page", PATHS)
def test_starts_and_lengths_at_the_ends_of_int32(backend, D, dtype, page):
    """A row sits at kv_len - (q_start[b + 1] - row), whatever the two are."""
    from irgen.serving import build_paged_attention_ir

    N, H, KVH = 6, 4, 2
    bt = R.batch([N], [4 * page], page)
    kp, vp = R.pools(bt, KVH, page, D, dtype)
    q = _rand(3, N, H, D, dtype=dtype)
    bt["kv_len"][0] = N
    out, mag, big = R.attention64(q, kp, vp, bt, page, D ** -0.5)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)   # noqa: E731
    t = {"q": q, "k_pages": kp, "v_pages": vp, **_meta(bt)}
    ir = build_paged_attention_ir(N, 1, bt["pages"], page, bt["block_table"].shape[1], H, KVH, D, dtype)
    far = [{"q_start": i32(0, LIM.max), "kv_len": i32(LIM.max)},      # row i at position i
           {"q_start": i32(LIM.min, LIM.max), "kv_len": i32(LIM.max)},
           {"q_start": i32(LIM.min, N), "kv_len": i32(N)}]
    none = [{"q_start": i32(0, LIM.max), "kv_len": i32(k)} for k in (LIM.min, -1, 0, 5, LIM.max - N)]
    none += [{"q_start": i32(LIM.min, k), "kv_len": i32(N)} for k in (LIM.min, -5, 0)]
    first, *got = _calls(backend, ir, t, far + none)
    tol = R.attention_tol(dtype, D, N, out, mag, big)
    for g in (first, *got[:len(far)]):
        worst = ((g.double() - out).abs() / tol).max().item()
        assert worst <= 1.0, worst
    for g in got[len(far):]:
        assert g.eq(0).all()


@pytest.mark.parametrize("D,dtype,page", PATHS)
@pytest.mark.parametrize("starts", [[0, 5, 2, 40], [3, 1, 0, 0], [0, 40] * 30 + [0], [9, LIM.min, LIM.max]])
def test_starts_that_descend_are_no_batch_on_any_path(backend, D, dtype, page, starts):
    from irgen.serving import build_paged_attention_ir

    B, N = len(starts) - 1, 41
    t = {"q": _rand(1, N, 4, D, dtype=dtype), "k_pages": _rand(2, 9, 2, page, D, dtype=dtype),
         "v_pages": _rand(3, 9, 2, page, D, dtype=dtype),
         "block_table": torch.arange(B * 4, dtype=torch.int32).view(B, 4) % 9,
         "q_start": torch.tensor([0] + [N] * B, dtype=torch.int32), "kv_len": torch.full((B,), 60, dtype=torch.int32)}
    ir = build_paged_attention_ir(N, B, 9, page, 4, 4, 2, D, dtype)
    before, got = _calls(backend, ir, t, [{"q_start": torch.tensor(starts, dtype=torch.int32)}])
    assert before.ne(0).any() and got.eq(0).all()


def _sink(news, kvs, sink, gap, D, page, H=4, KVH=2):
    """Every score is exact: q picks out one dim of k. Place ``sink`` leads all others by ``gap`` to ``gap`` + 1.5 nats, and
    holds the value 0, so that the output is what the others weigh."""
    bt = R.batch(news, kvs, page, seed=7)
    q = torch.zeros(bt["rows"], H, D, dtype=torch.float16)
    q[:, :, 0] = 1.0
    kp, vp = R.pools(bt, KVH, page, D, "float16")
    kp[..., 1:] = 0
    g = torch.Generator().manual_seed(5)
    kp[..., 0] = (-gap - 1.5 * torch.rand(kp.shape[:-1], generator=g)).to(torch.float16)
    for b in range(len(kvs)):
        pg, off = R.slot(bt, b, sink, page)
        kp[pg, :, off, 0], vp[pg, :, off] = 0.0, 0.0
    vp *= 256   # (the outputs are then no subnormal numbers)
    return bt, q, kp, vp


@pytest.mark.parametrize("gap", [12.0, 14.0, 15.5])
@pytest.mark.parametrize("D,page,news,kvs,sink", [
    (128, 16, [1], [4000], 0), (64, 32, [1, 1], [4000, 900], 0), (128, 16, [1], [4000], 890),   # narrow tiles
    (128, 16, [40], [3000], 0), (64, 32, [70], [2000], 1000)])                                  # wide ones
def test_float16_probabilities_far_below_the_largest(backend, gap, D, page, news, kvs, sink):
    """The probabilities are rounded to float16 for the second product, scaled by 2^7: half a step of each, or 2^-32 of
    the largest where that is more (half of 2^-24, the type's smallest step). Any sequence's largest weighs 1 before
    the division by their sum, which is at least 1."""
    from irgen.serving import build_paged_attention_ir

    bt, q, kp, vp = _sink(news, kvs, sink, gap, D, page)
    ir = build_paged_attention_ir(bt["rows"], len(news), bt["pages"], page, bt["block_table"].shape[1], 4, 2, D, "float16",
                                  scale=1.0)
    got, = _run(ir, backend, {"q": q, "k_pages": kp, "v_pages": vp, **_meta(bt)})
    out, mag, big = R.attention64(q, kp, vp, bt, page, 1.0)
    total = torch.zeros_like(out)   # sum |v| over the open places
    for row, b, p in R.places(bt, page):
        pg, off = zip(*(R.slot(bt, b, j, page) for j in range(p + 1)))
        total[row] = vp[list(pg), :, list(off)].double().abs().sum(0).repeat_interleave(2, 0)
    # the output itself may be subnormal: half of 2^-24
    tol = R.attention_tol("float16", D, max(kvs), out, mag, big) + 2.0 ** -32 * total + 2.0 ** -25
    worst = ((got.double() - out).abs() / tol).max().item()
    assert worst <= 1.0, worst


@pytest.mark.parametrize("D,page", [(128, 16), (64, 32)])
@pytest.mark.parametrize("new,kv,at", [(8, 9000, 8995), (40, 9000, 8980), (40, 9000, 8969)])
def test_float16_parts_done_row_by_row_join_the_others(backend, D, page, new, kv, at):
    """A value that is no number in the last part of a split tile, open to its later rows only: that part is done again
    row by row, and the earlier rows' parts join as if it were not there."""
    from irgen.serving import build_paged_attention_ir

    bt = R.batch([new], [kv], page, seed=1)
    kp, vp = R.pools(bt, 2, page, D, "float16")
    pg, off = R.slot(bt, 0, at, page)
    vp[pg, :, off] = float("nan")
    q = _rand(9, new, 4, D, dtype="float16")
    ir = build_paged_attention_ir(new, 1, bt["pages"], page, bt["block_table"].shape[1], 4, 2, D, "float16")
    got, = _run(ir, backend, {"q": q, "k_pages": kp, "v_pages": vp, **_meta(bt)})
    out, mag, big = R.attention64(q, kp, vp, bt, page, D ** -0.5)
    clean = at - (kv - new)
    assert 0 <= clean < new and got[clean:].isnan().all()
    tol = R.attention_tol("float16", D, kv, out[:clean], mag[:clean], big[:clean])
    worst = ((got[:clean].double() - out[:clean]).abs() / tol).max().item()
    assert worst <= 1.0, worst


@pytest.mark.parametrize("D,dtype", [(64, "bfloat16"), (128, "float16"), (80, "bfloat16")])
@pytest.mark.parametrize("offset", [0, 8, 4, 1])
def test_pools_that_are_ranges_of_an_input(backend, D, dtype, offset):
    from test_serving_edges import _sliced_pools

    bt = R.batch([3], [50], 16)
    bt["block_table"], bt["pages"] = torch.tensor([[2, 0, 3, 1]], dtype=torch.int32), 4
    kp, vp = R.pools(bt, 2, 16, D, dtype)
    q = _rand(9, 3, 4, D, dtype=dtype)
    flat = torch.cat([torch.full((offset,), float("nan"), dtype=kp.dtype), kp.flatten(), vp.flatten()])
    got, = _run(_sliced_pools(offset, D, dtype), backend, {"q": q, "flat": flat, **_meta(bt)})
    out, mag, big = R.attention64(q, kp, vp, bt, 16, D ** -0.5)
    worst = ((got.double() - out).abs() / R.attention_tol(dtype, D, 50, out, mag, big)).max().item()
    assert worst <= 1.0, worst


@pytest.mark.parametrize("D,dtype,page", PATHS)
def test_rows_whose_scores_are_all_negative_infinity(backend, D, dtype, page):
    from irgen.serving import build_paged_attention_ir
    from test_serving_edges import all_infinite

    q, kp, vp, (table, start, kv) = all_infinite(dtype, D, page)
    ir = build_paged_attention_ir(3, 1, kp.shape[0], page, table.shape[1], 4, 2, D, dtype, scale=0.2)
    got, = _run(ir, backend, {"q": q, "k_pages": kp, "v_pages": vp, "block_table": table, "q_start": start, "kv_len": kv})
    assert got[:2].eq(0).all() and torch.equal(got[2], vp[table[0, 0], :, 2].repeat_interleave(2, 0))


@pytest.mark.parametrize("n", [1000, 1025, 2500, 4000])
@pytest.mark.parametrize("B,dtype", [(2, "float32"), (2, "bfloat16"), (90, "float16")])
def test_sample_where_the_tokens_around_a_cut_lie_next_to_each_other(backend, B, dtype, n):
    """All of them in one part of the row, up to the 1,024 that a part lists and past it: the ranking is then from memory."""
    from irgen.serving import build_sample_ir
    from test_gpu_serving import _params

    V, g = 50021, torch.Generator().manual_seed(n)
    x = -40.0 + torch.randn(B, V, generator=g)
    x[:, 9000:9000 + n] = 4.0 + 0.01 * torch.randn(B, n, generator=g)
    x = x.to(R.DT[dtype])
    par = _params(B, n, T=(0.7, 1.0, 1.5), k=(0, n // 2, n - 1), p=(1.0, 0.9, 0.4), m=(0.0, 0.5))
    got, = _run(build_sample_ir(B, V, dtype), backend, {"logits": x, **par})
    assert torch.equal(got, R.sample64(x, **par))


@pytest.mark.parametrize("D,dtype,page", PATHS)
@pytest.mark.parametrize("news,kvs,lead,pad", [([1, 40, 0], [9, 300, 3], 5, 3), ([0, 0], [9, 0], 2, 2), ([0], [40], 0, 1),
                                               ([1], [1], 1, 0), ([33] * 5, [33, 600, 40, 35, 33], 70, 70)])
def test_rows_of_no_sequence_before_and_behind(backend, D, dtype, page, news, kvs, lead, pad):
    from irgen.serving import build_paged_attention_ir

    bt = R.batch(news, kvs, page, pad=pad, lead=lead, seed=2)
    kp, vp = R.pools(bt, 2, page, D, dtype, stale=float("nan"))
    q = _rand(9, bt["rows"], 4, D, dtype=dtype)
    ir = build_paged_attention_ir(bt["rows"], len(news), bt["pages"], page, bt["block_table"].shape[1], 4, 2, D, dtype)
    got, = _run(ir, backend, {"q": q, "k_pages": kp, "v_pages": vp, **_meta(bt)})
    out, mag, big = R.attention64(q, kp, vp, bt, page, D ** -0.5)
    tol = R.attention_tol(dtype, D, max(kvs + [1]), out, mag, big)
    worst = ((got.double() - out).abs() / tol).max().item()
    assert worst <= 1.0, worst
    s = bt["q_start"].tolist()
    assert got[:s[0]].eq(0).all() and got[s[-1]:].eq(0).all()


@pytest.mark.parametrize("D,dtype", [(128, "bfloat16"), (64, "float32")])
@pytest.mark.parametrize("B,M,P", [(0, 3, 4), (2, 0, 4), (2, 3, 0), (0, 0, 0)])
def test_no_sequences_no_table_no_pages(backend, D, dtype, B, M, P):
    """Nothing has a place: attention gives zeros, append rotates the rows of sequences and writes nothing."""
    from irgen.serving import build_paged_append_ir, build_paged_attention_ir
    from npu_runtime.serving_ops import paged_append
    from test_gpu_serving import _inv

    q, k, v = (_rand(i, 3, h, D, dtype=dtype) for i, h in ((1, 4), (2, 2), (3, 2)))
    kp, vp = _rand(4, P, 2, 16, D, dtype=dtype), _rand(5, P, 2, 16, D, dtype=dtype)
    meta = {"block_table": torch.zeros(B, M, dtype=torch.int32), "q_start": torch.tensor([0, 1, 3][:B + 1], dtype=torch.int32),
            "kv_len": torch.full((B,), 20, dtype=torch.int32)}
    got, = _run(build_paged_attention_ir(3, B, P, 16, M, 4, 2, D, dtype), backend, {"q": q, "k_pages": kp, "v_pages": vp, **meta})
    assert got.eq(0).all()
    t = {"q": q, "k": k, "v": v, "k_pages": kp, "v_pages": vp, **meta, "inv_freq": _inv(D // 2)}
    got = _run(build_paged_append_ir(3, B, P, 16, M, 4, 2, D, dtype), backend, t)
    want = paged_append(*t.values())
    assert torch.equal(got[1], kp) and torch.equal(got[2], vp)
    assert ((got[0].double() - want[0].double()).abs() <= 2.01 * R.HALF_STEP[dtype] * want[0].abs().double() + 2.0 ** -20).all()


@pytest.mark.parametrize("D,dtype,page", PATHS)
@pytest.mark.parametrize("scale", [-0.3, 0.0])
def test_negative_and_zero_scales(backend, D, dtype, page, scale):
    from irgen.serving import build_paged_attention_ir

    bt = R.batch([1, 50, 3], [900, 700, 3], page, pad=1, seed=3)
    kp, vp = R.pools(bt, 2, page, D, dtype, stale=float("nan"))
    q = _rand(9, bt["rows"], 4, D, dtype=dtype)
    ir = build_paged_attention_ir(bt["rows"], 3, bt["pages"], page, bt["block_table"].shape[1], 4, 2, D, dtype, scale=scale)
    got, = _run(ir, backend, {"q": q, "k_pages": kp, "v_pages": vp, **_meta(bt)})
    out, mag, big = R.attention64(q, kp, vp, bt, page, scale)
    worst = ((got.double() - out).abs() / R.attention_tol(dtype, D, 900, out, mag, big)).max().item()
    assert worst <= 1.0, worst
