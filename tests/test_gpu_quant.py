"""The kernels of the appends that norm heads or quantise them, and of attention over pages of 8 bits, against 64-bit forms
at the sizes, batches and values where they can go wrong.

Tolerances count roundings (``serving_ref``, ``quant_ref``)."""

import pytest
import torch

import quant_ref as Q
import serving_ref as R
import test_quant_ops as C
from conftest import gpu_available
from test_gpu_serving import GPU_BATCHES, _dag, _inv, _meta, _params, _rand, _run

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a ROCm GPU")]

E4M3FN = "float8_e4m3fn"
LIM = torch.iinfo(torch.int32)
NAMES = ("k_pages", "v_pages", "k_scales", "v_scales")


# ---------------------------------------------------------------- append

def _append(backend, bt, H, KVH, D, r, dtype, page, layout, norm, quant, x=None, eps=1e-6, scaling=1.25, change=None):
    from irgen.serving import build_paged_append_ir

    pools = Q.pools8(bt, KVH, page, D, layout) if quant else tuple(R.pools(bt, KVH, page, D, dtype, layout))
    q, k, v = (_rand(i, bt["rows"], h, D, dtype=dtype) for i, h in enumerate((H, KVH, KVH))) if x is None else x
    weights = tuple((1 + 0.3 * _rand(i, D)).to(R.DT[dtype]) for i in (5, 6)) if norm else None
    ir = build_paged_append_ir(bt["rows"], bt["kv_len"].numel(), bt["pages"], page, bt["block_table"].shape[1], H, KVH, D, dtype,
                               layout, rotary_dim=2 * r, attention_scaling=scaling, norm_eps=eps if norm else None,
                               cache=E4M3FN if quant else None)
    t = {"q": q, "k": k, "v": v, **dict(zip(NAMES, pools)), **_meta(bt), "inv_freq": _inv(r), **(change or {})}
    if norm:
        t |= {"q_weight": weights[0], "k_weight": weights[1]}
    return _run(ir, backend, t), pools, (q, k, v), weights


def _check_append(got, pools, qkv, weights, bt, r, page, D, dtype, layout, eps=1e-6, scaling=1.25):
    C.check(got, pools, *qkv, bt, _inv(r), page, D, dtype, layout, scaling, weights, eps)


SHAPES = [(12, 2, 128, 64, "bfloat16", 16, "hnd"), (14, 2, 64, 32, "float16", 32, "nhd"),
          (4, 4, 80, 16, "bfloat16", 48, "hnd"),     # 5 pieces of 16 in 8 lanes, part of the dims rotated
          (2, 1, 256, 128, "float16", 16, "nhd"), (3, 3, 16, 8, "bfloat16", 16, "hnd"), (5, 1, 208, 0, "bfloat16", 16, "hnd"),
          (3, 1, 20, 7, "float16", 5, "nhd"),        # odd everything: the plain kernels
          (4, 2, 16, 0, "float32", 1, "hnd"), (8, 1, 64, 32, "float32", 16, "hnd"), (2, 1, 320, 160, "bfloat16", 16, "hnd")]


@pytest.mark.parametrize("H,KVH,D,r,dtype,page,layout", SHAPES)
@pytest.mark.parametrize("news,kvs", [([1], [1]), ([1, 0, 5, 1], [130000, 5, 9, 64]), ([0, 37], [3, 37])])
@pytest.mark.parametrize("norm,quant", C.FORMS)
def test_append(backend, norm, quant, H, KVH, D, r, dtype, page, layout, news, kvs):
    kvs = [s if s < 1000 else s // 1000 * page for s in kvs] if page < 5 else kvs
    bt = R.batch(news, kvs, page, pad=3, seed=D)
    res = _append(backend, bt, H, KVH, D, r, dtype, page, layout, norm, quant)
    _check_append(*res, bt, r, page, D, dtype, layout)


@pytest.mark.parametrize("norm,quant", C.FORMS)
@pytest.mark.parametrize("H,KVH,D,dtype,layout", [(12, 2, 128, "bfloat16", "hnd"), (14, 2, 64, "float16", "nhd"), (3, 3, 80, "bfloat16", "hnd")])
def test_append_of_many_rows(backend, norm, quant, H, KVH, D, dtype, layout):
    """A wave per row."""
    bt = R.batch([1100, 1, 0, 30], [1300, 7, 2, 30], 16, pad=5, lead=2, seed=D)
    res = _append(backend, bt, H, KVH, D, D // 2, dtype, 16, layout, norm, quant)
    _check_append(*res, bt, D // 2, 16, D, dtype, layout)


@pytest.mark.parametrize("D,dtype", [(128, "bfloat16"), (64, "float16"), (80, "bfloat16"), (24, "float32")])
def test_append_of_special_heads(backend, D, dtype):
    """Heads of zeros, of one number, with infinities and NaN, of the type's largest and of its smallest numbers."""
    bt = R.batch([9], [40], 16)
    top = torch.finfo(R.DT[dtype]).max
    x = []
    for i, h in enumerate((4, 2, 2)):
        t = _rand(i, 9, h, D)
        t[1] = 0
        t[2] = 0
        t[2, :, 3] = -7.3
        t[3, :, 5], t[3, :, D - 2] = float("inf"), float("-inf")
        t[4, 0, 1] = float("nan")
        t[5] *= top / 8
        t[6] = top
        t[7] *= 2.0 ** -14 if dtype == "float16" else 2.0 ** -125
        t[8] *= 2.0 ** -30
        x.append(t.to(R.DT[dtype]))
    x[0] = _rand(0, 9, 4, D, dtype=dtype)   # (q's own: an infinity's rotation is no number)
    r = 0   # unrotated: sums of two of the largest numbers pass the type
    res = _append(backend, bt, 4, 2, D, r, dtype, 16, "hnd", False, True, x=x, scaling=1.0)
    _check_append(*res, bt, r, 16, D, dtype, "hnd", scaling=1.0)


@pytest.mark.parametrize("D,dtype", [(128, "bfloat16"), (64, "float16"), (40, "float32")])
def test_norms_of_small_and_large_heads(backend, D, dtype):
    """eps decides for heads near 0, and a head of zeros stays one."""
    bt = R.batch([5, 1], [30, 2], 16)
    x = [_rand(i, 6, h, D) for i, h in enumerate((4, 2, 2))]
    for t in x:
        t[1], t[2], t[3] = 0, t[2] * 1e-3, t[3] * 1e3
    x = [t.to(R.DT[dtype]) for t in x]
    for quant in (False, True):
        for eps in (1e-6, 0.5):
            res = _append(backend, bt, 4, 2, D, D // 4, dtype, 16, "nhd", True, quant, x=x, eps=eps)
            _check_append(*res, bt, D // 4, 16, D, dtype, "nhd", eps=eps)


@pytest.mark.parametrize("D,dtype", [(128, "bfloat16"), (72, "float16")])
@pytest.mark.parametrize("norm,quant", C.FORMS)
def test_append_of_places_that_do_not_exist(backend, norm, quant, D, dtype):
    bt = R.batch([2, 30, 1, 1], [100, 90, 33, 20], 16, pad=4, lead=3)
    bt["block_table"][0, 6], bt["block_table"][1, 4], bt["block_table"][2, :] = -7, 99999, -1
    bt["kv_len"][3] = 0                              # its new token sits at position -1
    res = _append(backend, bt, 4, 2, D, 8, dtype, 16, "hnd", norm, quant)
    _check_append(*res, bt, 8, 16, D, dtype, "hnd")
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)   # noqa: E731
    for start, kv in (((0, 9, 4, 2, 38), (5, 5, 5, 5)), ((0, 1, 2, 3, 4), (LIM.min, LIM.max, 1 << 30, -1)),
                      ((LIM.min, LIM.min, LIM.max, LIM.max, LIM.max), (3, LIM.max, 7, 9))):
        _append(backend, bt, 4, 2, D, 8, dtype, 16, "hnd", norm, quant, change={"q_start": i32(*start), "kv_len": i32(*kv)})


@pytest.mark.parametrize("norm,quant", C.FORMS)
def test_append_of_strided_rows(backend, norm, quant):
    """q, k, v as column ranges of one projection, and a k whose dims are strided; weights as ranges of one tensor that begin
    between 16-byte pieces."""
    from irgen.builder import IRBuilder
    from irgen.serving import append, batch_inputs, cache_inputs

    H, KVH, D, page = 4, 2, 64, 16
    bt = R.batch([3, 1, 20], [3, 40, 20], page, pad=1)
    N = bt["rows"]
    pools = Q.pools8(bt, KVH, page, D) if quant else tuple(R.pools(bt, KVH, page, D, "bfloat16"))
    y, kt = _rand(5, N, (H + 2 * KVH) * D, dtype="bfloat16"), _rand(6, KVH, D, N, dtype="bfloat16")
    ws = (1 + 0.2 * _rand(7, 2 * D + 3)).to(torch.bfloat16)
    for strided in (False, True):
        b = IRBuilder("AppendStrided")
        yt = b.input("y", list(y.shape), "bfloat16")
        cut = lambda i, j: b.op("aten.view.default", [b.op("aten.slice.Tensor", [yt], {"dim": 1, "start": i * D, "end": j * D})],  # noqa: E731
                                {"size": [N, j - i, D]})
        q, k, v = cut(0, H), cut(H, H + KVH), cut(H + KVH, H + 2 * KVH)
        if strided:
            k = b.op("aten.permute.default", [b.input("kt", list(kt.shape), "bfloat16")], {"dims": [2, 0, 1]})
        weights = None
        if norm:
            wt = b.input("ws", list(ws.shape), "bfloat16")
            weights = tuple(b.op("aten.slice.Tensor", [wt], {"dim": 0, "start": i, "end": i + D}) for i in (1, D + 2))
        caches = cache_inputs(b, bt["pages"], page, KVH, D, "hnd", "bfloat16", E4M3FN if quant else None)
        batch = batch_inputs(b, 3, bt["block_table"].shape[1])
        b.output(*append(b, q, k, v, caches, batch, b.input("inv_freq", [D // 2], "float32"), "hnd", 1.0, weights, 1e-6))
        t = {"y": y, **dict(zip(NAMES, pools)), **_meta(bt), "inv_freq": _inv(D // 2)}
        t |= {"kt": kt} if strided else {}
        t |= {"ws": ws} if norm else {}
        got = _run(b.to_dict(), backend, t)
        q, k, v = (x.reshape(N, -1, D) for x in y.split([H * D, KVH * D, KVH * D], 1))
        k = kt.permute(2, 0, 1) if strided else k
        _check_append(got, pools, (q, k, v), (ws[1:D + 1], ws[D + 2:2 * D + 2]) if norm else None, bt, D // 2, page, D, "bfloat16",
                      "hnd", scaling=1.0)


# ---------------------------------------------------------------- attention

def _attention(backend, bt, H, KVH, D, dtype, page, layout="hnd", scale=None, pools=None, q=None, rows=None):
    """``rows``: those whose reference is a number; the others' outputs are NaN where it is."""
    from irgen.serving import build_paged_attention_ir

    pools = Q.pools8(bt, KVH, page, D, layout) if pools is None else pools
    q = _rand(9, bt["rows"], H, D, dtype=dtype) if q is None else q
    ir = build_paged_attention_ir(bt["rows"], bt["kv_len"].numel(), bt["pages"], page, bt["block_table"].shape[1], H, KVH, D, dtype,
                                  layout, scale, cache=E4M3FN)
    got, = _run(ir, backend, {"q": q, **dict(zip(NAMES, pools)), **_meta(bt)})
    scale = D ** -0.5 if scale is None else scale
    out, mag, big = Q.attention64(q, pools, bt, page, scale, layout)
    rows = slice(None) if rows is None else rows
    S = int(bt["kv_len"].max()) if bt["kv_len"].numel() else 1
    tol = Q.attention_tol(dtype, D, S, out, mag, big, q, pools, bt, page, layout)[rows]
    assert torch.isfinite(got[rows].float()).all()
    worst = ((got[rows].double() - out[rows]).abs() / tol).max().item() if got.numel() else 0.0
    assert worst <= 1.0, worst
    return got, out


PATHS = [(128, "bfloat16", 16), (64, "float16", 32), (128, "float16", 48), (64, "bfloat16", 16), (80, "bfloat16", 16), (64, "float32", 16)]


@pytest.mark.parametrize("H,KVH,D,dtype,page,layout", [
    (12, 2, 128, "bfloat16", 16, "hnd"), (14, 2, 64, "float16", 32, "nhd"), (8, 8, 128, "bfloat16", 48, "nhd"),
    (16, 1, 128, "float16", 64, "hnd"), (40, 8, 64, "bfloat16", 128, "hnd"), (17, 1, 64, "bfloat16", 16, "hnd"),
    (6, 2, 80, "bfloat16", 16, "hnd"), (4, 2, 128, "bfloat16", 20, "hnd"), (4, 2, 64, "float32", 16, "nhd"),
    (2, 1, 256, "float16", 16, "hnd"), (3, 3, 20, "float16", 3, "hnd")])
@pytest.mark.parametrize("news,kvs", GPU_BATCHES)
def test_attention(backend, H, KVH, D, dtype, page, layout, news, kvs):
    _attention(backend, R.batch(news, kvs, page, pad=2, seed=D + page), H, KVH, D, dtype, page, layout)


@pytest.mark.parametrize("H,KVH,D,page,dtype", [(12, 2, 128, 16, "bfloat16"), (4, 4, 64, 32, "float16"), (8, 1, 128, 48, "float16")])
@pytest.mark.parametrize("new,kv", [(40, 3958), (70, 2040), (1, 9000), (2, 4095), (300, 5000)])
def test_attention_of_long_tiles(backend, H, KVH, D, page, dtype, new, kv):
    """Tiles split along their positions: parts that begin at the last block of a window of page ids, and at every other."""
    _attention(backend, R.batch([new, 1], [kv, 77], page, seed=new), H, KVH, D, dtype, page)


@pytest.mark.parametrize("D,dtype,page", PATHS)
def test_attention_of_places_that_do_not_exist(backend, D, dtype, page):
    bt = R.batch([2, 30, 1, 1], [6 * page + 4, 90, 33, 20], page, pad=4)
    bt["block_table"][0, 1], bt["block_table"][0, 6], bt["block_table"][1, 0] = 99999, -7, -1
    bt["block_table"][2, :] = -1                     # a sequence without one page that exists
    bt["kv_len"][3] = 0                              # its new token sits at position -1
    got, _ = _attention(backend, bt, 4, 2, D, dtype, page, pools=Q.pools8(bt, 2, page, D))
    assert (got[32:] == 0).all()


@pytest.mark.parametrize("what", ["number", "power"])
@pytest.mark.parametrize("D,dtype,page", PATHS)
def test_attention_of_nan_places_behind_a_row(backend, D, dtype, page, what):
    """What a later position holds does not enter an earlier row, also where one tile takes both; the rows that have it
    open are NaN."""
    bt = R.batch([60, 1], [130, 70], page)
    pools = Q.pools8(bt, 2, page, D)
    for p in (100, 117):   # rows 30 and 47 of the first sequence
        pg, off = R.slot(bt, 0, p, page)
        for i in (0, 1):
            if what == "number":
                pools[i][pg, :, off, 5] = 0xff
            else:
                pools[2 + i][pg, :, off] = 255
    clean = torch.ones(61, dtype=torch.bool)
    clean[30:60] = False
    got, out = _attention(backend, bt, 4, 2, D, dtype, page, pools=pools, rows=clean)
    assert got[30:60].isnan().any(-1).all() and out[30:60].isnan().any(-1).all()


@pytest.mark.parametrize("D,dtype,page", PATHS)
@pytest.mark.parametrize("news,kvs", [([1, 3], [300, 200]), ([150], [300])])
@pytest.mark.parametrize("which", ["k", "v", "both"])
def test_attention_of_powers_far_apart(backend, D, dtype, page, which, news, kvs):
    """Powers of 2^-30 to 2^12 in one head: keys past float16 where they are large, values that differ by 2^20 under weights
    that make up for it. Scores are kept in range by the scale; outputs past float16 are what float16 makes of them."""
    bt = R.batch(news, kvs, page, seed=3)
    kp, vp, ks, vs = Q.pools8(bt, 2, page, D, stale=False)
    g = torch.Generator().manual_seed(8)
    if which != "v":
        ks = torch.randint(97, 140, ks.shape, generator=g).to(torch.uint8)
    if which != "k":
        vs = torch.randint(97, 132, vs.shape, generator=g).to(torch.uint8)
    q = _rand(9, bt["rows"], 4, D, dtype=dtype)
    _attention(backend, bt, 4, 2, D, dtype, page, pools=(kp, vp, ks, vs), q=q, scale=2.0 ** -18 if which != "v" else None)


@pytest.mark.parametrize("D,page", [(128, 16), (64, 32), (80, 16)])
def test_attention_of_powers_at_the_ends(backend, D, page):
    """bfloat16 over numbers from 2^-126 to near its largest: exact powers all the way (row by row below 2^-100 and past 2^119).
    A byte of 0 stands for 0. (Numbers times powers, and their products with q before the scale, are 32-bit numbers by the
    definition: under 2^120 the numbers are subnormal ones, at most 7 2^-9, since 448 2^120 is none.)"""
    bt = R.batch([1, 40], [100, 200], page, seed=3)
    kp, vp, ks, vs = Q.pools8(bt, 2, page, D, stale=False)
    q = _rand(9, bt["rows"], 4, D, dtype="bfloat16")
    for kb, vb, scale in ((1, 1, 1e30), (27, 28, 1e25), (0, 60, 1.0), (127, 0, 1.0), (26, 26, 1e25), (230, 127, 2.0 ** -113), (240, 240, 2.0 ** -123), (127, 245, None), (247, 100, 2.0 ** -113)):
        pools = (kp, vp, torch.full_like(ks, kb), torch.full_like(vs, vb))
        if vb > 230:   # (numbers up to 32: sums of a few hundred stay below 2^128)
            pools = (kp, ((vp & 0x80) | (vp & 0x7f).clamp(max=0x60)), *pools[2:])
        if kb > 240:
            pools = (kp & 0x87, *pools[1:])
        _attention(backend, bt, 4, 2, D, "bfloat16", page, pools=pools, q=q, scale=scale)


@pytest.mark.parametrize("D,dtype,page", PATHS)
def test_attention_of_large_scores(backend, D, dtype, page):
    """Scores of a few hundred: one position takes nearly all, and exponentials of the others underflow."""
    bt = R.batch([40, 1], [200, 333], page)
    q = 8 * _rand(9, bt["rows"], 4, D, dtype=dtype)
    _attention(backend, bt, 4, 2, D, dtype, page, scale=2.0, q=q)


@pytest.mark.parametrize("gap", [12.0, 20.0, 30.0])
@pytest.mark.parametrize("D,dtype,page", PATHS)
def test_attention_of_probabilities_far_below_the_largest(backend, D, dtype, page, gap):
    """One position scores ``gap`` nats above all others and has a value of zero: the outputs are the others'."""
    bt = R.batch([1, 50], [600, 300], page, seed=5)
    kp, vp, ks, vs = Q.pools8(bt, 2, page, D, stale=False, powers=(121, 122))
    q = torch.ones(bt["rows"], 4, D, dtype=R.DT[dtype])
    kp[:] = 0
    for b in (0, 1):
        pg, off = R.slot(bt, b, 40, page)
        kp[pg, :, off], vp[pg, :, off], ks[pg, :, off] = 0x38, 0, 127   # ones
    _attention(backend, bt, 4, 2, D, dtype, page, pools=(kp, vp, ks, vs), q=q, scale=gap / D)


@pytest.mark.parametrize("D,dtype,page", PATHS)
@pytest.mark.parametrize("scale", [-0.1, 0.0])
def test_negative_and_zero_scales(backend, D, dtype, page, scale):
    _attention(backend, R.batch([1, 70, 3], [90, 100, 40], page), 4, 2, D, dtype, page, scale=scale)


@pytest.mark.parametrize("D,dtype,page", [(128, "bfloat16", 1), (80, "float16", 7), (64, "bfloat16", 24), (48, "float32", 16), (1, "float32", 3)])
def test_attention_of_other_pages_and_heads(backend, D, dtype, page):
    _attention(backend, R.batch([1, 0, 5, 33, 0, 1], [1, 0, 5, 70, 9, 130], page, pad=3, seed=D), 6, 2, D, dtype, page, "nhd")


@pytest.mark.parametrize("seqs", [1000, 1100])
def test_attention_of_many_sequences(backend, seqs):
    """As many as the list of a tiled launch holds, and more."""
    kv = torch.randint(0, 60, (seqs,), generator=torch.Generator().manual_seed(seqs)).tolist()
    _attention(backend, R.batch([min(k, 1) for k in kv], kv, 16, pad=5), 4, 1, 64, "bfloat16", 16)


@pytest.mark.parametrize("D,dtype,page", PATHS)
@pytest.mark.parametrize("news,kvs,before,behind", [([4, 1, 40, 3], [30, 9, 300, 8], 2, 20), ([70, 0, 90], [700, 3, 91], 33, 40)])
def test_sequences_that_reach_past_the_rows(backend, D, dtype, page, news, kvs, before, behind):
    from irgen.serving import build_paged_attention_ir

    bt = R.batch(news, kvs, page, seed=D)
    pools = Q.pools8(bt, 2, page, D)
    q = _rand(3, bt["rows"], 4, D, dtype=dtype)
    out, mag, big = Q.attention64(q, pools, bt, page, D ** -0.5)
    sl = slice(before, bt["rows"] - behind)
    ir = build_paged_attention_ir(bt["rows"] - before - behind, len(news), bt["pages"], page, bt["block_table"].shape[1], 4, 2, D, dtype,
                                  cache=E4M3FN)
    got, = _run(ir, backend, {"q": q[sl], **dict(zip(NAMES, pools)), **_meta(bt), "q_start": (bt["q_start"] - before).to(torch.int32)})
    tol = R.attention_tol(dtype, D, max(kvs), out[sl], mag[sl], big[sl])
    worst = ((got.double() - out[sl]).abs() / tol).max().item()
    assert worst <= 1.0, worst


@pytest.mark.parametrize("D,dtype,page", PATHS)
@pytest.mark.parametrize("starts", [[0, 5, 2, 40], [3, 1, 0, 0], [0, 40, 0, 40]])
def test_starts_that_descend_give_zeros(backend, D, dtype, page, starts):
    from irgen.serving import build_paged_attention_ir

    bt = R.batch([1, 1, 1], [60, 60, 60], page)
    t = {"q": _rand(1, 41, 4, D, dtype=dtype), **dict(zip(NAMES, Q.pools8(bt, 2, page, D))), **_meta(bt),
         "q_start": torch.tensor(starts, dtype=torch.int32)}
    out, = _run(build_paged_attention_ir(41, 3, bt["pages"], page, bt["block_table"].shape[1], 4, 2, D, dtype, cache=E4M3FN), backend, t)
    assert out.eq(0).all()


@pytest.mark.parametrize("B,M,P", [(0, 3, 5), (2, 0, 5), (2, 3, 0)])
@pytest.mark.parametrize("D,dtype", [(128, "bfloat16"), (80, "float32")])
def test_no_sequences_no_table_no_pages(backend, D, dtype, B, M, P):
    from irgen.serving import build_paged_append_ir, build_paged_attention_ir

    i32, u8 = dict(dtype=torch.int32), dict(dtype=torch.uint8)
    pools = [torch.zeros(P, 2, 16, D, **u8)] * 2 + [torch.zeros(P, 2, 16, **u8)] * 2
    t = {"q": _rand(1, 5, 4, D, dtype=dtype), **dict(zip(NAMES, pools)), "block_table": torch.zeros(B, M, **i32),
         "q_start": torch.arange(B + 1, **i32), "kv_len": torch.full((B,), 4, **i32)}
    out, = _run(build_paged_attention_ir(5, B, P, 16, M, 4, 2, D, dtype, cache=E4M3FN), backend, t)
    assert out.eq(0).all()
    kv = {n: _rand(2, 5, 2, D, dtype=dtype) for n in "kv"}
    got = _run(build_paged_append_ir(5, B, P, 16, M, 4, 2, D, dtype, cache=E4M3FN), backend, {**t, **kv, "inv_freq": _inv(D // 2)})
    assert got[0][B:].eq(0).all() and all(torch.equal(a, b) for a, b in zip(got[1:], pools))


@pytest.mark.parametrize("offset", [16, 3])
def test_pools_that_are_ranges_of_an_input(backend, offset):
    """Byte pools whose ranges begin between 16-byte pieces are copied, byte for byte."""
    from irgen.builder import IRBuilder
    from irgen.serving import attention, batch_inputs

    D, page, KVH = 64, 16, 2
    bt = R.batch([1, 9], [40, 77], page, seed=2)
    pools = Q.pools8(bt, KVH, page, D)
    q = _rand(9, bt["rows"], 4, D, dtype="bfloat16")
    b = IRBuilder("Ranges")
    qt = b.input("q", list(q.shape), "bfloat16")
    t, caches = {"q": q, **_meta(bt)}, []
    for name, x in zip(NAMES, pools):
        t[name] = torch.cat([torch.full((offset,), 0x55, dtype=torch.uint8), x.reshape(-1)])
        flat = b.op("aten.slice.Tensor", [b.input(name, [x.numel() + offset], "uint8")], {"dim": 0, "start": offset, "end": x.numel() + offset})
        caches.append(b.op("aten.view.default", [flat], {"size": list(x.shape)}))
    b.output(attention(b, qt, caches, batch_inputs(b, 2, bt["block_table"].shape[1]), 0.125))
    got, = _run(b.to_dict(), backend, t)
    out, mag, big = Q.attention64(q, pools, bt, page, 0.125)
    assert ((got.double() - out).abs() <= R.attention_tol("bfloat16", D, 77, out, mag, big)).all()


# ---------------------------------------------------------------- together, captured, on other streams

def _step_graph(N, B, P, page, M, H, KVH, D, V, dtype, layout, norm):
    """Append, attention and sampling from a projection of its output, as one program."""
    from irgen.builder import IRBuilder
    from irgen.serving import append, attention, batch_inputs, cache_inputs, sampling_inputs

    b = IRBuilder("QuantStep")
    q, k, v = (b.input(n, [N, h, D], dtype) for n, h in (("q", H), ("k", KVH), ("v", KVH)))
    weights = tuple(b.input(n, [D], dtype) for n in ("q_weight", "k_weight")) if norm else None
    pools = cache_inputs(b, P, page, KVH, D, layout, dtype, E4M3FN)
    batch = batch_inputs(b, B, M)
    inv, w, last = b.input("inv_freq", [D // 2], "float32"), b.input("w", [V, H * D], dtype), b.input("last_rows", [B], "int64")
    par = sampling_inputs(b, B)
    q, *pools = append(b, q, k, v, pools, batch, inv, layout, 1.0, weights, 1e-6)
    o = b.op("aten.reshape.default", [attention(b, q, pools, batch, D ** -0.5, layout)], {"shape": [N, H * D]})
    l = b.op("aten.linear.default", [b.op("aten.embedding.default", [o, last]), w])
    b.output(b.op("serving.sample.default", [l, *par]), o, q, *pools)
    return b.to_dict()


@pytest.mark.parametrize("D,dtype,layout,norm", [(128, "bfloat16", "hnd", True), (64, "float16", "nhd", False)])
@pytest.mark.parametrize("news,kvs", [([1, 1, 1, 1], [9, 700, 1, 64]), ([40, 1, 0, 200], [40, 300, 5, 260])])
def test_a_step_captured_and_replayed(backend, news, kvs, D, dtype, layout, norm):
    """One program under the caller's capture, replayed with other inputs, eager calls and synchronisations between, on
    the stream of the capture and on another: every output equals the eager one, rows and pages of no sequence too. The
    eager one against the 64-bit form over the pools as the append left them."""
    H, KVH, V, page = 8, 2, 5000, 16
    bt = R.batch(news, kvs, page, pad=4, seed=1)
    N, B, dt = bt["rows"], len(news), R.DT[dtype]
    last = (bt["q_start"][1:].long() - 1).clamp(min=0)
    sets = []
    for seed in (1, 2, 3):
        g = lambda i, *s: _rand(seed * 10 + i, *s).to(dt)   # noqa: E731, B023
        s = {"q": g(0, N, H, D), "k": g(1, N, KVH, D), "v": g(2, N, KVH, D), **dict(zip(NAMES, Q.pools8(bt, KVH, page, D, layout, seed=seed))),
             **_meta(bt), "inv_freq": _inv(D // 2), "w": (0.3 * _rand(seed, V, H * D)).to(dt), "last_rows": last,
             **_params(B, seed, T=(0.0, 1.0), k=(0, 50), p=(1.0, 0.9), m=(0.0,))}
        sets.append(s | ({"q_weight": 1 + g(3, D) / 8, "k_weight": 1 + g(4, D) / 8} if norm else {}))
    bufs = {k: backend.allocate_buffer(t.cuda()) for k, t in sets[0].items()}
    ir = _step_graph(N, B, bt["pages"], page, bt["block_table"].shape[1], H, KVH, D, V, dtype, layout, norm)
    dag, other = _dag(ir, backend), _dag(ir, backend)
    names = [o["name"] for o in ir["graph_outputs"]]
    print(f"[case] {news} {kvs} {D}", flush=True)

    def fill(s):
        for k, t in s.items():
            bufs[k].native_handle.copy_(t)

    def read(y):
        torch.cuda.synchronize()
        return [y[n].to_torch().clone() for n in names]

    same = lambda a, b: all(torch.equal(x, y) for x, y in zip(a, b))   # noqa: E731
    want = []
    for s in sets:
        fill(s)
        want.append(read(dag.execute(bufs)))
        for _ in range(2):   # (appending the same rows again changes nothing)
            assert same(read(dag.execute(bufs)), want[-1])
        o, q, *pools = (x.cpu() for x in want[-1][1:])
        out, mag, big = Q.attention64(q, pools, bt, page, D ** -0.5, layout)
        tol = R.attention_tol(dtype, D, max(kvs), out, mag, big)
        assert ((o.view(N, H, D).double() - out).abs() <= tol).all()
    assert want[0][1][int(bt["q_start"][-1]):].eq(0).all()
    g, h = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        out = dag.execute(bufs)
    with torch.cuda.graph(h):
        out2 = other.execute(bufs)
    side = torch.cuda.Stream()
    for _ in range(2):
        for s, w in zip(sets, want):
            fill(s)
            g.replay()
            assert same(read(out), w)
            assert same(read(dag.execute(bufs)), w)
            h.replay()
            g.replay()
            assert same(read(out2), w)
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                y = dag.execute(bufs)
            assert same(read(y), w)


def test_pools_that_start_between_pieces_are_refused(backend):
    from irgen.serving import build_paged_attention_ir

    bt = R.batch([1], [20], 16)
    t = {"q": _rand(1, bt["rows"], 4, 128, dtype="bfloat16"), **dict(zip(NAMES, Q.pools8(bt, 2, 16, 128))), **_meta(bt)}
    bufs = {k: backend.allocate_buffer(x.cuda()) for k, x in t.items()}
    dag = _dag(build_paged_attention_ir(bt["rows"], 1, bt["pages"], 16, bt["block_table"].shape[1], 4, 2, 128, cache=E4M3FN), backend)
    dag.execute(bufs)
    for name in ("v_pages", "k_scales"):
        odd = torch.empty(t[name].numel() + 1, dtype=torch.uint8, device="cuda")[1:].view(t[name].shape)
        odd.copy_(t[name])
        with pytest.raises(ValueError, match="16"):
            dag.execute({**bufs, name: backend.allocate_buffer(odd)})


@pytest.mark.parametrize("dtype,D,layout,norm", [("bfloat16", 128, "hnd", True), ("float16", 64, "nhd", False)])
def test_generation_over_pages_of_8_bits(backend, dtype, D, layout, norm):
    """The generator on the device: the same calls give the same tokens, over pools that hold the last run's too, and the
    likeliest token is drawn whatever cuts to one."""
    from irgen.qwen import QwenConfig
    from npu_runtime.paged_generation import SamplingParams
    from test_paged_generation import prompts

    cfg = QwenConfig(hidden=512, intermediate=1024, layers=2, heads=4, kv_heads=2, head_dim=D, vocab=8192, dtype=dtype)
    gen, _ = C.generator(cfg, rows=40, slots=6, pages=40, page_size=16, table_pages=12, backend=backend, layout=layout,
                         cache=E4M3FN, qk_norm=norm)
    ps = prompts(cfg, [1, 70, 33, 5, 150, 2, 40, 16])
    print(f"[case] {dtype} head_dim {D} {layout}: 8 prompts, 9 tokens each", flush=True)
    got = gen.generate(ps, 9, SamplingParams(temperature=0.0))
    assert [len(t) for t in got] == [9] * 8
    assert gen.generate(ps, 9, SamplingParams(temperature=0.0)) == got
    par = SamplingParams(temperature=1.1, top_k=40, top_p=0.9, min_p=0.01, seed=11)
    assert gen.generate(ps, 9, par) == gen.generate(ps, 9, par)
    assert gen.generate(ps, 9, SamplingParams(temperature=1.5, top_k=1, top_p=0.3)) == got
