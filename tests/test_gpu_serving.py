"""The serving operators' kernels against plain 64-bit forms, at the sizes, batches and values where they can go wrong.

Tolerances count roundings (``serving_ref``): half a step of the output's type per rounding, plus the 32-bit sums."""

import numpy as np
import pytest
import torch

import serving_ref as R
from conftest import gpu_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a ROCm GPU")]


def _dag(ir, backend):
    from hip_compiler import compile_subgraph, is_hip_op_supported
    from npu_compiler import partition
    from npu_runtime import DAGExecutor

    dag = DAGExecutor(partition(ir, is_hip_op_supported), backend, compile_fn=compile_subgraph)
    dag.load_weights({})
    return dag


def _run(ir, backend, tensors):
    bufs = {k: backend.allocate_buffer(t.cuda()) for k, t in tensors.items()}
    print(f"[case] {ir['model_name']} {[(i['name'], i['shape'], i['dtype']) for i in ir['graph_inputs'][:1]]}", flush=True)
    out = _dag(ir, backend).execute(bufs)
    torch.cuda.synchronize()
    return [out[o["name"]].to_torch().cpu() for o in ir["graph_outputs"]]


def _meta(bt):
    return {k: bt[k] for k in ("block_table", "q_start", "kv_len")}


def _rand(seed, *shape, dtype="float32"):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(R.DT[dtype])


def _inv(r, theta=1e6):
    return 1.0 / theta ** (torch.arange(r).float() / max(r, 1))


# ---------------------------------------------------------------- append

@pytest.mark.parametrize("H,KVH,D,r,dtype,page,layout", [
    (12, 2, 128, 64, "bfloat16", 16, "hnd"), (14, 2, 64, 32, "float16", 32, "nhd"),
    (4, 4, 80, 16, "bfloat16", 48, "hnd"),     # part of the dims rotated, the rest copied
    (3, 1, 20, 7, "float16", 5, "nhd"),        # odd everything
    (4, 2, 16, 0, "float32", 1, "hnd"),        # no rotation, one position per page
    (8, 1, 64, 32, "float32", 16, "hnd"), (5, 5, 24, 8, "bfloat16", 16, "nhd")])
@pytest.mark.parametrize("news,kvs", [([1], [1]), ([1, 0, 5, 1], [130000, 5, 9, 64]), ([0, 37], [3, 37])])
def test_paged_append(backend, H, KVH, D, r, dtype, page, layout, news, kvs):
    from irgen.serving import build_paged_append_ir

    kvs = [s if s < 1000 else s // 1000 * page for s in kvs] if page < 5 else kvs
    bt = R.batch(news, kvs, page, pad=3, lead=0, seed=D)
    kp, vp = R.pools(bt, KVH, page, D, dtype, layout)
    q, k, v = (_rand(i, bt["rows"], h, D, dtype=dtype) for i, h in enumerate((H, KVH, KVH)))
    ir = build_paged_append_ir(bt["rows"], len(news), bt["pages"], page, bt["block_table"].shape[1], H, KVH, D, dtype,
                               layout, rotary_dim=2 * r, attention_scaling=1.25)
    got = _run(ir, backend, {"q": q, "k": k, "v": v, "k_pages": kp, "v_pages": vp, **_meta(bt), "inv_freq": _inv(r)})
    ref = R.append64(q, k, v, kp, vp, bt, _inv(r), page, layout, 1.25)
    # c, d and their products with x: three roundings each in 32 bits of |x| 1.25 <= 8, two terms, then the output's
    for g, x in zip(got[:2], ref[:2]):
        assert (np.abs(g.double().numpy() - x) <= 1.001 * R.HALF_STEP[dtype] * np.abs(x) + 7 * 2.0 ** -24 * 16).all()
    assert np.array_equal(got[2].double().numpy(), ref[2])
    # places that no new token has stay as they were, bit for bit
    same = ref[1] == kp.double().numpy()
    assert torch.equal(got[1][torch.from_numpy(same)], kp[torch.from_numpy(same)])
    assert (got[0][bt["q_start"][-1]:] == 0).all()


def test_paged_append_of_strided_rows(backend):
    """q, k, v as column ranges of one [rows, (H + 2 KVH) D] projection, and a k whose dims are strided."""
    from irgen.builder import IRBuilder
    from irgen.serving import batch_inputs, paged_append

    H, KVH, D, page = 4, 2, 64, 16
    bt = R.batch([3, 1, 20], [3, 40, 20], page, pad=1)
    N = bt["rows"]
    kp, vp = R.pools(bt, KVH, page, D, "bfloat16")
    y = _rand(5, N, (H + 2 * KVH) * D, dtype="bfloat16")
    kt = _rand(6, KVH, D, N, dtype="bfloat16")
    for strided in (False, True):
        b = IRBuilder("AppendStrided")
        yt = b.input("y", list(y.shape), "bfloat16")
        cut = lambda i, j: b.op("aten.view.default", [b.op("aten.slice.Tensor", [yt], {"dim": 1, "start": i * D, "end": j * D})],
                                {"size": [N, j - i, D]})
        q, k, v = cut(0, H), cut(H, H + KVH), cut(H + KVH, H + 2 * KVH)
        if strided:
            k = b.op("aten.permute.default", [b.input("kt", list(kt.shape), "bfloat16")], {"dims": [2, 0, 1]})
        pools = [b.input(n, list(kp.shape), "bfloat16") for n in ("k_pages", "v_pages")]
        batch = batch_inputs(b, 3, bt["block_table"].shape[1])
        b.output(*paged_append(b, q, k, v, *pools, batch, b.input("inv_freq", [D // 2], "float32")))
        x = {"y": y, "k_pages": kp, "v_pages": vp, **_meta(bt), "inv_freq": _inv(D // 2)}
        got = _run(b.to_dict(), backend, {**x, "kt": kt} if strided else x)
        q, k, v = (t.reshape(N, -1, D) for t in y.split([H * D, KVH * D, KVH * D], 1))
        k = kt.permute(2, 0, 1) if strided else k
        ref = R.append64(q, k, v, kp, vp, bt, _inv(D // 2), page)
        for g, w in zip(got[:2], ref[:2]):
            assert (np.abs(g.double().numpy() - w) <= 1.001 * 2.0 ** -8 * np.abs(w) + 7 * 2.0 ** -24 * 16).all()
        assert np.array_equal(got[2].double().numpy(), ref[2])


# ---------------------------------------------------------------- attention

def _attention(backend, bt, H, KVH, D, dtype, page, layout, scale=None, kp=None, vp=None, q=None):
    from irgen.serving import build_paged_attention_ir

    if kp is None:
        kp, vp = R.pools(bt, KVH, page, D, dtype, layout, stale=float("nan"))
    q = _rand(9, bt["rows"], H, D, dtype=dtype) if q is None else q
    ir = build_paged_attention_ir(bt["rows"], bt["kv_len"].numel(), bt["pages"], page, bt["block_table"].shape[1], H, KVH,
                                  D, dtype, layout, scale)
    got, = _run(ir, backend, {"q": q, "k_pages": kp, "v_pages": vp, **_meta(bt)})
    out, mag, big = R.attention64(q, kp, vp, bt, page, D ** -0.5 if scale is None else scale, layout)
    tol = R.attention_tol(dtype, D, int(bt["kv_len"].max()) if bt["kv_len"].numel() else 1, out, mag, big)
    assert torch.isfinite(got.float()).all()
    worst = ((got.double() - out).abs() / tol).max().item() if got.numel() else 0.0
    assert worst <= 1.0, worst
    return got


# one token per sequence; idle slots; chunks that start in the middle of a page and end inside a tile; whole prompts
GPU_BATCHES = [([1], [1]), ([1], [300]), ([1, 1, 0, 1, 1], [64, 1, 9, 65, 700]), ([5, 1, 40], [5, 130, 170]),
               ([97], [97]), ([33, 0, 2], [289, 0, 2])]


@pytest.mark.parametrize("H,KVH,D,dtype,page,layout", [
    (12, 2, 128, "bfloat16", 16, "hnd"), (14, 2, 64, "float16", 32, "nhd"), (8, 8, 128, "bfloat16", 48, "nhd"),
    (16, 1, 128, "float16", 64, "hnd"), (40, 8, 64, "bfloat16", 128, "hnd"), (17, 1, 64, "bfloat16", 16, "hnd"),
    (6, 2, 80, "bfloat16", 16, "hnd"), (4, 2, 128, "bfloat16", 20, "hnd"), (4, 2, 64, "float32", 16, "nhd"),
    (2, 1, 256, "float16", 16, "hnd"), (3, 3, 20, "float16", 3, "hnd")])
@pytest.mark.parametrize("news,kvs", GPU_BATCHES)
def test_paged_attention(backend, H, KVH, D, dtype, page, layout, news, kvs):
    _attention(backend, R.batch(news, kvs, page, pad=2, seed=D + page), H, KVH, D, dtype, page, layout)


@pytest.mark.parametrize("D,dtype", [(128, "bfloat16"), (64, "float16"), (80, "bfloat16")])
def test_paged_attention_of_places_that_do_not_exist(backend, D, dtype):
    bt = R.batch([2, 30, 1, 1], [100, 90, 33, 20], 16, pad=4)
    bt["block_table"][0, 1], bt["block_table"][0, 6], bt["block_table"][1, 2] = 99999, -7, -1
    bt["block_table"][2, :] = -1                     # a sequence without one page that exists
    bt["kv_len"][3] = 0                              # its new token sits at position -1
    kp, vp = R.pools(bt, 2, 16, D, dtype, stale=float("nan"))
    got = _attention(backend, bt, 4, 2, D, dtype, 16, "hnd", kp=kp, vp=vp)
    assert (got[32:] == 0).all()


@pytest.mark.parametrize("D,dtype", [(128, "bfloat16"), (64, "float16"), (80, "float16")])
def test_paged_attention_of_infinite_and_nan_places_behind_a_row(backend, D, dtype):
    """What a later position holds does not enter an earlier row, also where one tile takes both."""
    from irgen.serving import build_paged_attention_ir

    bt = R.batch([60, 1], [130, 70], 16)
    kp, vp = R.pools(bt, 2, 16, D, dtype, stale=float("inf"))
    for p, bad in ((100, float("nan")), (117, float("inf"))):   # rows 30 and 47 of the first sequence
        page, off = R.slot(bt, 0, p, 16)
        kp[page, :, off], vp[page, :, off] = bad, bad
    q = _rand(9, bt["rows"], 4, D, dtype=dtype)
    ir = build_paged_attention_ir(bt["rows"], 2, bt["pages"], 16, bt["block_table"].shape[1], 4, 2, D, dtype)
    got, = _run(ir, backend, {"q": q, "k_pages": kp, "v_pages": vp, **_meta(bt)})
    out, mag, big = R.attention64(q, kp, vp, bt, 16, D ** -0.5)
    clean = torch.ones(61, dtype=torch.bool)
    clean[30:60] = False
    tol = R.attention_tol(dtype, D, 130, out[clean], mag[clean], big[clean])
    assert ((got[clean].double() - out[clean]).abs() <= tol).all()
    assert got[30:60].isnan().any(-1).all() and out[30:60].isnan().any(-1).all()


def test_paged_attention_of_large_scores(backend):
    """Scores of a few hundred: one position takes nearly all, and exponentials of the others underflow."""
    bt = R.batch([40, 1], [200, 333], 16)
    q = 8 * _rand(9, bt["rows"], 4, 128, dtype="bfloat16")
    kp, vp = R.pools(bt, 2, 16, 128, "bfloat16")
    _attention(backend, bt, 4, 2, 128, "bfloat16", 16, "hnd", scale=0.5, kp=8 * kp, vp=vp, q=q)


# ---------------------------------------------------------------- sampling

def _params(B, seed, T=(0.0, 0.5, 1.0, 2.0), k=(0, 1, 3, 50, 700, 10 ** 6), p=(1.0, 0.95, 0.5, 0.01, 0.0, 2.0),
            m=(0.0, 0.02, 0.5, 1.0)):
    r = np.random.default_rng(seed)
    f = lambda a: torch.tensor(r.choice(np.array(a, np.float32), B))
    return {"temperature": f(T), "top_k": torch.tensor(r.choice(np.array(k, np.int32), B)), "top_p": f(p), "min_p": f(m),
            "u": torch.tensor(r.random(B, np.float32))}


def _sample(backend, x, par, dtype):
    from irgen.serving import build_sample_ir

    got, = _run(build_sample_ir(x.shape[0], x.shape[1], dtype), backend, {"logits": x, **par})
    return got


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("B,V", [(64, 1), (64, 2), (64, 511), (70, 4096), (48, 50021), (24, 151936)])
def test_sample(backend, B, V, dtype):
    x = (2.5 * _rand(V, B, V)).to(R.DT[dtype])
    par = _params(B, V)
    assert torch.equal(_sample(backend, x, par, dtype), R.sample64(x, **par))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_sample_of_ties_and_flat_rows(backend, dtype):
    """Equal logits in one row (every split of the ranking is by index), two values, values within a few steps of
    each other, and one far above the rest."""
    V = 30011
    x = torch.zeros(40, V)
    x[10:20] = _rand(1, 10, V).sign()
    x[20:30] = 1.0 + (_rand(2, 10, V) * 3).round() * 2.0 ** -7
    x[30:40, 777] = 50.0
    par = _params(40, 5, T=(0.3, 1.0), k=(0, 1, 777, 5000, 29999), p=(1.0, 0.9, 0.37, 1e-6))
    x = x.to(R.DT[dtype])
    assert torch.equal(_sample(backend, x, par, dtype), R.sample64(x, **par))


def test_sample_of_special_values(backend):
    inf, nan = float("inf"), float("nan")
    x = torch.tensor([[-inf, nan, -inf, nan], [nan, 1.0, 1.0, -inf], [inf, 0.0, inf, nan], [-0.0, 0.0, -1.0, 0.0],
                      [2.0, 2.0, 2.0, 2.0], [3.0, -3.4e38, 3.4e38, 0.0]])
    from npu_runtime.serving_ops import sample

    for T in (1.0, 0.0, -1.0, nan, inf, 1e-40, 1e-3):
        for k in (0, 2, -3):
            for p in (1.0, 0.5, nan, -1.0):
                for m in (0.0, nan, 3.0):
                    for u in (0.0, 0.6, 0.99999994, 1.0, -1.0, nan):
                        par = {"temperature": torch.full((6,), T), "top_k": torch.full((6,), k, dtype=torch.int32),
                               "top_p": torch.full((6,), p), "min_p": torch.full((6,), m), "u": torch.full((6,), u)}
                        if u == u and u >= 0:
                            want = sample(x, **par)
                        else:   # counts as 0
                            want = sample(x, **{**par, "u": torch.zeros(6)})
                        if k == 0 and m == 0.0 and u == 0.6:
                            print(f"[case] T={T} p={p}", flush=True)
                        got = _special(backend, x, par)
                        assert torch.equal(got, want), (T, k, p, m, u, got, want)


_SPECIAL = {}


def _special(backend, x, par):
    from irgen.serving import build_sample_ir

    if not _SPECIAL:
        ir = build_sample_ir(6, 4, "float32")
        _SPECIAL.update(dag=_dag(ir, backend), out=ir["graph_outputs"][0]["name"],
                        bufs={k: backend.allocate_buffer(t.cuda()) for k, t in {"logits": x, **par}.items()})
    for k, t in {"logits": x, **par}.items():
        _SPECIAL["bufs"][k].native_handle.copy_(t)
    return _SPECIAL["dag"].execute(_SPECIAL["bufs"])[_SPECIAL["out"]].to_torch().cpu()


@pytest.mark.parametrize("H,KVH,D,page", [(12, 2, 128, 16), (4, 4, 64, 32), (8, 1, 128, 48)])
@pytest.mark.parametrize("new,kv", [(40, 3958), (70, 2040), (1, 9000), (2, 4095)])
def test_paged_attention_of_long_tiles(backend, H, KVH, D, page, new, kv):
    """Tiles split along their positions: parts that begin at the last block of a window of page ids, and at every other."""
    _attention(backend, R.batch([new, 1], [kv, 77], page, seed=new), H, KVH, D, "bfloat16", page, "hnd")


# ---------------------------------------------------------------- rows that bins do not split well, and other grids

@pytest.mark.parametrize("dtype,spread,shift", [
    ("float32", 0.3, 0.0),       # thousands of tokens in a bin: more than a row's list holds
    ("float32", 1.0, 0.0), ("bfloat16", 1.0, 0.0), ("float16", 0.01, 0.0),
    ("float32", 3.0, 3e4), ("float32", 3.0, -6e4),   # near and past the bound of the grid
    ("float32", 100.0, 1e7),     # past it
    ("float32", 40.0, 0.0)])     # most tokens weigh nothing, and whole parts
def test_sample_of_dense_and_distant_rows(backend, dtype, spread, shift):
    x = (spread * _rand(7, 8, 120011) + shift).to(R.DT[dtype])
    x[0, 0], x[1, -1] = float("inf"), float("nan")
    par = _params(8, 3, T=(0.3, 1.0, 8.0), k=(0, 50, 3000), p=(1.0, 0.95, 0.5), m=(0.0, 0.01))
    assert torch.equal(_sample(backend, x, par, dtype), R.sample64(x, **par))


@pytest.mark.parametrize("B,V,dtype", [(1, 151936, "bfloat16"), (1, 4097, "float32"), (3, 8200, "float16"),
                                       (300, 9001, "float32"), (1100, 4500, "float32"), (2, 500009, "bfloat16")])
def test_sample_over_parts_of_every_size(backend, B, V, dtype):
    x = (2.0 * _rand(B + V, B, V)).to(R.DT[dtype])
    par = _params(B, V + 1, T=(0.7, 1.0), k=(0, 40), p=(1.0, 0.9), m=(0.0, 0.03))
    assert torch.equal(_sample(backend, x, par, dtype), R.sample64(x, **par))


@pytest.mark.parametrize("D,page,dtype", [(128, 1, "bfloat16"), (80, 7, "float16"), (64, 24, "bfloat16"), (48, 16, "float32"),
                                          (256, 32, "float16"), (1, 3, "float32")])
def test_paged_attention_of_other_pages_and_heads(backend, D, page, dtype):
    _attention(backend, R.batch([1, 0, 5, 33, 0, 1], [1, 0, 5, 70, 9, 130], page, pad=3, seed=D), 6, 2, D, dtype, page, "nhd")


@pytest.mark.parametrize("seqs", [1000, 1100])
def test_paged_attention_of_many_sequences(backend, seqs):
    """As many as the list of a tiled launch holds, and more."""
    r = np.random.default_rng(seqs)
    kv = r.integers(0, 60, seqs)
    _attention(backend, R.batch([min(int(k), 1) for k in kv], [int(k) for k in kv], 16, pad=5), 4, 1, 64, "bfloat16", 16, "hnd")


@pytest.mark.parametrize("D,starts", [(128, [0, 5, 2, 40]), (64, [3, 1, 0, 0]), (128, [0, 40] * 30 + [0])])
def test_paged_attention_of_starts_that_descend(backend, D, starts):
    """No batch: nothing outside the tensors is touched, and every row is zero."""
    from irgen.serving import build_paged_attention_ir

    B, dt = len(starts) - 1, torch.bfloat16
    t = {"q": _rand(1, 41, 4, D).to(dt), "k_pages": _rand(2, 9, 2, 16, D).to(dt), "v_pages": _rand(3, 9, 2, 16, D).to(dt),
         "block_table": torch.arange(B * 4, dtype=torch.int32).view(B, 4) % 9, "q_start": torch.tensor(starts, dtype=torch.int32),
         "kv_len": torch.full((B,), 60, dtype=torch.int32)}
    out, = _run(build_paged_attention_ir(41, B, 9, 16, 4, 4, 2, D), backend, t)
    assert out.eq(0).all()


def test_lengths_far_out_of_range(backend):
    """Lengths at the ends of int32: positions before 0 have no place, those past the table neither."""
    from irgen.serving import build_paged_append_ir, build_paged_attention_ir

    dt, lim = torch.bfloat16, torch.iinfo(torch.int32)
    meta = {"block_table": torch.arange(12, dtype=torch.int32).view(3, 4), "q_start": torch.tensor([0, 2, 4, 6], dtype=torch.int32),
            "kv_len": torch.tensor([lim.min, lim.max, 70], dtype=torch.int32)}
    t = {"q": _rand(1, 6, 4, 128).to(dt), "k": _rand(4, 6, 2, 128).to(dt), "v": _rand(5, 6, 2, 128).to(dt),
         "k_pages": _rand(2, 12, 2, 16, 128).to(dt), "v_pages": _rand(3, 12, 2, 16, 128).to(dt), **meta, "inv_freq": _inv(64)}
    _, kp, vp = _run(build_paged_append_ir(6, 3, 12, 16, 4, 4, 2, 128), backend, t)
    assert torch.equal(kp, t["k_pages"]) and torch.equal(vp, t["v_pages"])
    a = {n: t[n] for n in ("q", "k_pages", "v_pages", *meta)}
    out, = _run(build_paged_attention_ir(6, 3, 12, 16, 4, 4, 2, 128), backend, a)
    full, = _run(build_paged_attention_ir(6, 3, 12, 16, 4, 4, 2, 128), backend,
                 {**a, "kv_len": torch.tensor([-1, 1 << 30, 66], dtype=torch.int32)})
    assert out[:2].eq(0).all() and torch.isfinite(out.float()).all() and torch.equal(out, full)


def test_rows_that_name_one_place(backend):
    """Two sequences on one page: each element of the place is one of theirs, and nothing else changes."""
    from irgen.serving import build_paged_append_ir

    t = {"q": _rand(1, 2, 4, 128), "k": _rand(2, 2, 2, 128), "v": _rand(3, 2, 2, 128), "k_pages": _rand(4, 3, 2, 16, 128),
         "v_pages": _rand(5, 3, 2, 16, 128)}
    t = {n: x.to(torch.bfloat16) for n, x in t.items()}
    t |= {"block_table": torch.ones(2, 1, dtype=torch.int32), "q_start": torch.arange(3, dtype=torch.int32),
          "kv_len": torch.full((2,), 6, dtype=torch.int32), "inv_freq": _inv(64)}
    _, _, vp = _run(build_paged_append_ir(2, 2, 3, 16, 1, 4, 2, 128), backend, t)
    got = vp[1, :, 5].clone()
    assert ((got == t["v"][0]) | (got == t["v"][1])).all()
    vp[1, :, 5] = t["v_pages"][1, :, 5]
    assert torch.equal(vp, t["v_pages"])


# ---------------------------------------------------------------- together, captured, on other streams

def _step_graph(N, B, P, page, M, H, KVH, D, V, dtype):
    """Append, attention and sampling from a projection of its output, as one program."""
    from irgen.builder import IRBuilder
    from irgen.serving import batch_inputs, paged_append, paged_attention, pool_shape, sampling_inputs

    b = IRBuilder("ServingStep")
    q, k, v = (b.input(n, [N, h, D], dtype) for n, h in (("q", H), ("k", KVH), ("v", KVH)))
    kp, vp = (b.input(n, pool_shape(P, page, KVH, D), dtype) for n in ("k_pages", "v_pages"))
    batch = batch_inputs(b, B, M)
    inv = b.input("inv_freq", [D // 2], "float32")
    w = b.input("w", [V, H * D], dtype)
    last = b.input("last_rows", [B], "int64")
    par = sampling_inputs(b, B)
    q, kp, vp = paged_append(b, q, k, v, kp, vp, batch, inv)
    o = b.op("aten.reshape.default", [paged_attention(b, q, kp, vp, batch, D ** -0.5)], {"shape": [N, H * D]})
    l = b.op("aten.linear.default", [b.op("aten.embedding.default", [o, last]), w])
    b.output(b.op("serving.sample.default", [l, *par]), o, kp, vp)
    return b.to_dict()


def _step_inputs(seed, bt, H, KVH, D, V, page, dtype):
    N, B, dt = bt["rows"], len(bt["kv_len"]), R.DT[dtype]
    kp, vp = R.pools(bt, KVH, page, D, dtype, seed=seed)
    g = lambda i, *s: _rand(seed * 10 + i, *s).to(dt)   # noqa: E731
    last = (bt["q_start"][1:].long() - 1).clamp(min=0)
    return {"q": g(0, N, H, D), "k": g(1, N, KVH, D), "v": g(2, N, KVH, D), "k_pages": kp, "v_pages": vp, **_meta(bt),
            "inv_freq": _inv(D // 2), "w": (0.3 * _rand(seed, V, H * D)).to(dt), "last_rows": last,
            **_params(B, seed, T=(0.0, 1.0), k=(0, 50), p=(1.0, 0.9), m=(0.0,))}


@pytest.mark.parametrize("news,kvs", [([1, 1, 1, 1], [9, 700, 1, 64]), ([40, 1, 0, 200], [40, 300, 5, 260])])
def test_a_step_captured_and_replayed(backend, news, kvs):
    """One program under the caller's capture, replayed with other inputs, eager calls and synchronisations between, on
    the stream of the capture and on another: every output equals the eager one, rows and pages of no sequence too."""
    H, KVH, D, V, page, dtype = 8, 2, 128, 5000, 16, "bfloat16"
    bt = R.batch(news, kvs, page, pad=4, seed=1)
    sets = [_step_inputs(s, bt, H, KVH, D, V, page, dtype) for s in (1, 2, 3)]
    bufs = {k: backend.allocate_buffer(t.cuda()) for k, t in sets[0].items()}
    ir = _step_graph(bt["rows"], len(news), sets[0]["k_pages"].shape[0], page, bt["block_table"].shape[1], H, KVH, D, V, dtype)
    dag, other = _dag(ir, backend), _dag(ir, backend)
    names = [o["name"] for o in ir["graph_outputs"]]
    print(f"[case] {news} {kvs}", flush=True)

    def fill(s):
        for k, t in s.items():
            bufs[k].native_handle.copy_(t)

    def read(y):
        torch.cuda.synchronize()
        return [y[n].to_torch().clone() for n in names]

    want = []
    for s in sets:
        fill(s)
        want.append(read(dag.execute(bufs)))
        for _ in range(2):   # (appending the same rows again changes nothing)
            assert all(torch.equal(a, b) for a, b in zip(read(dag.execute(bufs)), want[-1]))
    pad = want[0][1][int(bt["q_start"][-1]):]
    assert pad.shape[0] == 4 and pad.eq(0).all()
    g, h = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        out = dag.execute(bufs)
    with torch.cuda.graph(h):
        out2 = other.execute(bufs)
    side = torch.cuda.Stream()
    for rep in range(2):
        for s, w in zip(sets, want):
            fill(s)
            g.replay()
            assert all(torch.equal(a, b) for a, b in zip(read(out), w))
            assert all(torch.equal(a, b) for a, b in zip(read(dag.execute(bufs)), w))
            h.replay()
            g.replay()
            assert all(torch.equal(a, b) for a, b in zip(read(out2), w))
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                y = dag.execute(bufs)
            assert all(torch.equal(a, b) for a, b in zip(read(y), w))


def test_a_pool_that_starts_between_pieces_is_refused(backend):
    from irgen.serving import build_paged_attention_ir

    bt = R.batch([1], [20], 16)
    kp, vp = R.pools(bt, 2, 16, 128, "bfloat16")
    t = {"q": _rand(1, bt["rows"], 4, 128).to(torch.bfloat16), "k_pages": kp, "v_pages": vp, **_meta(bt)}
    bufs = {k: backend.allocate_buffer(x.cuda()) for k, x in t.items()}
    dag = _dag(build_paged_attention_ir(bt["rows"], 1, kp.shape[0], 16, bt["block_table"].shape[1], 4, 2, 128), backend)
    dag.execute(bufs)
    odd = torch.empty(vp.numel() + 1, dtype=torch.bfloat16, device="cuda")[1:].view(vp.shape)
    odd.copy_(vp)
    with pytest.raises(ValueError, match="16"):
        dag.execute({**bufs, "v_pages": backend.allocate_buffer(odd)})


def test_an_exported_module(backend):
    """A module that calls the ops, traced and run on the device, against its own eager run. float32 sums of up to 64
    products and 40 positions, in another order: 64 + 40 half steps of values under 10."""
    from irgen.exporter import extract_ir

    class Step(torch.nn.Module):
        def forward(self, q, k, v, k_pages, v_pages, table, start, kv, inv, logits, t, top_k, p, m, u):
            q, k_pages, v_pages = torch.ops.serving.paged_append(q, k, v, k_pages, v_pages, table, start, kv, inv,
                                                                 page_layout="nhd")
            o = torch.ops.serving.paged_attention(q, k_pages, v_pages, table, start, kv, 0.125, page_layout="nhd")
            return o.flatten(1), k_pages, v_pages, torch.ops.serving.sample(logits, t, top_k, p, m, u)

    bt = R.batch([5, 1, 0], [40, 17, 3], 8, pad=2, seed=4)
    kp, vp = R.pools(bt, 2, 8, 64, "float32", "nhd")
    par = _params(6, 9)
    args = (_rand(1, bt["rows"], 4, 64), _rand(2, bt["rows"], 2, 64), _rand(3, bt["rows"], 2, 64), kp, vp, *_meta(bt).values(),
            _inv(32), 3 * _rand(5, 6, 9000), *par.values())
    want = Step()(*(a.clone() for a in args))
    ir = extract_ir(Step(), args, "step")
    got = _run(ir, backend, {i["name"]: a.clone() for i, a in zip(ir["graph_inputs"], args)})
    for a, b in zip(got[:3], want[:3]):
        assert (a - b).abs().max() <= 10 * 104 * 2.0 ** -24
    assert torch.equal(got[3], want[3])
