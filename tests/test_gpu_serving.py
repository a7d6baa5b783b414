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
