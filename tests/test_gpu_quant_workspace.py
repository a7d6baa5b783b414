"""What a call leaves in its program's workspace is nothing to the next: the operators over pages of 8 bits with every byte of the
workspace set to 0xff (NaN, and no row or part) before each call, and inputs changed in place between calls."""

import pytest
import torch

import quant_ref as Q
import serving_ref as R
from conftest import gpu_available
from test_gpu_quant import E4M3FN, NAMES
from test_gpu_serving import _dag, _inv, _meta, _rand

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a ROCm GPU")]

BATCHES = [([1], [1]), ([1] * 5 + [0], [900, 3, 4000, 64, 65, 7]), ([1, 40, 0, 1], [5000, 3000, 9, 17]), ([300, 200], [300, 900]),
           ([90, 60, 31], [9000, 90, 31])]


def _spoil(dag):
    for ex in dag.npu_executors.values():
        ex.arena.fill_(0xff)


@pytest.mark.parametrize("D,dtype,page", [(128, "bfloat16", 16), (64, "float16", 32), (80, "bfloat16", 16)])
@pytest.mark.parametrize("news,kvs", BATCHES)
def test_attention(backend, D, dtype, page, news, kvs):
    from irgen.serving import build_paged_attention_ir

    bt = R.batch(news, kvs, page, pad=3, lead=1, seed=D)
    bt["block_table"][0, -1] = -1
    ir = build_paged_attention_ir(bt["rows"], len(news), bt["pages"], page, bt["block_table"].shape[1], 8, 2, D, dtype, cache=E4M3FN)
    sets = [{"q": _rand(seed, bt["rows"], 8, D, dtype=dtype), **dict(zip(NAMES, Q.pools8(bt, 2, page, D, seed=seed))), **_meta(bt)}
            for seed in (1, 2)]
    name = ir["graph_outputs"][0]["name"]
    want = []
    for s in sets:
        out = _dag(ir, backend).execute({k: backend.allocate_buffer(t.cuda()) for k, t in s.items()})[name].to_torch().clone()
        torch.cuda.synchronize()
        assert out.isfinite().all()
        want.append(out)
    assert not torch.equal(*want)
    bufs, dag = {k: backend.allocate_buffer(t.cuda()) for k, t in sets[0].items()}, _dag(ir, backend)
    print(f"[case] {news} {kvs} D {D}", flush=True)
    for _ in range(2):
        for s, w in zip(sets, want):
            for k, t in s.items():
                bufs[k].native_handle.copy_(t)
            _spoil(dag)
            out = dag.execute(bufs)[name].to_torch()
            torch.cuda.synchronize()
            assert torch.equal(out, w)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("D,dtype,page", [(128, "bfloat16", 16), (64, "float16", 32), (40, "float32", 16)])
@pytest.mark.parametrize("news,kvs", BATCHES)
def test_append(backend, norm, D, dtype, page, news, kvs):
    from irgen.serving import build_paged_append_ir

    bt = R.batch(news, kvs, page, pad=3, lead=1, seed=D)
    ir = build_paged_append_ir(bt["rows"], len(news), bt["pages"], page, bt["block_table"].shape[1], 8, 2, D, dtype,
                               norm_eps=1e-6 if norm else None, cache=E4M3FN)
    names = [o["name"] for o in ir["graph_outputs"]]
    x = {n: _rand(i, bt["rows"], h, D, dtype=dtype) for i, (n, h) in enumerate((("q", 8), ("k", 2), ("v", 2)))}
    x |= {**_meta(bt), "inv_freq": _inv(D // 2)} | ({n: _rand(i, D, dtype=dtype) for i, n in enumerate(("q_weight", "k_weight"))} if norm else {})
    pools = dict(zip(NAMES, Q.pools8(bt, 2, page, D)))
    bufs, dag = {k: backend.allocate_buffer(t.cuda()) for k, t in {**x, **pools}.items()}, _dag(ir, backend)
    runs = []
    for spoil in (False, True, True):
        for k, t in pools.items():
            bufs[k].native_handle.copy_(t)
        if spoil:
            _spoil(dag)
        out = dag.execute(bufs)
        torch.cuda.synchronize()
        runs.append([out[n].to_torch().clone() for n in names])
    assert all(torch.equal(a, b) for run in runs[1:] for a, b in zip(runs[0], run))
