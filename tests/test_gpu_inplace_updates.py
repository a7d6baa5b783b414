"""Graphs that read a pool's old contents beside updating it, on the device and split between device and host, against
the CPU fallback."""

import pytest
import torch

import serving_ref as R
from conftest import gpu_available
from irgen.builder import IRBuilder
from irgen.serving import batch_inputs, paged_append

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a ROCm GPU")]


@pytest.mark.parametrize("on_host", [(), ("aten.mul.Tensor",)])
@pytest.mark.parametrize("how", ["input", "view", "two views of one pool", "output"])
def test_old_contents_are_kept_for_their_readers(backend, how, on_host):
    """float32: a rotation's two products and its cosines, rounded in another order: 8 half steps of values under 10."""
    from hip_compiler import compile_subgraph, is_hip_op_supported
    from npu_compiler import partition
    from npu_runtime import DAGExecutor

    page, H, KVH, D = 8, 4, 2, 16
    bt = R.batch([5, 1], [20, 9], page)
    N, (kp, vp) = bt["rows"], R.pools(bt, KVH, page, D, "float32")
    g = torch.Generator().manual_seed(4)
    t = {"q": torch.randn(N, H, D, generator=g), "k": torch.randn(N, KVH, D, generator=g), "v": torch.randn(N, KVH, D, generator=g),
         "inv_freq": 1e4 ** -(torch.arange(D // 2) / (D // 2)), "k_pages": kp, "v_pages": vp,
         **{n: bt[n] for n in ("block_table", "q_start", "kv_len")}}
    b = IRBuilder("Reads")
    q, k, v = (b.input(n, list(t[n].shape), "float32") for n in "qkv")
    pools = [b.input(n, list(kp.shape), "float32") for n in ("k_pages", "v_pages")]
    batch, inv = batch_inputs(b, 2, bt["block_table"].shape[1]), b.input("inv_freq", [D // 2], "float32")
    view = lambda x: b.op("aten.view.default", [x], {"size": list(kp.shape)})   # noqa: E731
    at = {"input": [view(pools[0]), pools[1]], "view": [view(pools[0]), pools[1]],
          "two views of one pool": [view(pools[0]), view(pools[0])], "output": pools}[how]
    out = list(paged_append(b, q, k, v, *at, batch, inv))
    read = {"input": pools[0], "view": at[0]}.get(how, pools[1])
    out.append(b.op("aten.mul.Tensor", [read, read]))
    if how == "output":
        out.append(pools[0])
    b.output(*out)
    ir = b.to_dict()
    host = DAGExecutor(partition(ir, lambda *a: False), None)
    host.load_weights({})
    want = host.execute({n: x.numpy().copy() for n, x in t.items()})
    plan = partition(ir, lambda op, attrs=None: op not in on_host and is_hip_op_supported(op, attrs))
    dag = DAGExecutor(plan, backend, compile_fn=compile_subgraph)
    dag.load_weights({})
    print(f"[case] {how} {on_host}", flush=True)
    got = dag.execute({n: backend.allocate_buffer(x.cuda()) for n, x in t.items()})
    for o in ir["graph_outputs"]:
        y = got[o["name"]]
        y = torch.from_numpy(y.copy()) if not hasattr(y, "to_torch") else y.to_torch().cpu()
        assert (y - torch.from_numpy(want[o["name"]])).abs().max() <= 10 * 8 * 2.0 ** -24


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_generation_with_the_append_on_the_host(backend, dtype):
    """A plan that leaves the caches' update to the CPU: the generator takes the pools back to the device. Pools are then
    compared place by place with those of a generator whose plan is all on the device: the same rotations, rounded once
    (and what the layer before rounds otherwise: one layer)."""
    import test_paged_generation as M
    from hip_compiler import compile_subgraph, is_hip_op_supported
    from irgen.qwen import QwenConfig, build_paged_ir
    from npu_compiler import partition
    from npu_runtime import DAGExecutor
    from npu_runtime.paged_generation import PagedGenerator, SamplingParams

    cfg = QwenConfig(hidden=256, intermediate=512, layers=1, heads=4, kv_heads=2, head_dim=64, vocab=4096, dtype=dtype)
    ir = build_paged_ir(24, 3, 20, 16, 6, cfg)
    w = M.make_weights(ir, cfg)
    ps, greedy = M.prompts(cfg, [5, 40, 1]), SamplingParams(temperature=0.0)
    plan = partition(ir, lambda op, attrs=None: op != "serving.paged_append.default" and is_hip_op_supported(op, attrs))
    dag = DAGExecutor(plan, backend, compile_fn=compile_subgraph)
    dag.load_weights(w)
    print(f"[case] {dtype}", flush=True)
    gens = [PagedGenerator(d, ir, backend=backend) for d in (M.executor(ir, w, backend), dag)]
    got = [g.generate(ps, 1, greedy) for g in gens]
    assert got[0] == got[1]
    half = {"bfloat16": 2.0 ** -8, "float32": 2.0 ** -24}[dtype]
    for a, b in zip(*(g._pools().values() for g in gens)):
        a, b = a.native_handle.double(), b.native_handle.double()
        assert a.ne(0).any() and ((a - b).abs() <= 2.01 * half * torch.maximum(a.abs(), b.abs()) + 2.0 ** -20 * a.abs().max()).all()
