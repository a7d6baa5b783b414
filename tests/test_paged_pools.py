"""The generator's pools, where its two graphs treat them differently: host stand-ins for a device's buffers and programs."""

import numpy as np
import pytest
import torch

import test_paged_generation as M
from irgen.qwen import build_paged_ir
from npu_runtime.paged_generation import PagedGenerator, SamplingParams

CFG = M.CFG
SHAPE = dict(pages=12, page_size=8, table_pages=5)


class _Buffer:
    def __init__(self, a):
        self.native_handle = a if isinstance(a, torch.Tensor) else torch.from_numpy(a)

    def write_from_numpy(self, a):
        self.native_handle.copy_(torch.from_numpy(a))

    def to_numpy(self):
        return self.native_handle.numpy()


class _Backend:
    def allocate_buffer(self, a):
        return _Buffer(a)


class _Program:
    """A graph run on the host; pools are updated in place, or returned in buffers of its own or as host arrays (None)."""

    def __init__(self, ir, weights, inplace):
        self.dag, self.inplace, self.calls = M.executor(ir, weights), inplace, 0
        self.names = [o["name"] for o in ir["graph_outputs"]]
        self.pools = [i["name"] for i in ir["graph_inputs"] if "_pages_" in i["name"]]

    def execute(self, feed):
        self.calls += 1
        out = self.dag.execute({n: b.to_numpy().copy() for n, b in feed.items()})
        got = {self.names[0]: _Buffer(out[self.names[0]])}
        for pool, name in zip(self.pools, self.names[1:]):
            new = torch.from_numpy(np.array(out[name]))
            if self.inplace:
                feed[pool].native_handle.copy_(new)
            got[name] = feed[pool] if self.inplace else new.numpy() if self.inplace is None else _Buffer(new)
        return got


@pytest.mark.parametrize("step_inplace,decode_inplace", [(False, True), (True, False), (False, False), (None, True), (True, None)])
@pytest.mark.parametrize("rows,decode_rows", [(6, 6), (9, 3), (4, 7)])
def test_each_graph_carries_its_own_pools_over(step_inplace, decode_inplace, rows, decode_rows):
    """Also where both graphs have as many rows (one of them takes every step then), or the one of decode steps has more."""
    ir, dec = (build_paged_ir(n, 3, SHAPE["pages"], SHAPE["page_size"], SHAPE["table_pages"], CFG) for n in (rows, decode_rows))
    w = M.make_weights(ir, CFG)
    ps, greedy = M.prompts(CFG, [1, 13, 5, 20]), SamplingParams(temperature=0.0)
    ref = PagedGenerator(M.executor(ir, w), ir, M.executor(dec, w), dec)
    want = ref.generate(ps, 6, greedy)
    step, decode = _Program(ir, w, step_inplace), _Program(dec, w, decode_inplace)
    gen = PagedGenerator(step, ir, decode, dec, backend=_Backend())
    assert gen.generate(ps, 6, greedy) == want
    assert step.calls and bool(decode.calls) == (rows != decode_rows)
    # the same steps, and so the same sums: keys and values of every place are equal
    for name, pool in ref._pools().items():
        assert np.array_equal(gen._pools()[name].to_numpy(), pool)


def test_graphs_of_two_page_layouts_are_refused():
    """Pools of as many positions a page as K/V heads have one shape in both layouts."""
    irs = [build_paged_ir(n, 2, 6, CFG.kv_heads, 9, CFG, layout) for n, layout in ((8, "hnd"), (2, "nhd"))]
    with pytest.raises(ValueError, match="layout"):
        PagedGenerator(None, irs[0], object(), irs[1])
    mixed = build_paged_ir(8, 2, 6, CFG.kv_heads, 9, CFG)
    next(n for n in mixed["nodes"] if n["op_type"] == "serving.paged_attention.default")["attrs"]["page_layout"] = "nhd"
    with pytest.raises(ValueError, match="layout"):
        PagedGenerator(None, mixed)
