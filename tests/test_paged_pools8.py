"""The generator over step graphs whose inputs name the pools of 8 bits and their powers in other orders."""

import pytest

import test_paged_generation as M
import test_quant_ops as C
from irgen.qwen import build_paged_ir
from npu_runtime.paged_generation import PagedGenerator, SamplingParams


def _powers_first(ir):
    """The graph with each layer's powers before its pages, among its inputs and outputs alike."""
    def turned(specs, head):
        rest = specs[head:]
        return specs[:head] + [x for i in range(0, len(rest), 4) for x in rest[i + 2:i + 4] + rest[i:i + 2]]

    first = next(i for i, s in enumerate(ir["graph_inputs"]) if s["name"].startswith("k_pages"))
    return {**ir, "graph_inputs": turned(ir["graph_inputs"], first), "graph_outputs": turned(ir["graph_outputs"], 1)}


@pytest.mark.parametrize("layout", ["hnd", "nhd"])
def test_a_graph_whose_powers_come_before_its_pages(layout):
    """The size of a page is that of the pages, whichever pool comes first: the tokens are those of the graph in its own order."""
    kw = dict(cache="float8_e4m3fn", layout=layout)
    shape = dict(rows=16, slots=4, pages=9, page_size=8, table_pages=5)
    gen, w = C.generator(M.CFG, **shape, **kw)
    ps = M.prompts(M.CFG, [1, 23, 5, 30, 8])
    greedy = SamplingParams(temperature=0.0)
    want = gen.generate(ps, 6, greedy)
    irs = [_powers_first(build_paged_ir(n, 4, 9, 8, 5, M.CFG, **kw)) for n in (16, 4)]
    names = [s["name"] for s in irs[0]["graph_inputs"]]
    assert names.index("k_scales_0") < names.index("k_pages_0")
    dags = [M.executor(ir, w) for ir in irs]
    other = PagedGenerator(dags[0], irs[0], dags[1], irs[1])
    assert (other.pages, other.page_size) == (9, 8)
    assert other.generate(ps, 6, greedy) == want
