"""Which graph inputs a compiled program updates in place: those whose old contents nothing else reads, under any name."""

import pytest

from hip_compiler import compile_subgraph
from irgen.builder import IRBuilder
from irgen.serving import batch_inputs, paged_append, paged_attention

SHAPE = [6, 2, 8, 16]


class _Step:
    """Inputs of an append in a graph of its own; ``pool`` and ``view`` make graph inputs and views of them."""

    def __init__(self):
        self.b = IRBuilder("Update")
        self.q, self.k, self.v = (self.b.input(n, [3, h, 16], "float32") for n, h in (("q", 4), ("k", 2), ("v", 2)))
        self.batch = batch_inputs(self.b, 2, 4)
        self.inv = self.b.input("inv_freq", [8], "float32")

    def pool(self, name):
        return self.b.input(name, SHAPE, "float32")

    def view(self, t, shape=SHAPE):
        return self.b.op("aten.view.default", [t], {"size": list(shape)})

    def append(self, kp, vp):
        return paged_append(self.b, self.q, self.k, self.v, kp, vp, self.batch, self.inv)

    def twice(self, t):
        return self.b.op("aten.mul.Tensor", [t, t])

    def program(self, *outputs):
        self.b.output(*outputs)
        return compile_subgraph(self.b.to_dict())


def _updated(prog):
    return sorted(prog.stats["mutated_inputs"])


def _copied(prog, name):
    """Whether the program copies input ``name`` whole, before it appends."""
    kinds = [s.kind for s in prog.steps]
    at = kinds.index("paged_append")
    return any(s.kind == "copy" and s.inputs == [name] for s in prog.steps[:at])


def test_pools_that_nothing_else_reads():
    s = _Step()
    q, kp, vp = s.append(s.view(s.pool("k_pages")), s.view(s.view(s.pool("v_pages"), [12, 128])))
    o = paged_attention(s.b, q, kp, vp, s.batch, 0.25)
    prog = s.program(o, kp, vp)
    assert _updated(prog) == ["k_pages", "v_pages"] and not any(st.kind == "copy" for st in prog.steps)
    s = _Step()   # a second update of what a first one returned
    q, kp, vp = s.append(s.pool("k_pages"), s.pool("v_pages"))
    s.q = q
    q, kp, vp = s.append(kp, vp)
    prog = s.program(q, kp, vp)
    assert _updated(prog) == ["k_pages", "v_pages"] and not any(st.kind == "copy" for st in prog.steps)


@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("how", ["input", "view", "other view", "view of a view"])
def test_a_second_reader_under_another_name(how, first):
    """The old contents are promised to it, whether it stands before the update or behind it."""
    s = _Step()
    kp, vp = s.pool("k_pages"), s.pool("v_pages")
    kv = s.view(kp)
    read = {"input": lambda: kp, "view": lambda: kv, "other view": lambda: s.view(kp, [12, 128]),
            "view of a view": lambda: s.view(kv, [12, 128])}[how]
    other = s.twice(read()) if first else None
    q, k2, v2 = s.append(kv, vp)
    prog = s.program(q, k2, v2, other if first else s.twice(read()))
    assert _updated(prog) == ["v_pages"] and _copied(prog, "view")


def test_a_pool_that_is_a_graph_output():
    s = _Step()
    kp, vp = s.pool("k_pages"), s.pool("v_pages")
    q, k2, v2 = s.append(s.view(kp), vp)
    prog = s.program(q, k2, v2, kp)
    assert _updated(prog) == ["v_pages"] and _copied(prog, "view")


def test_two_pools_of_one_input():
    s = _Step()
    kp = s.pool("pages")
    q, k2, v2 = s.append(s.view(kp), s.view(kp))
    prog = s.program(q, k2, v2)
    assert _updated(prog) == [] and [st.kind for st in prog.steps].count("copy") == 2
    s = _Step()
    kp = s.pool("pages")
    q, k2, v2 = s.append(kp, kp)
    assert _updated(s.program(q, k2, v2)) == []


def test_rows_that_lie_in_the_pool():
    s = _Step()
    kp, vp = s.pool("k_pages"), s.pool("v_pages")
    s.k = s.b.op("aten.slice.Tensor", [s.view(kp, [96, 16])], {"dim": 0, "start": 0, "end": 6})
    s.k = s.view(s.k, [3, 2, 16])
    q, k2, v2 = s.append(kp, vp)
    assert _updated(s.program(q, k2, v2)) == ["v_pages"]


def test_a_later_update_of_contents_that_are_still_read():
    s = _Step()
    q, k1, v1 = s.append(s.pool("k_pages"), s.pool("v_pages"))
    q2, k2, v2 = s.append(k1, v1)
    prog = s.program(q, q2, k2, v2, s.twice(k1))
    kinds = [st.kind for st in prog.steps]
    assert _updated(prog) == ["k_pages", "v_pages"] and kinds.count("paged_append") == 2 and kinds.count("copy") == 1


def test_index_copy_of_a_view_with_another_reader():
    b = IRBuilder("Cache")
    past, idx, src = b.input("past", [1, 2, 8, 4], "float32"), b.input("idx", [1], "int64"), b.input("src", [1, 2, 1, 4], "float32")
    flat = b.op("aten.view.default", [past], {"size": [2, 8, 4]})
    new = b.op("aten.index_copy.default", [flat, idx, b.op("aten.view.default", [src], {"size": [2, 1, 4]})], {"dim": 1})
    b.output(new)
    assert _updated(compile_subgraph(b.to_dict())) == ["past"]
    b.output(b.op("aten.mul.Tensor", [past, past]))
    assert _updated(compile_subgraph(b.to_dict())) == []


class _Backend:
    def create_executor(self, program):
        return program


def _partitions(ir, on_host):
    """Inputs that each device partition updates in place, ``on_host`` being the ops that stay on the CPU."""
    from hip_compiler import is_hip_op_supported
    from npu_compiler import partition
    from npu_runtime import DAGExecutor

    plan = partition(ir, lambda op, attrs=None: op not in on_host and is_hip_op_supported(op, attrs))
    dag = DAGExecutor(plan, _Backend(), compile_fn=compile_subgraph)
    return [_updated(dag.npu_programs[i]) for i in sorted(dag.npu_programs)]


@pytest.mark.parametrize("first", [True, False])
def test_a_reader_in_another_partition(first):
    """A partition on the host that reads a pool behind the update gets what the graph's input held; one before it is
    done by then."""
    s = _Step()
    kp, vp = s.pool("k_pages"), s.pool("v_pages")
    other = s.twice(kp) if first else None
    q, k2, v2 = s.append(kp, vp)
    s.b.output(q, k2, v2, other if first else s.twice(kp))
    ir = s.b.to_dict()
    assert _partitions(ir, {"aten.mul.Tensor"}) == [["k_pages", "v_pages"] if first else ["v_pages"]]
    assert _partitions(ir, set()) == [["v_pages"]]


def test_a_pool_that_two_partitions_update():
    """What the first returned is updated by the second, unless it is a graph output."""
    for out in (False, True):
        s = _Step()
        kp, vp = s.pool("k_pages"), s.pool("v_pages")
        q, k1, v1 = s.append(kp, vp)
        s.q = s.twice(q)   # on the host, between the two
        q, k2, v2 = s.append(k1, v1)
        s.b.output(q, k2, v2, *([k1] if out else []))
        k1, v1 = k1.name, v1.name
        assert _partitions(s.b.to_dict(), {"aten.mul.Tensor"}) == [["k_pages", "v_pages"], [v1] if out else sorted([k1, v1])]


def test_a_graph_input_that_is_an_output_of_the_whole():
    s = _Step()
    kp, vp = s.pool("k_pages"), s.pool("v_pages")
    q, k2, v2 = s.append(kp, vp)
    s.b.output(q, k2, v2, kp)
    assert _partitions(s.b.to_dict(), set()) == [["v_pages"]]
