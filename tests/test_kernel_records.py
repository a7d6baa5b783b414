"""Argument records of kernels against what reading them costs."""

import ctypes as C

from hip_compiler import compile_subgraph
from hip_runtime.kernels import STRUCTS, check_layouts
from irgen.serving import build_paged_attention_ir


def test_attention_over_16_bit_pages_reads_the_launch_size_beside_its_record():
    """The three words behind a record are the launch's workgroups, which the kernels read, as they do the record's grid_narrow. In
    other 64 bytes than that they are one more fetch from memory before the first work: 0.25 of 13.6 us for one token."""
    record = STRUCTS["PagedAttnArgs"]
    assert (C.sizeof(record) + 11) // 64 == record.grid_narrow.offset // 64


def test_each_attention_takes_its_own_record():
    assert not check_layouts()
    for cache, record in ((None, "PagedAttnArgs"), ("float8_e4m3fn", "PagedQuantAttnArgs")):
        for dtype in ("bfloat16", "float32"):
            steps = compile_subgraph(build_paged_attention_ir(3, 1, 4, 16, 4, 2, 1, 64, dtype, cache=cache)).steps
            assert {s.arg_struct for s in steps} == {record}
            assert all(set(s.args) == {n for n, _ in STRUCTS[record]._fields_} for s in steps)
