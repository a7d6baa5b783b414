"""Saved programs whose argument records are not those of the built kernels."""

import pytest

from hip_compiler import compile_subgraph
from hip_compiler.program_io import program_from_dict, program_to_dict
from irgen.serving import build_paged_append_ir, build_paged_attention_ir


def _saved(cache):
    return compile_subgraph(build_paged_attention_ir(3, 1, 4, 16, 4, 2, 1, 64, cache=cache))


def _steps(data):
    return data["program"]["steps"]


def test_attention_saved_with_one_record_for_both_kinds_of_pages_loads_as_what_it_is():
    """Its record held the 8-bit pages' pointers, empty where pages are of 16 bits."""
    prog = _saved("float8_e4m3fn")
    data = program_to_dict(prog)
    for s in _steps(data):
        s["arg_struct"] = "PagedAttnArgs"
    assert program_from_dict(data) == prog
    prog = _saved(None)
    data = program_to_dict(prog)
    for s in _steps(data):
        s["args"] |= {"k_scales": None, "v_scales": None, "joins": None}
    assert program_from_dict(data) == prog


def test_values_that_a_record_has_no_field_for_are_refused():
    for change in ({"args": {"k_scales": 7}}, {"arg_struct": "PagedAppendArgs"}, {"arg_struct": "NoSuchArgs"}):
        data = program_to_dict(_saved(None))
        for s in _steps(data):
            s["args"] |= change.get("args", {})
            s["arg_struct"] = change.get("arg_struct", s["arg_struct"])
        with pytest.raises(ValueError, match="compile it again"):
            program_from_dict(data)


def test_fields_that_a_saved_program_does_not_know_are_empty():
    prog = compile_subgraph(build_paged_append_ir(3, 1, 4, 16, 4, 2, 1, 64))
    data = program_to_dict(prog)
    for s in _steps(data):
        for name in ("q_weight", "k_weight", "k_scales", "v_scales", "eps", "pad"):
            del s["args"][name]
    assert program_from_dict(data).steps[0].kernel == prog.steps[0].kernel


def test_copies_of_bytes_saved_with_the_kernel_of_all_types_load_as_copies_of_bytes():
    from irgen.builder import IRBuilder

    for dtype, kernel in (("uint8", "k_copy_bytes"), ("bool", "k_copy_bytes"), ("int32", "k_copy"), ("bfloat16", "k_copy")):
        b = IRBuilder("Turned")
        x = b.op("aten.permute.default", [b.input("x", [3, 5], dtype)], {"dims": [1, 0]})
        b.output(b.op("aten.contiguous.default", [x]))
        prog = compile_subgraph(b.to_dict())
        assert [s.kernel for s in prog.steps] == [kernel]
        data = program_to_dict(prog)
        for s in _steps(data):
            s["kernel"] = "k_copy"
        assert program_from_dict(data) == prog
