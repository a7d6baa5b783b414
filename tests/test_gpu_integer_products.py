"""Products of integer matrices on the device, against ATen: bytes modulo 256, sums past a float's 24 bits."""

import pytest
import torch

from conftest import gpu_available
from test_gpu_serving import _run

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a ROCm GPU")]


@pytest.mark.parametrize("dtype,most", [("uint8", 255), ("int32", 5000), ("int64", 1 << 20)])
@pytest.mark.parametrize("op,a,b", [("aten.mm.default", (5, 33), (33, 7)), ("aten.bmm.default", (2, 3, 20), (2, 20, 9)),
                                    ("aten.matmul.default", (2, 4, 17), (17, 3)), ("aten.linear.default", (4, 19), (6, 19))])
def test_integer_products(backend, dtype, most, op, a, b):
    from irgen.builder import IRBuilder

    dt = {"uint8": torch.uint8, "int32": torch.int32, "int64": torch.int64}[dtype]
    g = torch.Generator().manual_seed(len(a))
    x, y = (torch.randint(0, most + 1, s, generator=g).to(dt) for s in (a, b))
    ir = IRBuilder("IntegerProduct")
    ir.output(ir.op(op, [ir.input("x", list(a), dtype), ir.input("y", list(b), dtype)]))
    got, = _run(ir.to_dict(), backend, {"x": x, "y": y})
    want = x.long() @ (y.long().T if op == "aten.linear.default" else y.long())
    assert got.dtype == dt and torch.equal(got, want.to(dt))
