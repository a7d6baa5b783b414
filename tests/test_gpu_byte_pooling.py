"""Max pooling of bytes on the device, against ATen."""

import pytest
import torch

from conftest import gpu_available
from test_gpu_serving import _run

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a ROCm GPU")]


@pytest.mark.parametrize("kernel,stride,padding", [(2, 2, 0), (3, 2, 1)])
def test_max_pooling_of_bytes(backend, kernel, stride, padding):
    from irgen.builder import IRBuilder

    x = torch.randint(0, 256, (2, 3, 9, 11), generator=torch.Generator().manual_seed(1), dtype=torch.uint8)
    attrs = {"kernel_size": [kernel] * 2, "stride": [stride] * 2, "padding": [padding] * 2}
    b = IRBuilder("BytePooling")
    b.output(b.op("aten.max_pool2d.default", [b.input("x", list(x.shape), "uint8")], attrs))
    got, = _run(b.to_dict(), backend, {"x": x})
    assert torch.equal(got, torch.nn.functional.max_pool2d(x, kernel, stride, padding))
