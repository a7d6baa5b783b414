"""index_copy of tensors of one byte per element on the device, against ATen: pools of 8 bits, and truth values."""

import pytest
import torch

from conftest import gpu_available
from test_gpu_serving import _dag

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a ROCm GPU")]


@pytest.mark.parametrize("dtype", ["uint8", "bool"])
@pytest.mark.parametrize("shape,dim,index", [((2, 16, 64), 1, [3, 15, 0]), ((1, 9, 5), 1, [8, 2]), ((7,), 0, [6, 1]),
                                             ((3, 4, 33), 2, [32, 5, 7, 0]), ((5, 2, 3, 11), 0, [4, 0])])
def test_index_copy_of_bytes(backend, dtype, shape, dim, index):
    """What lies before and behind the tensor stays as it was."""
    from irgen.builder import IRBuilder

    g = torch.Generator().manual_seed(len(shape) + dim)
    dt = {"uint8": torch.uint8, "bool": torch.bool}[dtype]
    x = torch.randint(0, 256, shape, generator=g, dtype=torch.uint8).to(dt)
    new_shape = [len(index) if i == dim else s for i, s in enumerate(shape)]
    new = torch.randint(0, 256, new_shape, generator=g, dtype=torch.uint8).to(dt)
    idx = torch.tensor(index)
    b = IRBuilder("IndexCopyBytes")
    xt, it, st = b.input("x", list(shape), dtype), b.input("i", [len(index)], "int64"), b.input("s", new_shape, dtype)
    b.output(b.op("aten.index_copy.default", [xt, it, st], {"dim": dim}))
    ir = b.to_dict()
    n = x.numel()
    room = torch.randint(0, 256, (n + 512,), generator=g, dtype=torch.uint8)   # the tensor in the middle of other bytes
    room[256:256 + n] = x.reshape(-1).view(torch.uint8)
    dev = room.cuda()
    bufs = {"x": backend.allocate_buffer(dev[256:256 + n].view(dt).view(shape)), "i": backend.allocate_buffer(idx.cuda()),
            "s": backend.allocate_buffer(new.cuda())}
    print(f"[case] index_copy {dtype} {shape} dim {dim}", flush=True)
    out = _dag(ir, backend).execute(bufs)[ir["graph_outputs"][0]["name"]].to_torch()
    torch.cuda.synchronize()
    want = x.index_copy(dim, idx, new)
    assert torch.equal(out.cpu(), want)
    room[256:256 + n] = want.reshape(-1).view(torch.uint8)
    assert torch.equal(dev.cpu(), room)
