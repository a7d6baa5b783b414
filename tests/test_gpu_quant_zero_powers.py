"""Attention over pages of 8 bits with power bytes of 0, which stand for 0, on narrow tiles, wide tiles and the plain kernel.

Tolerances count roundings (``serving_ref``, ``quant_ref``)."""

import pytest
import torch

import quant_ref as Q
import serving_ref as R
from conftest import gpu_available
from test_gpu_quant import E4M3FN, NAMES, _attention
from test_gpu_quant_powers import LONG, PATHS, SHORT, _scaled
from test_gpu_serving import _meta, _rand, _run

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a ROCm GPU")]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("D,page", PATHS)
@pytest.mark.parametrize("news,kvs", [SHORT, LONG, ([1], [3000]), ([200], [2000])])
@pytest.mark.parametrize("run", [1, 16, 64, 128])
def test_zeros_beside_small_and_larger_powers(backend, dtype, D, page, news, kvs, run):
    """Positions in turn, ``run`` at a time, of large numbers with a small power, of small numbers with one 2^10 above it, and
    of any numbers with a byte of 0: every third stretch each, so that blocks, groups and neighbours differ in kind."""
    bt = R.batch(news, kvs, page, seed=5)
    kp, vp, ks, vs = Q.pools8(bt, 2, page, D)
    for b, s in enumerate(kvs):
        for p in range(s):
            pg, off = R.slot(bt, b, p, page)
            kind = p // run % 3
            ks[pg, :, off] = (92, 102, 0)[kind]
            if kind == 1:   # (exponents of 2^-4 to 2^-1 rather than 2^5 to 2^8)
                x = kp[pg, :, off]
                kp[pg, :, off] = (x & 0x87) | (((x >> 3) & 15).clamp(min=9) - 9 << 3)
    _attention(backend, bt, 4, 2, D, dtype, page, pools=(kp, vp, ks, vs), scale=_scaled(92, D))


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("D,page", PATHS)
@pytest.mark.parametrize("news,kvs", [SHORT, LONG])
def test_powers_of_zero(backend, dtype, D, page, news, kvs):
    """A byte of 0 stands for 0: keys score 0 under any scale, values add nothing; a NaN stays one."""
    bt = R.batch(news, kvs, page, seed=3)
    kp, vp, ks, vs = Q.pools8(bt, 2, page, D, stale=False)
    none = torch.zeros_like(ks)
    got, _ = _attention(backend, bt, 4, 2, D, dtype, page, pools=(kp, vp, ks, none))
    assert got.eq(0).all()
    _attention(backend, bt, 4, 2, D, dtype, page, pools=(kp, vp, none, vs), scale=2.0 ** 120)
    pg, off = R.slot(bt, 0, 0, page)   # open to every row of the first sequence
    vp[pg, 0, off, 5], vs[pg, 0, off] = 0xff, 0
    clean = torch.arange(bt["rows"]) >= news[0]
    got, out = _attention(backend, bt, 4, 2, D, dtype, page, pools=(kp, vp, ks, vs), rows=clean)
    assert torch.equal(got[:news[0], :, 5].isnan(), out[:news[0], :, 5].isnan()) and got[:news[0], :2, 5].isnan().all()
    assert not got[:news[0], 2:].isnan().any()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("D,page", PATHS)
@pytest.mark.parametrize("news,kvs", [SHORT, LONG])
def test_values_of_zero_beside_others(backend, dtype, D, page, news, kvs):
    """Half of the powers are 0. Where the likeliest positions' are, an output is far below its values: under 2^-14 half a step
    of float16 is 2^-25, whatever the output."""
    from irgen.serving import build_paged_attention_ir

    bt = R.batch(news, kvs, page, seed=3)
    kp, vp, ks, vs = Q.pools8(bt, 2, page, D, stale=False)
    vs[torch.rand(vs.shape, generator=torch.Generator().manual_seed(1)) < 0.5] = 0
    q = _rand(9, bt["rows"], 4, D, dtype=dtype)
    ir = build_paged_attention_ir(bt["rows"], len(news), bt["pages"], page, bt["block_table"].shape[1], 4, 2, D, dtype, cache=E4M3FN)
    got, = _run(ir, backend, {"q": q, **dict(zip(NAMES, (kp, vp, ks, vs))), **_meta(bt)})
    out, mag, big = Q.attention64(q, (kp, vp, ks, vs), bt, page, D ** -0.5)
    tol = Q.attention_tol(dtype, D, max(kvs), out, mag, big, q, (kp, vp, ks, vs), bt, page) + Q.LEAST_HALF[dtype]
    assert ((got.double() - out).abs() <= tol).all()
