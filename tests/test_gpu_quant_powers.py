"""Attention over pages of 8 bits whose powers are small, on narrow tiles, wide tiles and the plain kernel.

Tolerances count roundings (``serving_ref``, ``quant_ref``)."""

import pytest
import torch

import quant_ref as Q
import serving_ref as R
from conftest import gpu_available
from test_gpu_quant import E4M3FN, NAMES, _attention
from test_gpu_serving import _meta, _rand, _run

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a ROCm GPU")]

PATHS = [(128, 16), (64, 32), (80, 16)]
SHORT, LONG = ([1, 3], [300, 200]), ([150, 2], [300, 90])   # narrow tiles alone; wide ones too


def _scaled(kb, D):
    """A scale with which keys of some 110 2^(kb - 127) score a few units."""
    return 2.0 ** (127 - kb) / (64 * D ** 0.5)


@pytest.mark.parametrize("D,page", PATHS)
@pytest.mark.parametrize("news,kvs", [SHORT, LONG])
@pytest.mark.parametrize("kb", [27, 60, 90, 95, 105, 111, 112, 118])
def test_float16_over_keys_of_small_powers(backend, D, page, news, kvs, kb):
    """Keys far below float16's smallest numbers, under a scale that brings their scores to a few units: the numbers that the
    pools hold enter the scores as they are."""
    bt = R.batch(news, kvs, page, seed=3)
    kp, vp, ks, vs = Q.pools8(bt, 2, page, D)
    ks = torch.where(ks == 255, ks, torch.full_like(ks, kb))
    _attention(backend, bt, 4, 2, D, "float16", page, pools=(kp, vp, ks, vs), scale=_scaled(kb, D))


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("D,page", PATHS)
@pytest.mark.parametrize("news,kvs", [SHORT, LONG, ([1], [3000]), ([200], [2000])])
@pytest.mark.parametrize("run", [1, 16, 64, 128])
def test_small_powers_beside_larger_ones(backend, dtype, D, page, news, kvs, run):
    """Positions in turn, ``run`` at a time, of large numbers with a small power, of small numbers with one 2^10 above it, and
    of numbers 2^20 above the first, at most 2^-9: every third stretch each, so that blocks, groups and neighbours differ in
    kind."""
    bt = R.batch(news, kvs, page, seed=5)
    kp, vp, ks, vs = Q.pools8(bt, 2, page, D)
    for b, s in enumerate(kvs):
        for p in range(s):
            pg, off = R.slot(bt, b, p, page)
            kind = p // run % 3
            ks[pg, :, off] = (92, 102, 112)[kind]
            if kind == 1:   # (exponents of 2^-4 to 2^-1 rather than 2^5 to 2^8)
                x = kp[pg, :, off]
                kp[pg, :, off] = (x & 0x87) | (((x >> 3) & 15).clamp(min=9) - 9 << 3)
            elif kind == 2:   # (multiples of 2^-9 up to 7 2^-9)
                kp[pg, :, off] &= 0x87
    _attention(backend, bt, 4, 2, D, dtype, page, pools=(kp, vp, ks, vs), scale=_scaled(92, D))


@pytest.mark.parametrize("D,page", PATHS)
@pytest.mark.parametrize("news,kvs", [SHORT, LONG])
@pytest.mark.parametrize("vb", [95, 105, 112])
def test_float16_over_values_of_small_powers(backend, D, page, news, kvs, vb):
    """Outputs below float16's normal numbers: half a step there, 2^-25, for the output, and another for the values, which a
    wide tile holds in float16."""
    from irgen.serving import build_paged_attention_ir

    bt = R.batch(news, kvs, page, seed=3)
    kp, vp, ks, vs = Q.pools8(bt, 2, page, D)
    vs = torch.where(vs == 255, vs, torch.full_like(vs, vb))
    pools = (kp, vp, ks, vs)
    q = _rand(9, bt["rows"], 4, D, dtype="float16")
    ir = build_paged_attention_ir(bt["rows"], len(news), bt["pages"], page, bt["block_table"].shape[1], 4, 2, D, "float16", cache=E4M3FN)
    got, = _run(ir, backend, {"q": q, **dict(zip(NAMES, pools)), **_meta(bt)})
    out, mag, big = Q.attention64(q, pools, bt, page, D ** -0.5)
    tol = Q.attention_tol("float16", D, max(kvs), out, mag, big, q, pools, bt, page) + 2 * 2.0 ** -25
    assert ((got.double() - out).abs() <= tol).all()
