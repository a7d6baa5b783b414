"""Appends that norm heads, or quantise them, of heads and weights far from 1, and of metadata that is no batch.

Tolerances count roundings (``serving_ref``, ``quant_ref``)."""

import pytest
import torch

import quant_ref as Q
import serving_ref as R
import test_quant_ops as C
from conftest import gpu_available
from test_gpu_quant import E4M3FN, LIM, NAMES, _append
from test_gpu_serving import _inv, _meta, _rand, _run

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a ROCm GPU")]


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("news,kvs", [([5, 1], [30, 2]), ([1100], [1200])])
@pytest.mark.parametrize("size,weight", [(60, -90), (-50, 100), (-50, -60)])
def test_norms_whose_root_times_weight_is_no_number(backend, quant, news, kvs, size, weight):
    """Heads of about 2^size under weights of about 2^weight: the result is of the weights' size, whatever the product of the
    weight and the root mean square's inverse is."""
    from irgen.serving import build_paged_append_ir

    D, dtype = 64, "bfloat16"
    bt = R.batch(news, kvs, 16)
    x = [(_rand(i, bt["rows"], h, D) * 2.0 ** size).to(R.DT[dtype]) for i, h in enumerate((4, 2, 2))]
    ws = tuple(((1 + 0.3 * _rand(i, D)) * 2.0 ** weight).to(R.DT[dtype]) for i in (5, 6))
    pools = Q.pools8(bt, 2, 16, D) if quant else tuple(R.pools(bt, 2, 16, D, dtype))
    ir = build_paged_append_ir(bt["rows"], len(news), bt["pages"], 16, bt["block_table"].shape[1], 4, 2, D, dtype, rotary_dim=32,
                               norm_eps=0.0, cache=E4M3FN if quant else None)
    got = _run(ir, backend, {**dict(zip("qkv", x)), **dict(zip(NAMES, pools)), **_meta(bt), "inv_freq": _inv(16),
                             "q_weight": ws[0], "k_weight": ws[1]})
    C.check(got, pools, *x, bt, _inv(16), 16, D, dtype, "hnd", 1.0, ws, 0.0)


@pytest.mark.parametrize("D,dtype", [(128, "bfloat16"), (72, "float16")])
@pytest.mark.parametrize("norm,quant", [(True, False), (False, True), (True, True)])
@pytest.mark.parametrize("start,kv", [((0, 9, 4, 2, 38), (5, 5, 5, 5)), ((0, 1, 2, 3, 4), (LIM.min, LIM.max, 1 << 30, -1)),
                                      ((LIM.min, LIM.min, LIM.max, LIM.max, LIM.max), (3, LIM.max, 7, 9)),
                                      ((-4, 3, 3, 30, 90), (40, 0, 33, 70))])
def test_appends_of_any_metadata_write_the_places_that_rows_name(backend, norm, quant, D, dtype, start, kv):
    """Starts that descend, and starts and lengths at the ends of 32 bits: a row is of the sequence that as many starts do not pass,
    and only places that a row has by that are written."""
    page, r, scaling, eps = 16, 8, 1.25, 1e-6
    bt = R.batch([2, 30, 1, 1], [100, 90, 33, 20], page, pad=4, lead=3)
    meta = {"q_start": torch.tensor(start, dtype=torch.int32), "kv_len": torch.tensor(kv, dtype=torch.int32)}
    got, pools, (q, k, v), ws = _append(backend, bt, 4, 2, D, r, dtype, page, "hnd", norm, quant, change=meta)
    places, rows, at = {}, {}, {}
    for row in range(bt["rows"]):
        b = sum(s <= row for s in start[1:])
        if b < 4 and row >= start[0]:
            places[row] = b, max(kv[b] - (start[b + 1] - row), -(1 << 30))
    inv = _inv(r).double().numpy()
    q64, k64 = (x.double().numpy() if ws is None else Q.normed(x, w, eps) for x, w in zip((q, k), ws or (0, 0)))
    for row, (b, p) in places.items():
        rows[row] = Q.turned(q64[row], p, inv, scaling)
        place = R.slot(bt, b, p, page)
        if place is not None:
            assert place not in at
            v64 = v[row].double().numpy()
            at[place] = (Q.turned(k64[row], p, inv, scaling), (v64, 0 * v64))
    Q.check_rows(got[0], rows, dtype, D)
    for i in range(2):
        if quant:
            Q.check_places8(got[1 + i], got[3 + i], pools[i], pools[2 + i], at, i, D, "hnd")
        else:
            Q.check_places16(got[1 + i], pools[i], at, i, dtype, D, "hnd")
