"""Appends that norm heads, or quantise them, of heads and weights far from 1, and of metadata that is no batch.

Tolerances count roundings (``serving_ref``, ``quant_ref``)."""

import pytest
import torch

import quant_ref as Q
import serving_ref as R
import test_quant_ops as C
from conftest import gpu_available
from test_gpu_quant import E4M3FN, NAMES
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
