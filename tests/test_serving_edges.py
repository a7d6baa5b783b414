"""The serving operators at the edges of what their arguments may be: definitions, refusals and lowering on the CPU."""

import pytest
import torch

import serving_ref as R
from npu_runtime.serving_ops import paged_attention


@pytest.mark.parametrize("news,kvs,before,behind", [([4, 1, 40, 3], [30, 9, 300, 8], 2, 20), ([6], [40], 2, 0),
                                                    ([70, 0, 90], [700, 3, 91], 33, 40)])
def test_sequences_that_reach_past_the_rows(news, kvs, before, behind):
    bt = R.batch(news, kvs, 16, seed=1)
    kp, vp = R.pools(bt, 2, 16, 32, "float32", stale=float("nan"))
    q = torch.randn(bt["rows"], 4, 32, generator=torch.Generator().manual_seed(2))
    cut = slice(before, bt["rows"] - behind)
    out, mag, big = (t[cut] for t in R.attention64(q, kp, vp, bt, 16, 32 ** -0.5))
    got = paged_attention(q[cut], kp, vp, bt["block_table"], bt["q_start"] - before, bt["kv_len"], 32 ** -0.5)
    assert ((got.double() - out).abs() <= R.attention_tol("float32", 32, max(kvs), out, mag, big)).all()
