"""Pools of 8 bits and 64-bit forms of the operators over them, and of the appends that norm, for their tests."""

import numpy as np
import torch

import serving_ref as R

# half a step of a type is HALF_STEP of the value down to its smallest normal number, and this below: float16 has steps of 2^-24
# under 2^-14
LEAST_HALF = {"bfloat16": 2.0 ** -134, "float16": 2.0 ** -25, "float32": 2.0 ** -150}
E4M3 = 2.0 ** -4   # half a step of e4m3, relative; below 2^-6 half a step is 2^-10


def pools8(bt, kv_heads, page_size, head_dim, layout="hnd", seed=1, stale=True, powers=(117, 124)):
    """Random k and v pools of 8 bits and their power bytes. ``stale``: every place that holds no position of the batch is NaN,
    as a number and as a power."""
    g = torch.Generator().manual_seed(seed)
    pages, scales = [], []
    used = torch.zeros(bt["pages"], page_size, dtype=torch.bool)
    for b, s in enumerate(bt["kv_len"].tolist()):
        for p in range(s):
            at = R.slot(bt, b, p, page_size)
            if at is not None:
                used[at] = True
    for _ in range(2):
        x = (110 * torch.randn(bt["pages"], page_size, kv_heads, head_dim, generator=g)).clamp(-448, 448)
        x = x.to(torch.float8_e4m3fn).view(torch.uint8)
        s = torch.randint(*powers, (bt["pages"], kv_heads, page_size), generator=g).to(torch.uint8)
        if stale:
            x[~used] = 0x7f
            s.transpose(1, 2)[~used] = 255
        pages.append(x if layout == "nhd" else x.transpose(1, 2).contiguous())
        scales.append(s)
    return pages[0], pages[1], scales[0], scales[1]


def numbers(pages, scales, layout="hnd"):
    """What a pool of 8 bits holds, in 64 bits."""
    s = torch.where(scales == 255, torch.nan, torch.where(scales == 0, 0.0, 2.0 ** (scales.double() - 127)))
    s = s if layout == "hnd" else s.transpose(1, 2)
    return pages.view(torch.float8_e4m3fn).double() * s[..., None]


def normed(x, weight, eps):
    x = x.double().numpy()
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight.double().numpy()


def turned(x, p, inv, scaling):
    """(rotated heads [h, D], sum of the magnitudes that each element adds up) of float64 heads at position p."""
    r = inv.size
    c, s = scaling * np.cos(p * inv), scaling * np.sin(p * inv)
    y, mag = x.copy(), np.abs(x)
    y[:, :r], y[:, r:2 * r] = x[:, :r] * c - x[:, r:2 * r] * s, x[:, r:2 * r] * c + x[:, :r] * s
    lo, hi = np.abs(x[:, :r]), np.abs(x[:, r:2 * r])
    mag[:, :r], mag[:, r:2 * r] = (lo + hi) * abs(scaling), (lo + hi) * abs(scaling)
    return y, mag


def fp32(D):
    """What 32-bit arithmetic may add to a normed and rotated element, relative to ``turned``'s magnitudes: the sum of D
    squares (D halves, as its root enters), quotient, root and products (6), cosine and product (4), one more for the sum."""
    return 1.01 * (D / 2 + 12) * 2.0 ** -24


def append64(q, k, v, bt, inv_freq, page_size, scaling=1.0, weights=None, eps=0.0):
    """({row: (heads of q, magnitudes)}, {place: ((k, magnitudes), (v, 0))}) in float64."""
    inv = inv_freq.double().numpy()
    q64 = q.double().numpy() if weights is None else normed(q, weights[0], eps)
    k64 = k.double().numpy() if weights is None else normed(k, weights[1], eps)
    rows, at = {}, {}
    for row, b, p in R.places(bt, page_size):
        rows[row] = turned(q64[row], p, inv, scaling)
        place = R.slot(bt, b, p, page_size)
        if place is not None:
            v64 = v[row].double().numpy()
            at[place] = (turned(k64[row], p, inv, scaling), (v64, 0 * v64))
    return rows, at


def check_rows(got, rows, dtype, D):
    """q's rows, one rounding each; zeros elsewhere."""
    got = got.double().numpy()
    for r in range(got.shape[0]):
        if r not in rows:
            assert (got[r] == 0).all()
            continue
        y, mag = rows[r]
        assert (np.abs(got[r] - y) <= np.maximum(1.001 * R.HALF_STEP[dtype] * np.abs(y), LEAST_HALF[dtype]) + fp32(D) * mag + 1e-30).all(), r


def check_places16(got, was, at, which, dtype, D, layout):
    by = lambda x: x if layout == "nhd" else x.transpose(1, 2)   # noqa: E731
    got, same = by(got), by(was).clone()
    for place, new in at.items():
        y, mag = new[which]
        g = got[place].double().numpy()
        assert (np.abs(g - y) <= np.maximum(1.001 * R.HALF_STEP[dtype] * np.abs(y), LEAST_HALF[dtype]) + fp32(D) * mag + 1e-30).all(), place
        same[place] = got[place]
    assert torch.equal(got, same)   # all other places are as they were


def check_places8(pages, scales, was_pages, was_scales, at, which, D, layout):
    """Each head's power is the smallest that holds it, each number half a step of e4m3 from x / power."""
    by = lambda x: x if layout == "nhd" else x.transpose(1, 2)   # noqa: E731
    pages, same = by(pages), by(was_pages).clone()
    scales, same_s = scales.transpose(1, 2), was_scales.transpose(1, 2).clone()
    for place, new in at.items():
        y, mag = new[which]
        err = fp32(D) * mag
        fin = np.isfinite(y)
        most = np.where(fin, np.abs(y), 0).max(-1)
        slack = np.where(fin, err, 0).max(-1)
        s = 2.0 ** (scales[place].double().numpy() - 127)
        assert (most - slack <= 448 * s).all() and ((most + slack > 224 * s) | (s == 2.0 ** -100)).all(), (place, most, s)
        g = pages[place].contiguous().view(torch.float8_e4m3fn).double().numpy() * s[:, None]
        assert (np.isnan(g) == ~fin).all(), place
        half = np.maximum(E4M3 * np.abs(y), 2.0 ** -10 * s[:, None])
        off = np.where(fin, np.abs(g - np.where(fin, y, 0)) - 1.001 * half - err, -1)
        assert (off <= 0).all(), (place, off.max())
        same[place], same_s[place] = pages[place], scales[place]
    assert torch.equal(pages, same) and torch.equal(scales, same_s)


def attention64(q, pools, bt, page_size, scale, layout="hnd"):
    k, v, ks, vs = pools
    return R.attention64(q, numbers(k, ks, layout), numbers(v, vs, layout), bt, page_size, scale, layout)


def attention_tol(dtype, D, S, out, mag, big, q, pools, bt, page_size, layout="hnd"):
    """``serving_ref.attention_tol``, and where probabilities go to the product in float16: they are taken times 2^7, the largest
    at least 2^7 then, and below 2^-14 float16 has steps of 2^-24. Half a step is 2^-32 of the largest, for the row's sum is no
    less than that, so each open value adds up to 2^-32 of itself."""
    tol = R.attention_tol(dtype, D, S, out, mag, big)
    if dtype != "float16":
        return tol
    V = numbers(pools[1], pools[3], layout)
    V = (V if layout == "nhd" else V.transpose(1, 2)).abs().nan_to_num()
    G, run = q.shape[1] // V.shape[2], {}
    more = torch.zeros_like(tol)
    for row, b, p in R.places(bt, page_size):
        if b not in run:
            at = [R.slot(bt, b, j, page_size) for j in range(int(bt["kv_len"][b]))]
            run[b] = torch.stack([V[a] if a is not None else torch.zeros_like(V[0, 0]) for a in at]).cumsum(0) if at else None
        if p >= 0:
            more[row] = 2.0 ** -32 * run[b][min(p, len(run[b]) - 1)].repeat_interleave(G, 0)
    return tol + more
