"""The operators of a server that runs a decoder model for many requests at once, as torch custom ops.

No counterpart in the reference, which runs one sequence over a static cache and takes the argmax on the
host (`examples/run_qwen.py:84-200`). The ops are functional, like ``aten.index_copy``: IR nodes carry them under
their overload names, ``torch.export`` traces them, the CPU fallback runs the definitions below, and the HIP
backend lowers them to kernels that update caches in place where ``index_copy`` would.

Three tensors say which sequence a row belongs to (all int32):

* ``q_start`` [B + 1], non-decreasing: rows ``q_start[b] .. q_start[b + 1] - 1`` of the packed new tokens are
  sequence b's, none for an idle one. Rows of no sequence are padding: they are computed as zeros and
  written nowhere. Of a sequence that begins before the rows or ends behind them, those that there are count.
* ``kv_len`` [B]: positions in b's cache with the new tokens as the last of them, so that row
  ``q_start[b] + i`` of n sits at position ``kv_len[b] - n + i``.
* ``block_table`` [B, M]: position p of b lies in row ``p % page_size`` of page ``block_table[b, p // page_size]``.

The definitions below refuse a ``q_start`` that descends. A device takes the three as they come, since reading them
would wait for it: attention then gives zeros, append writes what it writes within the pools.

A position that has no place (before 0, past the table, in a page that is not one of the pool's) is not
written and is closed to attention: its key and value are not read, whatever they hold. Where two rows name
one place, each element of it is one of theirs. Pools are [P, KVH, page_size, D] (page_layout "hnd") or
[P, page_size, KVH, D] ("nhd").

Pools of 8 bits (the ``quant`` operators) are uint8 of the same shapes: bytes of e4m3 numbers (``torch.float8_e4m3fn``),
beside ``k_scales`` and ``v_scales``, uint8 [P, KVH, page_size] in either layout: a byte s per position and head stands
for the power of two 2^(s - 127) that its numbers are multiplied by (``torch.float8_e8m0fnu``, 255 is NaN; but 0, as places
that nothing was written to may hold, stands for 0). A power of two costs e4m3 no precision, since its steps are
relative, and is exact to divide and multiply by.

``norm`` operators divide each head of q and k by its root mean square first, as models do that norm their heads.
"""

from __future__ import annotations

import torch

LAYOUTS = ("hnd", "nhd")

_LIB = torch.library.Library("serving", "DEF")
_LIB.define("paged_append(Tensor q, Tensor k, Tensor v, Tensor k_pages, Tensor v_pages, Tensor block_table, "
            "Tensor q_start, Tensor kv_len, Tensor inv_freq, float attention_scaling=1.0, str page_layout=\"hnd\") "
            "-> (Tensor, Tensor, Tensor)")
_LIB.define("paged_attention(Tensor q, Tensor k_pages, Tensor v_pages, Tensor block_table, Tensor q_start, "
            "Tensor kv_len, float scale, str page_layout=\"hnd\") -> Tensor")
_CACHE8 = "Tensor k_pages, Tensor v_pages, Tensor k_scales, Tensor v_scales, Tensor block_table, Tensor q_start, Tensor kv_len, "
_LIB.define("paged_norm_append(Tensor q, Tensor k, Tensor v, Tensor q_weight, Tensor k_weight, Tensor k_pages, Tensor v_pages, "
            "Tensor block_table, Tensor q_start, Tensor kv_len, Tensor inv_freq, float eps, float attention_scaling=1.0, "
            "str page_layout=\"hnd\") -> (Tensor, Tensor, Tensor)")
_LIB.define("paged_quant_append(Tensor q, Tensor k, Tensor v, " + _CACHE8 + "Tensor inv_freq, float attention_scaling=1.0, "
            "str page_layout=\"hnd\") -> (Tensor, Tensor, Tensor, Tensor, Tensor)")
_LIB.define("paged_norm_quant_append(Tensor q, Tensor k, Tensor v, Tensor q_weight, Tensor k_weight, " + _CACHE8 +
            "Tensor inv_freq, float eps, float attention_scaling=1.0, str page_layout=\"hnd\") "
            "-> (Tensor, Tensor, Tensor, Tensor, Tensor)")
_LIB.define("paged_quant_attention(Tensor q, " + _CACHE8 + "float scale, str page_layout=\"hnd\") -> Tensor")
_LIB.define("sample(Tensor logits, Tensor temperature, Tensor top_k, Tensor top_p, Tensor min_p, Tensor u) -> Tensor")


# ---------------------------------------------------------------- what every backend checks

def _need(ok: bool, msg: str) -> None:
    if not ok:
        raise ValueError(msg)


def _is(t, name: str) -> bool:
    return str(t.dtype).replace("torch.", "") == name


def _check_pages(op: str, q, k_pages, v_pages, block_table, q_start, kv_len, page_layout: str, scales=None) -> None:
    _need(page_layout in LAYOUTS, f"{op}: page_layout {page_layout!r} is not one of {LAYOUTS}")
    _need(len(q.shape) == 3, f"{op}: q must be [rows, heads, head_dim], got {list(q.shape)}")
    _need(len(k_pages.shape) == 4 and tuple(k_pages.shape) == tuple(v_pages.shape),
          f"{op}: k_pages and v_pages must be pools of one 4-dimensional shape")
    kvh, page_size = (k_pages.shape[i] for i in ((1, 2) if page_layout == "hnd" else (2, 1)))
    _need(page_size > 0, f"{op}: pages of no position")
    _need(k_pages.shape[3] == q.shape[2], f"{op}: pools of head_dim {k_pages.shape[3]}, q of {q.shape[2]}")
    _need(kvh > 0 and q.shape[1] > 0 and q.shape[1] % kvh == 0, f"{op}: {q.shape[1]} query heads do not divide among {kvh} K/V heads")
    _need(len(kv_len.shape) == 1 and tuple(q_start.shape) == (kv_len.shape[0] + 1,)
          and len(block_table.shape) == 2 and block_table.shape[0] == kv_len.shape[0],
          f"{op}: need kv_len [B], q_start [B + 1] and block_table [B, M]")
    for name, t in (("block_table", block_table), ("q_start", q_start), ("kv_len", kv_len)):
        _need(_is(t, "int32"), f"{op}: {name} must be int32, got {t.dtype}")
    floating = any(_is(q, d) for d in ("bfloat16", "float16", "float32"))
    if scales is None:
        _need(str(q.dtype) == str(k_pages.dtype) == str(v_pages.dtype) and floating,
              f"{op}: q and the pools must share one floating type")
        return
    _need(floating, f"{op}: q must be bfloat16, float16 or float32, got {q.dtype}")
    for name, t in (("k_pages", k_pages), ("v_pages", v_pages), ("k_scales", scales[0]), ("v_scales", scales[1])):
        _need(_is(t, "uint8"), f"{op}: {name} must be uint8, got {t.dtype}")
    for name, t in (("k_scales", scales[0]), ("v_scales", scales[1])):
        _need(tuple(t.shape) == (k_pages.shape[0], kvh, page_size), f"{op}: {name} must be [{k_pages.shape[0]}, {kvh}, {page_size}]")


def check_paged_append(q, k, v, k_pages, v_pages, block_table, q_start, kv_len, inv_freq, page_layout: str, weights=None,
                       scales=None, eps=None) -> None:
    """Raise ``ValueError`` unless the operands (tensors, specs or views: shape and dtype are read) fit. ``weights``: (q_weight,
    k_weight) of the forms that norm, with their ``eps``; ``scales``: (k_scales, v_scales) of those that quantise."""
    op = "serving.paged_" + ("norm_" if weights else "") + ("quant_" if scales else "") + "append"
    _check_pages(op, q, k_pages, v_pages, block_table, q_start, kv_len, page_layout, scales)
    kvh = k_pages.shape[1 if page_layout == "hnd" else 2]
    if weights:
        for name, t in zip(("q_weight", "k_weight"), weights):
            _need(tuple(t.shape) == (q.shape[2],) and str(t.dtype) == str(q.dtype), f"{op}: {name} must be [{q.shape[2]}] of q's type")
        _need(eps >= 0, f"{op}: eps must not be negative, got {eps}")
    for name, t in (("k", k), ("v", v)):
        _need(tuple(t.shape) == (q.shape[0], kvh, q.shape[2]) and str(t.dtype) == str(q.dtype),
              f"{op}: {name} must be [{q.shape[0]}, {kvh}, {q.shape[2]}] of q's type")
    _need(len(inv_freq.shape) == 1 and _is(inv_freq, "float32") and 2 * inv_freq.shape[0] <= q.shape[2],
          f"{op}: inv_freq must be float32 [r] with 2 r <= head_dim")


def check_paged_attention(q, k_pages, v_pages, block_table, q_start, kv_len, page_layout: str) -> None:
    _check_pages("serving.paged_attention", q, k_pages, v_pages, block_table, q_start, kv_len, page_layout)


def check_paged_quant_attention(q, k_pages, v_pages, k_scales, v_scales, block_table, q_start, kv_len, page_layout: str) -> None:
    _check_pages("serving.paged_quant_attention", q, k_pages, v_pages, block_table, q_start, kv_len, page_layout,
                 (k_scales, v_scales))


def check_sample(logits, temperature, top_k, top_p, min_p, u) -> None:
    op = "serving.sample"
    _need(len(logits.shape) == 2 and logits.shape[1] > 0 and
          any(_is(logits, d) for d in ("bfloat16", "float16", "float32")),
          f"{op}: logits must be a floating [rows, vocab] with vocab > 0")
    for name, t, dt in (("temperature", temperature, "float32"), ("top_k", top_k, "int32"),
                        ("top_p", top_p, "float32"), ("min_p", min_p, "float32"), ("u", u, "float32")):
        _need(tuple(t.shape) == (logits.shape[0],) and _is(t, dt), f"{op}: {name} must be {dt} [{logits.shape[0]}]")


# ---------------------------------------------------------------- definitions (CPU)

def row_places(rows: int, q_start, kv_len):
    """(sequence, position) of each packed row, sequence -1 for padding."""
    s = q_start.long()
    _need(bool((s[1:] >= s[:-1]).all()), "q_start must be non-decreasing")
    r = torch.arange(rows)
    b = torch.searchsorted(s[1:].contiguous(), r, right=True)
    pad = (b >= kv_len.numel()) | (r < s[0])
    b = b.clamp(max=max(kv_len.numel() - 1, 0))
    if kv_len.numel() == 0:
        return torch.full((rows,), -1), torch.zeros(rows, dtype=torch.long)
    return torch.where(pad, -1, b), kv_len.long()[b] - s[b + 1] + r


def _slots(b, pos, block_table, pages: int, page_size: int):
    """(page, row in it, whether the place exists) of position ``pos`` of sequence ``b``, elementwise."""
    M = block_table.shape[1]
    ok = (b >= 0) & (pos >= 0) & (pos < M * page_size)
    if M == 0 or block_table.shape[0] == 0:
        return torch.zeros_like(pos), torch.zeros_like(pos), torch.zeros_like(ok)
    at = torch.where(ok, pos, 0)
    page = block_table.long()[b.clamp(min=0), at // page_size]
    ok = ok & (page >= 0) & (page < pages)
    return torch.where(ok, page, 0), at % page_size, ok


def _by_token(pool, page_layout: str):
    """The pool as [P, page_size, KVH, D]."""
    return pool if page_layout == "nhd" else pool.transpose(1, 2)


def paged_append(q, k, v, k_pages, v_pages, block_table, q_start, kv_len, inv_freq, attention_scaling=1.0,
                 page_layout="hnd"):
    """Rotate q and k to their rows' positions and write k and v into the pages.

    With f = position * inv_freq[j] (exact, not rounded to 32 bits: an angle of position 100,000 would be off by
    4e-3), c = s cos f, d = s sin f and r = inv_freq's length: x'[j] = x[j] c - x[j + r] d,
    x'[j + r] = x[j + r] c + x[j] d for j < r, the dimensions from 2 r on as they are, one rounding at the
    end. Returns (rotated q, k_pages, v_pages)."""
    check_paged_append(q, k, v, k_pages, v_pages, block_table, q_start, kv_len, inv_freq, page_layout)
    return _append(q, k, v, k_pages, v_pages, block_table, q_start, kv_len, inv_freq, attention_scaling, page_layout)


def paged_norm_append(q, k, v, q_weight, k_weight, k_pages, v_pages, block_table, q_start, kv_len, inv_freq, eps,
                      attention_scaling=1.0, page_layout="hnd"):
    """``paged_append`` of heads that are normed first: x / sqrt(mean(x^2) + eps) * weight over a head's dimensions, in 32
    bits, not rounded before the rotation."""
    check_paged_append(q, k, v, k_pages, v_pages, block_table, q_start, kv_len, inv_freq, page_layout, (q_weight, k_weight), eps=eps)
    return _append(q, k, v, k_pages, v_pages, block_table, q_start, kv_len, inv_freq, attention_scaling, page_layout,
                   (q_weight, k_weight), eps)


def paged_quant_append(q, k, v, k_pages, v_pages, k_scales, v_scales, block_table, q_start, kv_len, inv_freq,
                       attention_scaling=1.0, page_layout="hnd"):
    """``paged_append`` into pools of 8 bits. Of each head's k (rotated, unrounded) and v: s = 2^e with the smallest e >= -100
    for which its largest finite magnitude is at most 448 s, then x / s rounded to e4m3 once; NaN and infinities become
    NaN. Returns (rotated q, k_pages, v_pages, k_scales, v_scales). Where two rows name one place, its numbers and its power
    may be of different rows."""
    check_paged_append(q, k, v, k_pages, v_pages, block_table, q_start, kv_len, inv_freq, page_layout, scales=(k_scales, v_scales))
    return _append(q, k, v, k_pages, v_pages, block_table, q_start, kv_len, inv_freq, attention_scaling, page_layout,
                   scales=(k_scales, v_scales))


def paged_norm_quant_append(q, k, v, q_weight, k_weight, k_pages, v_pages, k_scales, v_scales, block_table, q_start, kv_len,
                            inv_freq, eps, attention_scaling=1.0, page_layout="hnd"):
    """``paged_quant_append`` of heads normed as by ``paged_norm_append``."""
    check_paged_append(q, k, v, k_pages, v_pages, block_table, q_start, kv_len, inv_freq, page_layout, (q_weight, k_weight),
                       (k_scales, v_scales), eps)
    return _append(q, k, v, k_pages, v_pages, block_table, q_start, kv_len, inv_freq, attention_scaling, page_layout,
                   (q_weight, k_weight), eps, (k_scales, v_scales))


def quantise(x):
    """(bytes of e4m3 numbers, byte of the power of two) of heads [..., D], as ``paged_quant_append`` defines them."""
    x = x.float()
    m, two = torch.frexp(torch.where(x.isfinite(), x.abs(), torch.zeros(())).amax(-1).clamp(min=2.0 ** -92))
    e = two - 9 + (m > 0.875)   # m 2^two <= 448 2^e = 0.875 2^(9 + e)
    return torch.ldexp(x, -e[..., None]).to(torch.float8_e4m3fn).view(torch.uint8), (e + 127).to(torch.uint8)


def dequantise(pages, scales, page_layout="hnd"):
    """float32 pools of the numbers that pools of 8 bits hold."""
    s = torch.where(scales == 0, torch.zeros(()), scales.view(torch.float8_e8m0fnu).float())
    s = (s if page_layout == "hnd" else s.transpose(1, 2))[..., None]
    return pages.view(torch.float8_e4m3fn).float() * s


def _append(q, k, v, k_pages, v_pages, block_table, q_start, kv_len, inv_freq, attention_scaling, page_layout, weights=None,
            eps=0.0, scales=None):
    b, pos = row_places(q.shape[0], q_start, kv_len)
    r = inv_freq.shape[0]
    f = pos[:, None].double() * inv_freq.double()
    c = (f.cos() * attention_scaling).float()[:, None]
    d = (f.sin() * attention_scaling).float()[:, None]

    def normed(x, i):
        x = x.float()
        return x if weights is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * weights[i].float()

    def rotated(x):
        lo, hi, rest = x[..., :r], x[..., r:2 * r], x[..., 2 * r:]
        return torch.cat([lo * c - hi * d, hi * c + lo * d, rest], -1)

    q_out = torch.where((b >= 0)[:, None, None], rotated(normed(q, 0)), torch.zeros(())).to(q.dtype)
    ps = k_pages.shape[2 if page_layout == "hnd" else 1]
    page, off, ok = _slots(b, pos, block_table, k_pages.shape[0], ps)
    pools, powers = [], []
    for i, (pool, new) in enumerate(((k_pages, rotated(normed(k, 1))), (v_pages, v))):
        pool = pool.clone()
        if scales is not None:
            new, s = quantise(new)
            powers.append(scales[i].clone())
            powers[i].transpose(1, 2)[page[ok], off[ok]] = s[ok]
        _by_token(pool, page_layout)[page[ok], off[ok]] = new[ok].to(pool.dtype)
        pools.append(pool)
    return (q_out, *pools, *powers)


def paged_attention(q, k_pages, v_pages, block_table, q_start, kv_len, scale, page_layout="hnd"):
    """softmax(scale q . k) v over the positions up to each row's own; query heads h of one K/V head h // (H / KVH)
    share its pages. A row with no open position is zero, and so is one whose open positions all score -inf."""
    check_paged_attention(q, k_pages, v_pages, block_table, q_start, kv_len, page_layout)
    return _attention(q, k_pages, v_pages, block_table, q_start, kv_len, scale, page_layout)


def paged_quant_attention(q, k_pages, v_pages, k_scales, v_scales, block_table, q_start, kv_len, scale, page_layout="hnd"):
    """``paged_attention`` over the numbers that pools of 8 bits hold. A power byte of 255 makes them NaN. They, and their
    products with q before the scale, are held in 32 bits; where q is float16, a device may round values below 2^-14 to
    multiples of 2^-24, as such outputs are."""
    check_paged_quant_attention(q, k_pages, v_pages, k_scales, v_scales, block_table, q_start, kv_len, page_layout)
    return _attention(q, dequantise(k_pages, k_scales, page_layout), dequantise(v_pages, v_scales, page_layout), block_table,
                      q_start, kv_len, scale, page_layout)


def _attention(q, k_pages, v_pages, block_table, q_start, kv_len, scale, page_layout):
    N, H, D = q.shape
    K, V = _by_token(k_pages, page_layout), _by_token(v_pages, page_layout)
    G = H // K.shape[2]
    seq, pos = row_places(N, q_start, kv_len)
    out = torch.zeros(N, H, D)
    for b in range(kv_len.numel()):
        rows = (seq == b).nonzero()[:, 0]
        S = min(int(kv_len[b]), block_table.shape[1] * K.shape[1])   # (no places past the table)
        if rows.numel() == 0 or S <= 0:
            continue
        p = torch.arange(S)
        page, off, ok = _slots(torch.full_like(p, b), p, block_table, K.shape[0], K.shape[1])
        k = K[page, off].float().transpose(0, 1)   # [KVH, S, D]
        v = torch.where(ok[:, None, None], V[page, off].float(), torch.zeros(())).transpose(0, 1)
        open_ = ok & (p <= pos[rows][:, None])   # [n, S]
        qq = q[rows].float().reshape(len(rows), -1, G, D).permute(1, 2, 0, 3)   # [KVH, G, n, D]
        s = (qq @ k.transpose(1, 2).unsqueeze(1)) * scale
        s = s.masked_fill(~open_, float("-inf"))
        m = s.amax(-1, keepdim=True)
        e = torch.where(open_, (s - torch.where(m == float("-inf"), torch.zeros(()), m)).exp(), torch.zeros(()))
        z = e.sum(-1, keepdim=True)
        o = (e @ v.unsqueeze(1)) / torch.where(z == 0, torch.ones(()), z)
        out[rows] = o.permute(2, 0, 1, 3).reshape(len(rows), H, D)
    return out.to(q.dtype)


def sample(logits, temperature, top_k, top_p, min_p, u):
    """One token per row from the uniform number ``u`` in [0, 1) (0 where it is negative or NaN), int64 [rows].

    Tokens are ranked by logit, the lower index first among equals, and weigh w = exp((l - max) / temperature).
    ``top_k`` keeps the first k (all for k <= 0); ``top_p`` < 1 of these the ones whose preceding weights sum to
    less than top_p times the sum of them all; ``min_p`` those of weight >= min_p (the largest weight is 1).
    The first ranked is always kept. The token is the first, by index, at which the running sum of the kept
    weights passes u times their sum (the last of positive weight where none does). ``temperature`` <= 0 or NaN
    takes the first ranked; ``top_p`` and ``min_p`` that are NaN keep all. A NaN logit counts as -inf; where some are
    +inf they alone weigh, 1 each; a row without any number gives 0. Weights and sums are held in 64 bits."""
    check_sample(logits, temperature, top_k, top_p, min_p, u)
    x = logits.double()
    x = torch.where(x.isnan(), -torch.inf, x)
    B, V = x.shape
    if B == 0:
        return torch.zeros(0, dtype=torch.int64)
    s, order = torch.sort(x, dim=1, descending=True, stable=True)
    top = s[:, :1]
    T = temperature.double()[:, None]
    greedy = ~(T > 0) | (top == -torch.inf)
    # (inf - inf: the infinite logits weigh 1, all others 0)
    d = torch.where(s == top, 0.0, s - top)
    z = torch.where(d == -torch.inf, d, d / torch.where(T > 0, T, 1.0))
    w = z.exp()
    rank = torch.arange(V)
    k, p, m = top_k.long()[:, None], top_p.double()[:, None], min_p.double()[:, None].clamp(max=1.0)
    w = torch.where((k <= 0) | (rank < k), w, 0.0)
    run = w.cumsum(1)
    before = torch.cat([torch.zeros(B, 1, dtype=torch.float64), run[:, :-1]], 1)
    kept = (~(p < 1) | (before < p * run[:, -1:])) & ~(w < m)
    kept[:, 0] = True
    w = torch.where(kept, w, 0.0)
    byidx = torch.zeros_like(w).scatter_(1, order, w)
    c = byidx.cumsum(1)
    u = torch.where(u > 0, u, torch.zeros(())).double()[:, None]
    token = (c <= u * c[:, -1:]).sum(1)
    last = torch.where(byidx > 0, rank, 0).amax(1)
    return torch.where(greedy[:, 0], order[:, 0], torch.minimum(token, last))


# ---------------------------------------------------------------- shapes (meta)

def _paged_append_meta(q, k, v, k_pages, v_pages, block_table, q_start, kv_len, inv_freq, attention_scaling=1.0,
                       page_layout="hnd"):
    check_paged_append(q, k, v, k_pages, v_pages, block_table, q_start, kv_len, inv_freq, page_layout)
    return _like(q, k_pages, v_pages)


def _like(*ts):
    return tuple(torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in ts)


def _paged_norm_append_meta(q, k, v, q_weight, k_weight, k_pages, v_pages, block_table, q_start, kv_len, inv_freq, eps,
                            attention_scaling=1.0, page_layout="hnd"):
    check_paged_append(q, k, v, k_pages, v_pages, block_table, q_start, kv_len, inv_freq, page_layout, (q_weight, k_weight), eps=eps)
    return _like(q, k_pages, v_pages)


def _paged_quant_append_meta(q, k, v, k_pages, v_pages, k_scales, v_scales, block_table, q_start, kv_len, inv_freq,
                             attention_scaling=1.0, page_layout="hnd"):
    check_paged_append(q, k, v, k_pages, v_pages, block_table, q_start, kv_len, inv_freq, page_layout, scales=(k_scales, v_scales))
    return _like(q, k_pages, v_pages, k_scales, v_scales)


def _paged_norm_quant_append_meta(q, k, v, q_weight, k_weight, k_pages, v_pages, k_scales, v_scales, block_table, q_start,
                                  kv_len, inv_freq, eps, attention_scaling=1.0, page_layout="hnd"):
    check_paged_append(q, k, v, k_pages, v_pages, block_table, q_start, kv_len, inv_freq, page_layout, (q_weight, k_weight),
                       (k_scales, v_scales), eps)
    return _like(q, k_pages, v_pages, k_scales, v_scales)


def _paged_quant_attention_meta(q, k_pages, v_pages, k_scales, v_scales, block_table, q_start, kv_len, scale, page_layout="hnd"):
    check_paged_quant_attention(q, k_pages, v_pages, k_scales, v_scales, block_table, q_start, kv_len, page_layout)
    return _like(q)[0]


def _paged_attention_meta(q, k_pages, v_pages, block_table, q_start, kv_len, scale, page_layout="hnd"):
    check_paged_attention(q, k_pages, v_pages, block_table, q_start, kv_len, page_layout)
    return torch.empty(q.shape, dtype=q.dtype, device=q.device)


def _sample_meta(logits, temperature, top_k, top_p, min_p, u):
    check_sample(logits, temperature, top_k, top_p, min_p, u)
    return torch.empty(logits.shape[0], dtype=torch.int64, device=logits.device)


for _name, _cpu, _meta in (("paged_append", paged_append, _paged_append_meta),
                           ("paged_norm_append", paged_norm_append, _paged_norm_append_meta),
                           ("paged_quant_append", paged_quant_append, _paged_quant_append_meta),
                           ("paged_norm_quant_append", paged_norm_quant_append, _paged_norm_quant_append_meta),
                           ("paged_attention", paged_attention, _paged_attention_meta),
                           ("paged_quant_attention", paged_quant_attention, _paged_quant_attention_meta),
                           ("sample", sample, _sample_meta)):
    _LIB.impl(_name, _cpu, "CPU")
    _LIB.impl(_name, _meta, "Meta")
