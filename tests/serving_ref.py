"""Batches of packed rows and plain 64-bit forms of the serving operators for their tests, written row by row and
without torch ops in common with ``npu_runtime.serving_ops``."""

import math

import numpy as np
import torch

DT = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
HALF_STEP = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11, "float32": 2.0 ** -24}   # largest relative rounding


def batch(news, kvs, page_size, pad=0, spare=2, seed=0, extra_pages=1, lead=0):
    """A batch of sequences with ``news`` new tokens and ``kvs`` positions, pages in random order, ``lead`` rows before
    the first sequence and ``pad`` behind the last. Table entries past a sequence's end hold -1."""
    g = torch.Generator().manual_seed(seed)
    counts = [-(-s // page_size) for s in kvs]
    P, M = sum(counts) + spare, max(counts + [0]) + extra_pages
    free = torch.randperm(P, generator=g).tolist()
    table = torch.full((len(kvs), M), -1, dtype=torch.int32)
    for b, c in enumerate(counts):
        table[b, :c] = torch.tensor([free.pop() for _ in range(c)], dtype=torch.int32)
    start = np.concatenate([[lead], lead + np.cumsum(news)]) if len(news) else np.array([lead])
    return {"block_table": table, "q_start": torch.tensor(start, dtype=torch.int32),
            "kv_len": torch.tensor(kvs, dtype=torch.int32), "rows": int(start[-1]) + pad, "pages": P}


def pools(bt, kv_heads, page_size, head_dim, dtype, layout="hnd", seed=1, stale=None):
    """Random k and v pools; ``stale`` fills every place that holds no position of the batch."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for _ in range(2):
        x = torch.randn(bt["pages"], page_size, kv_heads, head_dim, generator=g).to(DT[dtype])
        if stale is not None:
            used = torch.zeros(bt["pages"], page_size, dtype=torch.bool)
            for b, s in enumerate(bt["kv_len"].tolist()):
                for p in range(s):
                    page = int(bt["block_table"][b, p // page_size])
                    if 0 <= page < bt["pages"]:
                        used[page, p % page_size] = True
            x[~used] = stale
        out.append(x if layout == "nhd" else x.transpose(1, 2).contiguous())
    return out


def places(bt, page_size):
    """(row, sequence, position) of every row of a sequence."""
    s, kv = bt["q_start"].tolist(), bt["kv_len"].tolist()
    return [(r, b, kv[b] - s[b + 1] + r) for b in range(len(kv)) for r in range(s[b], s[b + 1])]


def slot(bt, b, p, page_size):
    """(page, row) of position p, or None."""
    if not 0 <= p < bt["block_table"].shape[1] * page_size:
        return None
    page = int(bt["block_table"][b, p // page_size])
    return (page, p % page_size) if 0 <= page < bt["pages"] else None


def append64(q, k, v, kp, vp, bt, inv_freq, page_size, layout="hnd", scaling=1.0):
    """(rotated q, k pages, v pages, bound on what the fp32 arithmetic may add to q and k) in float64."""
    kp, vp = kp.double().numpy().copy(), vp.double().numpy().copy()
    q64, k64, v64, inv = q.double().numpy(), k.double().numpy(), v.double().numpy(), inv_freq.double().numpy()
    out, r = np.zeros_like(q64), inv.size

    def turn(x, p):
        c, s = scaling * np.cos(p * inv), scaling * np.sin(p * inv)
        y = x.copy()
        y[:, :r], y[:, r:2 * r] = x[:, :r] * c - x[:, r:2 * r] * s, x[:, r:2 * r] * c + x[:, :r] * s
        return y

    for row, b, p in places(bt, page_size):
        out[row] = turn(q64[row], p)
        at = slot(bt, b, p, page_size)
        if at is None:
            continue
        for pool, new in ((kp, turn(k64[row], p)), (vp, v64[row])):
            if layout == "hnd":
                pool[at[0], :, at[1]] = new
            else:
                pool[at[0], at[1]] = new
    return out, kp, vp


def attention64(q, kp, vp, bt, page_size, scale, layout="hnd"):
    """(output, sum of p |v|, sum of |q| |k| scaled and largest over the open positions) per row and head, float64."""
    N, H, D = q.shape
    K, V = ((x if layout == "nhd" else x.transpose(1, 2)).double() for x in (kp, vp))
    G = H // K.shape[2]
    out, mag, big = (torch.zeros(N, H, D, dtype=torch.float64), torch.zeros(N, H, D, dtype=torch.float64),
                     torch.zeros(N, H, 1, dtype=torch.float64))
    for row, b, p in places(bt, page_size):
        at = [a for a in (slot(bt, b, j, page_size) for j in range(p + 1)) if a is not None]
        if not at:
            continue
        pg, off = torch.tensor([a[0] for a in at]), torch.tensor([a[1] for a in at])
        for h in range(H):
            kk, vv, qq = K[pg, off, h // G], V[pg, off, h // G], q[row, h].double()
            w = torch.softmax(kk @ qq * scale, 0)
            out[row, h], mag[row, h] = w @ vv, w @ vv.abs()
            big[row, h] = (kk.abs() @ qq.abs()).max() * abs(scale)
    return out, mag, big


def attention_tol(dtype, D, S, out, mag, big):
    """What the roundings may add: the output's one (u |o|), one of each probability before the product with the
    values where it is taken in 16 bits (u sum p |v|), and 32-bit sums: (D + 4) 2^-24 of a score's magnitude moves its
    exponential by as much, twice with the normalising sum's, and the two sums over positions (S + 8) 2^-24 each."""
    u = HALF_STEP[dtype]
    fp32 = 2.0 ** -23 * ((D + 4) * big + S + 16)
    return 1.01 * (u * out.abs() + (u + fp32) * mag) + 1e-30


def sample64(logits, temperature, top_k, top_p, min_p, u):
    """Row by row in numpy: rank, cut, walk."""
    tokens = []
    for x, T, k, p, m, r in zip(logits.double().numpy(), *(t.double().numpy() for t in (temperature, top_k, top_p, min_p, u))):
        x = np.where(np.isnan(x), -np.inf, x)
        ranked = np.lexsort((np.arange(x.size), -x))
        top = x[ranked[0]]
        if not T > 0 or top == -np.inf:
            tokens.append(int(ranked[0]))
            continue
        w = np.array([1.0 if v == top else 0.0 if v == -np.inf else math.exp((v - top) / T) for v in x])
        if 0 < k < x.size:
            ranked = ranked[:int(k)]
        if p < 1:
            total, run, n = math.fsum(w[ranked]), 0.0, 0
            while n < ranked.size and run < p * total:
                run += w[ranked[n]]
                n += 1
            ranked = ranked[:max(n, 1)]
        ranked = np.sort([i for i in ranked if not w[i] < min(m, 1.0)])
        c = np.cumsum(w[ranked])
        i = int(np.searchsorted(c, r * c[-1], side="right"))
        positive = np.nonzero(w[ranked] > 0)[0]
        tokens.append(int(ranked[min(i, positive[-1])]))
    return torch.tensor(tokens)
