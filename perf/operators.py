"""What is timed when the serving operators are measured: one call of one operator, as cases.

A server that runs a decoder model for many requests at once calls three operators besides the layers'
linears. Their metadata is the same: the new tokens of all sequences are packed into rows, sequence ``b``
owning rows ``q_start[b] .. q_start[b + 1] - 1``; its cache holds ``kv_len[b]`` positions, the new ones the
last of them, and position ``p`` lies in page ``block_table[b, p // page]``. Rows from ``q_start[-1]`` on
are padding (a captured graph's unused slots); sequences without new tokens are idle slots.

kinds:

* ``append``     q and k rotated to their positions, k and v written into the pages.
* ``attention``  causal attention of the new tokens over the pages, ``heads / kv_heads`` heads per K/V head.
* ``sample``     one token per row of logits from a uniform number, after temperature, top-k, top-p and min-p.
"""

from __future__ import annotations

import math
import os
import random
import sys

import numpy as np
import torch

_PKG = os.path.join(os.getcwd(), "pytorch-apple_amd")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

own = False

THETA = 1e6
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
_BATCH = {"seqs": 1, "decodes": 0, "idle": 0, "new": 1, "context": 0, "pad": 0, "lengths": 0, "heads": 12, "kv_heads": 2,
          "head_dim": 128, "page": 16, "layout": "hnd", "dtype": "bfloat16"}


def _case(name, kind, **kw):
    base = _BATCH if kind != "sample" else {"rows": 1, "vocab": 151936, "dtype": "bfloat16"}
    return {"name": name, "kind": kind, **base, **kw}


def listed():
    return [
        # one request, one token: what a chat with a single user pays per layer for the cache update
        _case("append_one_token", "append", seqs=1, decodes=1, context=2047),
        # a server's step: most slots decode, two prompts come in, two slots are idle, the graph has spare rows
        _case("append_mixed", "append", seqs=48, decodes=44, idle=2, new=700, context=4000, pad=37, heads=14, head_dim=64,
              page=32, dtype="float16", lengths=1),
        # a batch of whole prompts, the pages kept token by token
        _case("append_prompts", "append", seqs=6, new=1500, heads=32, kv_heads=8, page=64, layout="nhd", lengths=2),
        # one request, one token over a short cache: latency
        _case("attention_one_token", "attention", seqs=1, decodes=1, context=2047),
        # a full decode batch over ragged caches of a few thousand positions
        _case("attention_decode_64", "attention", seqs=64, decodes=64, context=4096, heads=32, kv_heads=8, dtype="float16",
              lengths=3),
        # few requests with very long documents
        _case("attention_decode_long", "attention", seqs=4, decodes=4, context=131071, page=64, lengths=4),
        # the next chunk of a long prompt
        _case("attention_chunk_long", "attention", seqs=1, new=500, context=30000, layout="nhd", page=32, lengths=5),
        # a batch of whole prompts
        _case("attention_prompts", "attention", seqs=6, new=1500, heads=32, kv_heads=8, page=64, lengths=2),
        # a server's step: decoding slots beside a prompt chunk, idle slots and spare rows
        _case("attention_mixed", "attention", seqs=64, decodes=60, idle=3, new=448, context=4000, pad=21, heads=14,
              head_dim=64, page=32, dtype="float16", lengths=6),
        # one request's next token
        _case("sample_one_row", "sample"),
        # a large batch's next tokens, from logits kept in 32 bits
        _case("sample_256_rows", "sample", rows=256, dtype="float32"),
        # a middling batch over a small odd vocabulary
        _case("sample_odd_vocab", "sample", rows=33, vocab=50021, dtype="float16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "sample"])
    if kind == "sample":
        vocab = _log(rng, 1000, 152000)
        c = _case("", kind, rows=_log(rng, 1, min(256, 256 * 151936 // vocab)), vocab=vocab,
                  dtype=rng.choice(["bfloat16", "float16", "float32"]))
        del c["name"]
        return c
    heads, kv_heads, dim = rng.choice([(12, 2, 128), (14, 2, 64), (32, 8, 128), (8, 8, 64), (16, 1, 128), (40, 8, 128)])
    seqs = _log(rng, 1, 64)
    decodes = rng.choice([seqs, seqs, rng.randint(0, seqs), max(0, seqs - 1)])
    while True:
        new = _log(rng, 2, 2000) if decodes < seqs else 1
        context = rng.choice([0, _log(rng, 16, 32000)]) if decodes < seqs else _log(rng, 16, 120000)
        c = _case("", kind, seqs=seqs, decodes=decodes, idle=rng.choice([0, rng.randint(0, (seqs - 1) // 4)]), new=new,
                  context=context, pad=rng.choice([0, rng.randint(0, 40)]), lengths=rng.randint(0, 1 << 30), heads=heads,
                  kv_heads=kv_heads, head_dim=dim, page=rng.choice([16, 32, 48, 64, 128]),
                  layout=rng.choice(["hnd", "hnd", "nhd"]), dtype=rng.choice(["bfloat16", "float16"]))
        n, kv = _lengths(c)
        scores = seqs * heads * max(n) * (max(kv) + 1)
        w = work(c)
        if max(n) > 0 and sum(n) <= 6000 and scores <= 1 << 29 and w["bytes"] <= 4 << 27 and w["flops"] <= 9e10 and \
                _pages(c, kv) * c["page"] * kv_heads * dim <= 1 << 28:
            del c["name"]
            return c


def _lengths(case):
    """New tokens and cache length (the new ones counted) of every sequence: the case's own, not the seed's."""
    r = random.Random(case["lengths"])
    B = case["seqs"]
    n = [1] * case["decodes"] + [r.randint(max(1, case["new"] // 2), case["new"]) for _ in range(B - case["decodes"])]
    past = [r.randint((case["context"] + 1) // 2, case["context"]) for _ in range(B)]
    if B == 1:
        past = [case["context"]]
    for b in r.sample(range(case["decodes"]), min(case["idle"], case["decodes"])):
        n[b] = 0
    order = list(range(B))
    r.shuffle(order)
    n = [n[b] for b in order]
    return n, [p + k for p, k in zip(past, n)]


def _table_pages(case, kv):
    return -(-max(kv) // case["page"]) + 1


def _pages(case, kv):
    return sum(-(-s // case["page"]) for s in kv) + 3


def _rows(case, n):
    return sum(n) + case["pad"]


# ---------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _inputs(case, seed):
    g, dt = _gen(seed), DTYPES[case["dtype"]]

    def normal(shape, std=1.0):
        return torch.empty(shape, dtype=dt, device="cuda").normal_(0.0, std, generator=g)

    if case["kind"] == "sample":
        B, V = case["rows"], case["vocab"]
        x = torch.empty((B, V), device="cuda").normal_(0.0, 2.0, generator=g)
        peaks = torch.randint(0, V, (B, 24), device="cuda", generator=g)   # the few tokens that a model is sure of
        x.scatter_add_(1, peaks, 4.0 + 6.0 * torch.rand((B, 24), device="cuda", generator=g))
        r = random.Random(seed)
        f = lambda vals, t: torch.tensor([r.choice(vals) for _ in range(B)], dtype=t, device="cuda")
        return {"logits": x.to(dt), "temperature": f([0.7, 0.7, 1.0, 1.0, 1.3, 0.0 if B > 1 else 1.0], torch.float32),
                "top_k": f([0, 0, 20, 50, 1000], torch.int32), "top_p": f([1.0, 0.95, 0.95, 0.8], torch.float32),
                "min_p": f([0.0, 0.0, 0.05], torch.float32), "u": torch.rand(B, device="cuda", generator=g)}
    n, kv = _lengths(case)
    N, P, M = _rows(case, n), _pages(case, kv), _table_pages(case, kv)
    H, KVH, D, ps = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    pool = (P, KVH, ps, D) if case["layout"] == "hnd" else (P, ps, KVH, D)
    q = normal((N, H, D), 1.5 if case["kind"] == "attention" else 1.0)
    t = {"q": q}
    if case["kind"] == "append":
        t["k"], t["v"] = normal((N, KVH, D)), normal((N, KVH, D))
        t["inv_freq"] = 1.0 / THETA ** (torch.arange(0, D, 2, dtype=torch.float32, device="cuda") / D)
    t["k_pages"], t["v_pages"] = normal(pool), normal(pool)
    free = torch.randperm(P, device="cuda", generator=g).to(torch.int32)
    table = torch.full((len(kv), M), -1, dtype=torch.int32, device="cuda")   # entries past a sequence's end are unset
    at = 0
    for b, s in enumerate(kv):
        m = -(-s // ps)
        table[b, :m] = free[at:at + m]
        at += m
    start = [0]
    for k in n:
        start.append(start[-1] + k)
    t["block_table"] = table
    t["q_start"] = torch.tensor(start, dtype=torch.int32, device="cuda")
    t["kv_len"] = torch.tensor(kv, dtype=torch.int32, device="cuda")
    return t


def prepare(case, seed):
    state = {"case": case, "in": _inputs(case, seed)}
    if case["kind"] != "sample":
        n, kv = _lengths(case)
        # what the program that packs the batch knows of it
        state.update(rows=_rows(case, n), tokens=sum(n), most_new=max(n), most_kv=max(kv))
    if own:
        state.update(_program(case, state["in"]))
    return state


def _program(case, t):
    from hip_compiler import compile_subgraph, is_hip_op_supported
    from hip_runtime import HIPBackend
    from irgen.serving import build_paged_append_ir, build_paged_attention_ir, build_sample_ir
    from npu_compiler import partition
    from npu_runtime import DAGExecutor

    if case["kind"] == "sample":
        ir = build_sample_ir(case["rows"], case["vocab"], case["dtype"])
    else:
        n, kv = _lengths(case)
        build = build_paged_append_ir if case["kind"] == "append" else build_paged_attention_ir
        ir = build(tokens=_rows(case, n), seqs=case["seqs"], pages=_pages(case, kv), page_size=case["page"],
                   table_pages=_table_pages(case, kv), heads=case["heads"], kv_heads=case["kv_heads"],
                   head_dim=case["head_dim"], dtype=case["dtype"], layout=case["layout"])
    backend = HIPBackend(0)
    ex = DAGExecutor(partition(ir, is_hip_op_supported), backend, compile_fn=compile_subgraph)
    ex.load_weights({})
    return {"executor": ex, "buffers": {k: backend.allocate_buffer(v) for k, v in t.items()},
            "outputs": [o["name"] for o in ir["graph_outputs"]]}


def run(state):
    if own:
        out = state["executor"].execute(state["buffers"])
        return [out[name].to_torch() for name in state["outputs"]]
    kind = state["case"]["kind"]
    return [_plain_sample(state["in"])] if kind == "sample" else \
        _plain_append(state) if kind == "append" else [_plain_attention(state)]


# ---------------------------------------------------------------- plain forms

def _sequence_of(t, rows):
    """Sequence and position of each of the first ``rows`` rows."""
    r = torch.arange(rows, device="cuda")
    b = torch.searchsorted(t["q_start"][1:].contiguous(), r.to(torch.int32), right=True)
    return b, t["kv_len"][b].long() - t["q_start"][b + 1].long() + r


def _plain_append(state):
    t, case, N = state["in"], state["case"], state["tokens"]
    ps = case["page"]
    b, pos = _sequence_of(t, N)
    angle = pos[:, None].double() * t["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def rotate(x):
        a, c = x[:N].float().chunk(2, -1)
        return torch.cat([a * cos - c * sin, c * cos + a * sin], -1).to(x.dtype)

    q = torch.zeros_like(t["q"])
    q[:N] = rotate(t["q"])
    page, off = t["block_table"][b, pos // ps].long(), pos % ps
    for pool, new in ((t["k_pages"], rotate(t["k"])), (t["v_pages"], t["v"][:N])):
        if case["layout"] == "hnd":
            pool[page, :, off] = new
        else:
            pool[page, off] = new
    return [q, t["k_pages"], t["v_pages"]]


def _plain_attention(state):
    t, case = state["in"], state["case"]
    H, KVH, D, ps = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    n, S = state["most_new"], state["most_kv"]
    start, kv = t["q_start"].long(), t["kv_len"].long()
    B, G = kv.shape[0], H // KVH
    new = start[1:] - start[:-1]
    i = torch.arange(n, device="cuda")
    row = (start[:-1, None] + i).clamp(max=state["rows"] - 1)                 # [B, n]
    q = t["q"][row].float().reshape(B, n, KVH, G, D).permute(0, 2, 3, 1, 4).reshape(B, KVH, G * n, D)
    page = t["block_table"][:, :-(-S // ps)].clamp(min=0).long()

    def cache(pool):
        x = pool[page]
        x = x if case["layout"] == "nhd" else x.transpose(2, 3)               # [B, pages, page, KVH, D]
        return x.reshape(B, -1, KVH, D)[:, :S].transpose(1, 2).float()

    scores = torch.matmul(q, cache(t["k_pages"]).transpose(2, 3).contiguous()).reshape(B, KVH, G, n, S) * D ** -0.5
    pos = (kv - new)[:, None] + i
    closed = torch.arange(S, device="cuda") > pos[:, :, None]
    scores = scores.masked_fill_(closed[:, None, None], -math.inf)
    scores = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    weights = scores.div_(scores.sum(-1, keepdim=True)).reshape(B, KVH, G * n, S)
    o = torch.matmul(weights, cache(t["v_pages"]).contiguous()).reshape(B, KVH, G, n, D)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, n, H, D)
    out = torch.zeros_like(t["q"])
    b, pos = _sequence_of(t, state["tokens"])
    r = torch.arange(state["tokens"], device="cuda")
    out[:state["tokens"]] = o[b, r - start[b]].to(out.dtype)
    return out


def _plain_sample(t):
    x, T, u = t["logits"].double(), t["temperature"].double()[:, None], t["u"].double()[:, None]
    V = x.shape[1]
    s, order = torch.sort(x, dim=1, descending=True, stable=True)   # equal logits: the lowest index first
    w = ((s - s[:, :1]) / torch.where(T > 0, T, 1.0)).exp()
    rank, k, p = torch.arange(V, device="cuda"), t["top_k"][:, None], t["top_p"].double()[:, None]
    w = torch.where((k <= 0) | (rank < k), w, 0.0)
    total = w.cumsum(1)
    before = torch.cat([torch.zeros_like(total[:, :1]), total[:, :-1]], 1)
    kept = ((p >= 1) | (before < p * total[:, -1:])) & (w >= t["min_p"].double()[:, None])
    kept[:, 0] = True
    c = torch.zeros_like(w).scatter_(1, order, w * kept).cumsum(1)
    token = (c <= u * c[:, -1:]).sum(1).clamp(max=V - 1)
    return torch.where(T[:, 0] > 0, token, order[:, 0])


# ---------------------------------------------------------------- the same in 64 bits

def exact(case, seed):
    t = _inputs(case, seed)
    if case["kind"] == "sample":
        return [_exact_sample(t)]
    n, kv = _lengths(case)
    H, KVH, D, ps = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    out = torch.zeros((_rows(case, n), H, D), dtype=torch.float64, device="cuda")
    pools = [t[k] if case["layout"] == "nhd" else t[k].transpose(1, 2) for k in ("k_pages", "v_pages")]   # [P, page, KVH, D]
    if case["kind"] == "append":
        pools = [x.double() for x in pools]
    at = 0
    for b, (new, have) in enumerate(zip(n, kv)):
        if new == 0:
            continue
        q = t["q"][at:at + new].double()
        slot = torch.arange(have - new if case["kind"] == "append" else 0, have, device="cuda")
        page, off = t["block_table"][b].long()[slot // ps], slot % ps
        if case["kind"] == "append":
            z = torch.polar(torch.ones(new, D // 2, dtype=torch.float64, device="cuda"),
                            torch.outer(slot.double(), t["inv_freq"].double()))[:, None]

            def turn(x):
                y = torch.complex(x[..., :D // 2].contiguous(), x[..., D // 2:].contiguous()) * z
                return torch.cat([y.real, y.imag], -1)

            out[at:at + new] = turn(q)
            pools[0][page, off] = turn(t["k"][at:at + new].double())
            pools[1][page, off] = t["v"][at:at + new].double()
        else:
            open_ = slot <= torch.arange(have - new, have, device="cuda")[:, None]
            k, v = (x[page, off].double() for x in pools)
            for h in range(H):
                s = q[:, h] @ k[:, h // (H // KVH)].T / math.sqrt(D)
                out[at:at + new, h] = torch.softmax(s.masked_fill(~open_, -math.inf), 1) @ v[:, h // (H // KVH)]
        at += new
    if case["kind"] == "attention":
        return [out]
    return [out] + [x if case["layout"] == "nhd" else x.transpose(1, 2).contiguous() for x in pools]


def _exact_sample(t):
    a = {k: v.double().cpu().numpy() for k, v in t.items()}
    tokens = []
    for x, T, k, p, m, u in zip(*(a[key] for key in ("logits", "temperature", "top_k", "top_p", "min_p", "u"))):
        if T <= 0:
            tokens.append(int(np.argmax(x)))
            continue
        prob = np.exp((x - x.max()) / T)
        ranked = np.lexsort((np.arange(x.size), -x))
        if k > 0:
            ranked = ranked[:int(k)]
        mass = np.cumsum(prob[ranked])
        if p < 1:
            ranked = ranked[:1 + int(np.searchsorted(mass[:-1], p * mass[-1], side="left"))]
        ranked = np.sort(ranked[prob[ranked] >= m])
        mass = np.cumsum(prob[ranked])
        tokens.append(int(ranked[min(np.searchsorted(mass, u * mass[-1], side="right"), ranked.size - 1)]))
    return torch.tensor(tokens)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["kind"] == "sample":
        size = 4 if case["dtype"] == "float32" else 2
        return {"bytes": case["rows"] * (case["vocab"] * size + 28), "flops": 4 * case["rows"] * case["vocab"]}
    n, kv = _lengths(case)
    N, B = _rows(case, n), case["seqs"]
    H, KVH, D = case["heads"], case["kv_heads"], case["head_dim"]
    meta = 4 * (2 * B + 1 + sum(-(-s // case["page"]) for s in kv))
    if case["kind"] == "append":
        T = sum(n)
        return {"bytes": 2 * D * (T * (2 * H + 4 * KVH) + (N - T) * H) + meta, "flops": 3 * T * (H + KVH) * D}
    read = sum(s for k, s in zip(n, kv) if k)                               # idle slots are not read
    pairs = sum(k * s - k * (k - 1) // 2 for k, s in zip(n, kv))            # open (token, position) pairs
    return {"bytes": 2 * D * (2 * read * KVH + 2 * N * H) + meta, "flops": 4 * H * D * pairs}
