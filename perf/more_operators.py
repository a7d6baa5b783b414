"""What is timed when the operators of 8-bit caches and of normed heads are measured: one call of one operator, as cases.

They stand beside the paged append and attention of ``npu_runtime.serving_ops`` and take the same metadata: the new tokens of
all sequences are packed into rows, sequence ``b`` owning rows ``q_start[b] .. q_start[b + 1] - 1``; its cache holds
``kv_len[b]`` positions, the new ones the last of them, and position ``p`` lies in page ``block_table[b, p // page]``. Rows
from ``q_start[-1]`` on are padding.

kinds:

* ``append``     q and k rotated to their positions, k and v written into the pages. With ``norm`` each head of q and k is
                 first divided by its root mean square and multiplied by a weight. With ``cache`` 8 the pages hold e4m3 bytes
                 beside one power of two per position and K/V head (``k_scales``, ``v_scales``, its exponent + 127): the
                 smallest one, 2^-100 at least, with which the head's largest magnitude is at most 448.
* ``attention``  causal attention of the new tokens over such pages of 8 bits.

8-bit outputs are returned as tensors of the 8-bit floating types that their bytes are.
"""

from __future__ import annotations

import math
import os
import random
import sys

import torch

_PKG = os.path.join(os.getcwd(), "pytorch-apple_amd")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

own = False

THETA, EPS = 1e6, 1e-6
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16}
_BASE = {"seqs": 1, "decodes": 0, "idle": 0, "new": 1, "context": 0, "pad": 0, "lengths": 0, "heads": 12, "kv_heads": 2,
         "head_dim": 128, "page": 16, "layout": "hnd", "dtype": "bfloat16", "norm": False, "cache": 8}


def _case(name, kind, **kw):
    return {"name": name, "kind": kind, **_BASE, **kw}


def listed():
    return [
        # one request, one token of a model that norms its heads: what a single user's chat pays a layer for the cache update
        _case("norm_append_one_token", "append", seqs=1, decodes=1, context=2047, norm=True, cache=16),
        # a server's step of such a model: most slots decode, two prompts come in, two slots idle, spare rows
        _case("norm_append_mixed", "append", seqs=48, decodes=44, idle=2, new=700, context=4000, pad=37, heads=14, head_dim=64,
              page=32, dtype="float16", lengths=1, norm=True, cache=16),
        # one token into 8-bit pages
        _case("quant_append_one_token", "append", seqs=1, decodes=1, context=2047),
        # a server's step into 8-bit pages that are kept token by token
        _case("quant_append_mixed", "append", seqs=48, decodes=44, idle=2, new=700, context=4000, pad=37, heads=14, head_dim=64,
              page=32, layout="nhd", dtype="float16", lengths=1),
        # a batch of whole prompts, normed and quantised
        _case("norm_quant_append_prompts", "append", seqs=6, new=1500, heads=32, kv_heads=8, page=64, lengths=2, norm=True),
        # one request, one token over a short cache: latency
        _case("quant_attention_one_token", "attention", seqs=1, decodes=1, context=2047),
        # a full decode batch over ragged caches of a few thousand positions
        _case("quant_attention_decode_64", "attention", seqs=64, decodes=64, context=4096, heads=32, kv_heads=8,
              dtype="float16", lengths=3),
        # few requests with very long documents
        _case("quant_attention_decode_long", "attention", seqs=4, decodes=4, context=131071, page=64, lengths=4),
        # the next chunk of a long prompt, the pages kept token by token
        _case("quant_attention_chunk_long", "attention", seqs=1, new=500, context=30000, layout="nhd", page=32, lengths=5),
        # a batch of whole prompts
        _case("quant_attention_prompts", "attention", seqs=6, new=1500, heads=32, kv_heads=8, page=64, lengths=2),
        # a server's step: decoding slots beside a prompt chunk, idle slots and spare rows
        _case("quant_attention_mixed", "attention", seqs=64, decodes=60, idle=3, new=448, context=4000, pad=21, heads=14,
              head_dim=64, page=32, dtype="float16", lengths=6),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "append", "attention", "attention"])
    norm, cache = rng.choice([(True, 16), (False, 8), (True, 8)]) if kind == "append" else (False, 8)
    heads, kv_heads, dim = rng.choice([(12, 2, 128), (14, 2, 64), (32, 8, 128), (8, 8, 64), (16, 1, 128), (40, 8, 128)])
    seqs = _log(rng, 1, 64)
    decodes = rng.choice([seqs, seqs, rng.randint(0, seqs), max(0, seqs - 1)])
    while True:
        new = _log(rng, 2, 2000) if decodes < seqs else 1
        context = rng.choice([0, _log(rng, 16, 32000)]) if decodes < seqs else _log(rng, 16, 120000)
        c = _case("", kind, seqs=seqs, decodes=decodes, idle=rng.choice([0, rng.randint(0, (seqs - 1) // 4)]), new=new,
                  context=context, pad=rng.choice([0, rng.randint(0, 40)]), lengths=rng.randint(0, 1 << 30), heads=heads,
                  kv_heads=kv_heads, head_dim=dim, page=rng.choice([16, 32, 48, 64, 128]),
                  layout=rng.choice(["hnd", "hnd", "nhd"]), dtype=rng.choice(["bfloat16", "float16"]), norm=norm, cache=cache)
        n, kv = _lengths(c)
        scores = seqs * heads * max(n) * (max(kv) + 1)
        w = work(c)
        if max(n) > 0 and sum(n) <= 6000 and scores <= 1 << 29 and w["bytes"] <= 4 << 26 and w["flops"] <= 9e10 and \
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

def _inputs(case, seed):
    g, dt = torch.Generator(device="cuda").manual_seed(seed), DTYPES[case["dtype"]]

    def normal(shape, std=1.0, mean=0.0, dtype=dt):
        return torch.empty(shape, dtype=dtype, device="cuda").normal_(mean, std, generator=g)

    n, kv = _lengths(case)
    N, P, M = _rows(case, n), _pages(case, kv), _table_pages(case, kv)
    H, KVH, D, ps = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    pool = (P, KVH, ps, D) if case["layout"] == "hnd" else (P, ps, KVH, D)
    t = {"q": normal((N, H, D), 1.5 if case["kind"] == "attention" else 1.0)}
    if case["kind"] == "append":
        t["k"], t["v"] = normal((N, KVH, D), 2.0), normal((N, KVH, D), 0.5)
        t["inv_freq"] = 1.0 / THETA ** (torch.arange(0, D, 2, dtype=torch.float32, device="cuda") / D)
    if case["norm"]:
        t["q_weight"], t["k_weight"] = normal((D,), 0.2, 1.0), normal((D,), 0.2, 1.0)
    if case["cache"] == 8:
        # heads of standard deviation 2^-1 .. 2: their largest magnitudes, some 3 of them, come to 224 .. 448 in 8 bits
        for which in ("k", "v"):
            t[which + "_pages"] = normal(pool, 110.0, dtype=torch.float16).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
            t[which + "_scales"] = torch.randint(119, 122, (P, KVH, ps), device="cuda", generator=g).to(torch.uint8)
    else:
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
    n, kv = _lengths(case)
    # what the program that packs the batch knows of it
    state = {"case": case, "in": _inputs(case, seed), "rows": _rows(case, n), "tokens": sum(n), "most_new": max(n),
             "most_kv": max(kv)}
    if own:
        state.update(_program(case, state["in"]))
    return state


def _program(case, t):
    from hip_compiler import compile_subgraph, is_hip_op_supported
    from hip_runtime import HIPBackend
    from irgen.serving import build_paged_append_ir, build_paged_attention_ir
    from npu_compiler import partition
    from npu_runtime import DAGExecutor

    n, kv = _lengths(case)
    sizes = dict(tokens=_rows(case, n), seqs=case["seqs"], pages=_pages(case, kv), page_size=case["page"],
                 table_pages=_table_pages(case, kv), heads=case["heads"], kv_heads=case["kv_heads"],
                 head_dim=case["head_dim"], dtype=case["dtype"], layout=case["layout"],
                 cache="float8_e4m3fn" if case["cache"] == 8 else None)
    ir = build_paged_append_ir(**sizes, norm_eps=EPS if case["norm"] else None) if case["kind"] == "append" else \
        build_paged_attention_ir(**sizes)
    backend = HIPBackend(0)
    ex = DAGExecutor(partition(ir, is_hip_op_supported), backend, compile_fn=compile_subgraph)
    ex.load_weights({})
    return {"executor": ex, "buffers": {k: backend.allocate_buffer(v) for k, v in t.items()},
            "outputs": [o["name"] for o in ir["graph_outputs"]]}


def _as_floats(out):
    """[q, k pages, v pages, k scales, v scales]: bytes as the floating types that they are."""
    return out[:1] + [x.view(torch.float8_e4m3fn) for x in out[1:3]] + [x.view(torch.float8_e8m0fnu) for x in out[3:]]


def run(state):
    case = state["case"]
    if own:
        out = state["executor"].execute(state["buffers"])
        out = [out[name].to_torch() for name in state["outputs"]]
    else:
        out = _plain_append(state) if case["kind"] == "append" else [_plain_attention(state)]
    return _as_floats(out) if len(out) == 5 else out


# ---------------------------------------------------------------- plain forms

def _sequence_of(t, rows):
    """Sequence and position of each of the first ``rows`` rows."""
    r = torch.arange(rows, device="cuda")
    b = torch.searchsorted(t["q_start"][1:].contiguous(), r.to(torch.int32), right=True)
    return b, t["kv_len"][b].long() - t["q_start"][b + 1].long() + r


def _plain_quantise(x):
    """(e4m3 bytes, exponent bytes) of float32 heads."""
    m, x2 = torch.frexp(x.abs().amax(-1).clamp(min=2.0 ** -92))
    e = x2 - 9 + (m > 0.875)             # the largest magnitude is m 2^x2, and 448 is 0.875 2^9
    y = torch.ldexp(x, -e[..., None]).to(torch.float8_e4m3fn)
    return y.view(torch.uint8), (e + 127).to(torch.uint8)


def _plain_append(state):
    t, case, N = state["in"], state["case"], state["tokens"]
    ps = case["page"]
    b, pos = _sequence_of(t, N)
    angle = pos[:, None].double() * t["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def rotated(x, weight):
        x = x[:N].float()
        if case["norm"]:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * t[weight].float()
        a, c = x.chunk(2, -1)
        return torch.cat([a * cos - c * sin, c * cos + a * sin], -1)

    q = torch.zeros_like(t["q"])
    q[:N] = rotated(t["q"], "q_weight").to(q.dtype)
    page, off = t["block_table"][b, pos // ps].long(), pos % ps
    out = [q, t["k_pages"], t["v_pages"]]
    new = [rotated(t["k"], "k_weight"), t["v"][:N].float()]
    if case["cache"] == 8:
        out += [t["k_scales"], t["v_scales"]]
        (new[0], ke), (new[1], ve) = _plain_quantise(new[0]), _plain_quantise(new[1])
        t["k_scales"][page, :, off] = ke
        t["v_scales"][page, :, off] = ve
    for pool, x in zip(out[1:3], new):
        if case["layout"] == "hnd":
            pool[page, :, off] = x.to(pool.dtype)
        else:
            pool[page, off] = x.to(pool.dtype)
    return out


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

    def cache(pool, scales):
        x = pool.view(torch.float8_e4m3fn)[page].float()
        x = x.transpose(2, 3) if case["layout"] == "nhd" else x               # [B, pages, KVH, page, D]
        x = torch.ldexp(x, scales[page].int()[..., None] - 127)
        return x.transpose(2, 3).reshape(B, -1, KVH, D)[:, :S].transpose(1, 2)

    keys = cache(t["k_pages"], t["k_scales"]).transpose(2, 3).contiguous()
    scores = torch.matmul(q, keys).reshape(B, KVH, G, n, S) * D ** -0.5
    pos = (kv - new)[:, None] + i
    closed = torch.arange(S, device="cuda") > pos[:, :, None]
    scores = scores.masked_fill_(closed[:, None, None], -math.inf)
    scores = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    weights = scores.div_(scores.sum(-1, keepdim=True)).reshape(B, KVH, G * n, S)
    o = torch.matmul(weights, cache(t["v_pages"], t["v_scales"]).contiguous()).reshape(B, KVH, G, n, D)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, n, H, D)
    out = torch.zeros_like(t["q"])
    b, pos = _sequence_of(t, state["tokens"])
    r = torch.arange(state["tokens"], device="cuda")
    out[:state["tokens"]] = o[b, r - start[b]].to(out.dtype)
    return out


# ---------------------------------------------------------------- the same in 64 bits

def exact(case, seed):
    t = _inputs(case, seed)
    n, kv = _lengths(case)
    H, D, ps = case["heads"], case["head_dim"], case["page"]
    eight = case["cache"] == 8
    out = torch.zeros((_rows(case, n), H, D), dtype=torch.float64, device="cuda")
    pools = [t[k].view(torch.float8_e4m3fn).float() if eight else t[k] for k in ("k_pages", "v_pages")]
    pools = [x if case["layout"] == "nhd" else x.transpose(1, 2) for x in pools]   # [P, page, KVH, D]
    scales = [2.0 ** (t[k].double() - 127).transpose(1, 2) for k in ("k_scales", "v_scales")] if eight else []
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

            def turn(x, weight):
                if case["norm"]:
                    x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS) * t[weight].double()
                y = torch.complex(x[..., :D // 2].contiguous(), x[..., D // 2:].contiguous()) * z
                return torch.cat([y.real, y.imag], -1)

            out[at:at + new] = turn(q, "q_weight")
            heads = [turn(t["k"][at:at + new].double(), "k_weight"), t["v"][at:at + new].double()]
            for i, x in enumerate(heads):
                if eight:
                    s = 2.0 ** torch.ceil(torch.log2(x.abs().amax(-1) / 448)).clamp(min=-100)
                    scales[i][page, off], x = s, x / s[..., None]
                pools[i][page, off] = x
        else:
            open_ = slot <= torch.arange(have - new, have, device="cuda")[:, None]
            k, v = (x[page, off].double() * s[page, off][..., None] for x, s in zip(pools, scales))
            for h in range(H):
                g = h // (H // case["kv_heads"])
                w = torch.softmax((q[:, h] @ k[:, g].T / math.sqrt(D)).masked_fill(~open_, -math.inf), 1)
                out[at:at + new, h] = w @ v[:, g]
        at += new
    if case["kind"] == "attention":
        return [out]
    return [out] + [x if case["layout"] == "nhd" else x.transpose(1, 2).contiguous() for x in pools] + \
        [s.transpose(1, 2).contiguous() for s in scales]


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    n, kv = _lengths(case)
    N, B = _rows(case, n), case["seqs"]
    H, KVH, D = case["heads"], case["kv_heads"], case["head_dim"]
    place = D + 1 if case["cache"] == 8 else 2 * D                          # bytes of a cached head
    meta = 4 * (2 * B + 1 + sum(-(-s // case["page"]) for s in kv))
    if case["kind"] == "append":
        T = sum(n)
        per = 3 + (4 if case["norm"] else 0) + (2 if case["cache"] == 8 else 0)
        return {"bytes": T * (4 * D * H + 2 * KVH * (2 * D + place)) + 2 * D * (N - T) * H + meta, "flops": per * T * (H + 2 * KVH) * D}
    read = sum(s for k, s in zip(n, kv) if k)                               # idle slots are not read
    pairs = sum(k * s - k * (k - 1) // 2 for k, s in zip(n, kv))            # open (token, position) pairs
    return {"bytes": 2 * read * KVH * place + 4 * D * N * H + meta, "flops": 4 * H * D * pairs}
