"""Lowering of the serving operators (``npu_runtime.serving_ops``) to the kernels of csrc/kernels/paged.hip and
sample.hip. No counterpart in the reference.
"""

from __future__ import annotations

from hip_compiler.program import DTYPE_CODE, ELEM_SIZE, LaunchStep, TView
from npu_compiler.ir_reader import OpNode
from npu_runtime.serving_ops import check_paged_append, check_paged_attention, check_sample

PAGED_ANY_MAX_D = 256          # paged.hip PG_ANY_D
PAGED_APPEND_MAX_R = 256       # paged.hip PG_APPEND_R
# Up to this many rows a workgroup per row, past it a wave. us by workgroups / by waves, in 16 bits: 16 rows of 12 + 2 heads
# of 128 3.8 / 5.1, 1,024 5.1 / 5.7, 2,048 7.5 / 6.8, 8,192 21.9 / 14.8; 14 + 2 of 64: 3.9 / 3.9, 4.6 / 4.3, 6.5 / 5.0,
# 18.8 / 10.2; 32 + 8 of 128, whose rows keep four waves busy: 4.1 / 7.2, 6.7 / 8.7, 10.5 / 12.9, 32.4 / 34.4.
PAGED_APPEND_ROW_N = 1024
# paged.hip: sequences of a list, rows of a tile, fewest blocks of a narrow workgroup and of a wide tile's split, items
# that wide tiles are split towards
PT_MAXB, PT_NARROW, PT_WIDE, PT_NARROW_LEAST, PT_WIDE_LEAST, PT_WIDE_ITEMS = 1024, 32, 128, 4, 8, 480
PT_GRID = 512                  # two workgroups per CU
# sample.hip: SM_GROUPS groups of 64 pieces of 16 bytes, bins, tokens of a list
SAMPLE_MAX_PIECES, SAMPLE_BINS, SAMPLE_LIST = 4096 * 64, 512, 16384
# Up to this many pieces k_sample_pick alone, past it the four launches. us alone / four, top-k 50 and top-p 0.95, bfloat16:
# 500 pieces 30.7 / 30.4 for one row and 32.7 / 34.0 for 256, 1,000 35.3 / 29.8 and 36.8 / 36.2, 2,000 44.1 / 30.6 and
# 47.3 / 39.9; float32: 500 27.3 / 28.7 and 28.7 / 32.3, 1,000 30.7 / 28.4 and 31.6 / 34.5, 2,000 36.8 / 29.2 and 38.3 / 36.6.
SAMPLE_PICK_PIECES = 1024


def _rows_view(low, name: str) -> TView:
    """The [rows, heads, dims] view ``name`` with contiguous dims (rows and heads may be strided)."""
    v = low.view(name)
    return v if v.shape[2] <= 1 or v.strides[2] == 1 else low.contiguous(name, v)


def _pool_strides(shape, layout: str) -> dict:
    _, d1, d2, D = (int(s) for s in shape)
    head, row = (d2 * D, D) if layout == "hnd" else (D, d2 * D)
    return dict(page_stride=d1 * d2 * D, head_stride=head, row_stride=row)


def _pool_dims(shape, layout: str) -> tuple[int, int]:
    """(K/V heads, page size)"""
    return (int(shape[1]), int(shape[2])) if layout == "hnd" else (int(shape[2]), int(shape[1]))


def _check_i32(op: str, **sizes) -> None:
    for name, n in sizes.items():
        if n >= 2 ** 31:
            raise NotImplementedError(f"{op}: {name} = {n} does not fit 32 bits")


def _aligned_rows(low, name: str, v: TView) -> TView:
    """``v`` when its rows and heads start on 16-byte boundaries, else a contiguous copy of it."""
    per = 16 // ELEM_SIZE[v.dtype]
    if v.offset % per == 0 and all(s % per == 0 for n, s in zip(v.shape[:2], v.strides[:2]) if n > 1):
        return v
    out = low.new_storage(name + ".rows", v.shape, v.dtype)
    low.emit_copy(v, out, [name], [name + ".rows"])
    return out


def paged_tiles(N: int, B: int, M: int, P: int, H: int, KVH: int, D: int, page_size: int, dtype: str) -> dict | None:
    """Launch of the tiled attention kernels (paged.hip), None where they do not apply: other types or head sizes,
    pages that are no multiple of 16 positions, more sequences than the item list holds, or sizes whose item
    counts could pass 32 bits. Wide tiles are left out where the rows average at most two tokens per sequence: a
    decode step's batches then need no workgroups that look for chunks, and a longer chunk in one takes several
    narrow tiles. us with wide tiles / without, 32 heads over 8 of 128: 64 sequences over up to 4,000 positions, all but
    one of them decoding, the chunk of 1 token 160 / 156, of 64 168 / 160, of 200 187 / 177, of 400 203 / 205; six prompts
    of 1,000 111 / 299, 16 of 100 26 / 54; one chunk over 30,000 positions, of 16 tokens 39 / 35, of 64 59 / 61, of 256
    146 / 188. So between two and some six tokens per sequence the rule costs up to 6% (with 12 over 2 heads, whose caches
    are read in a third of the time, up to 29%: 46 / 35 at 2.5): a launch does not know whether its rows are one chunk or many."""
    if dtype not in ("bfloat16", "float16") or D not in (64, 128) or page_size % 16 or not 0 < B <= PT_MAXB or M < 1 or P < 1:
        return None
    G, block = H // KVH, 8192 // (2 * D)
    blocks = -(-M * page_size // block)
    tiles = lambda R: KVH * (N * G // R + min(N, B))
    if (tiles(PT_NARROW) + 2 * PT_GRID) * (2 * blocks + 3) >= 2 ** 31 or M * page_size * page_size >= 2 ** 40 \
            or KVH * page_size * D >= 2 ** 30:
        return None
    wide = N > 2 * B and N * G > PT_NARROW
    # a split tile has ceil(blocks / share) < 2 blocks / share parts, all together under twice the items aimed at;
    # nor can a tile have more than its blocks allow
    slots = min(2 * PT_WIDE_ITEMS, tiles(PT_WIDE) * -(-blocks // PT_WIDE_LEAST))
    return {"grid_wide": min(PT_GRID, 8 * -(-(tiles(PT_WIDE) + PT_WIDE_ITEMS) // 8)) if wide else 0,
            "grid_narrow": min(PT_GRID, -(-tiles(PT_NARROW) * blocks // PT_NARROW_LEAST)),
            "wide_slots": slots if wide else 0}


def _batch(low, table, q_start, kv_len) -> dict:
    return dict(table=low.ref(low.contiguous(table.name)), q_start=low.ref(low.contiguous(q_start.name)),
                kv_len=low.ref(low.contiguous(kv_len.name)), B=int(kv_len.shape[0]), M=int(table.shape[1]))


def lower_paged_append(low, node: OpNode) -> None:
    q, k, v, kp, vp, table, q_start, kv_len, inv = node.inputs
    layout = node.attrs.get("page_layout", "hnd")
    check_paged_append(q, k, v, kp, vp, table, q_start, kv_len, inv, layout)
    N, H, D = (int(s) for s in q.shape)
    KVH, ps = _pool_dims(kp.shape, layout)
    _check_i32(node.op_type, rows=N * H * D, table=int(table.shape[0]) * int(table.shape[1]), page=KVH * ps * D)
    qv, kv, vv = (_rows_view(low, t.name) for t in (q, k, v))
    q_out = low.new_storage(node.outputs[0].name, q.shape, q.dtype)
    low.views[node.outputs[0].name] = q_out
    pools = [low.inplace_or_copy(node, t, o) for t, o in ((kp, node.outputs[1]), (vp, node.outputs[2]))]
    if N == 0:
        return
    kernel, grid = "k_paged_append_any", N
    R = 2 * int(inv.shape[0])
    if q.dtype in ("bfloat16", "float16") and D % 8 == 0 and R % 16 == 0 and R <= PAGED_APPEND_MAX_R:
        qv, kv, vv = (_aligned_rows(low, t.name, v) for t, v in ((q, qv), (k, kv), (v, vv)))
        few = N <= PAGED_APPEND_ROW_N
        kernel = f"k_paged_append_{'bf16' if q.dtype == 'bfloat16' else 'f16'}" + ("_row" if few else "")
        grid = N if few else -(-N // 4)
    low.emit(LaunchStep(
        kind="paged_append", kernel=kernel, module="paged", arg_struct="PagedAppendArgs",
        args=dict(q=low.ref(qv), k=low.ref(kv), v=low.ref(vv), k_pages=low.ref(pools[0]), v_pages=low.ref(pools[1]),
                  q_out=low.ref(q_out), **_batch(low, table, q_start, kv_len),
                  inv_freq=low.ref(low.contiguous(inv.name)), q_rs=qv.strides[0], q_hs=qv.strides[1], k_rs=kv.strides[0],
                  k_hs=kv.strides[1], v_rs=vv.strides[0], v_hs=vv.strides[1], **_pool_strides(kp.shape, layout),
                  pages=int(kp.shape[0]), N=N, H=H, KVH=KVH, D=D, R=R, page_size=ps,
                  scaling=float(node.attrs.get("attention_scaling", 1.0)), dtype=DTYPE_CODE[q.dtype]),
        grid=(grid, 1, 1), inputs=[t.name for t in node.inputs], outputs=[o.name for o in node.outputs],
        params={"rows": N, "seqs": int(kv_len.shape[0]), "heads": H, "kv_heads": KVH, "head_dim": D,
                "pieces16": [] if kernel == "k_paged_append_any" else ["q", "k", "v", "k_pages", "v_pages"]}))


def lower_paged_attention(low, node: OpNode) -> None:
    q, kp, vp, table, q_start, kv_len = node.inputs
    layout = node.attrs.get("page_layout", "hnd")
    check_paged_attention(q, kp, vp, table, q_start, kv_len, layout)
    N, H, D = (int(s) for s in q.shape)
    KVH, ps = _pool_dims(kp.shape, layout)
    # (the plain kernel steps by 64 positions up to a table's last)
    _check_i32(node.op_type, rows=N * H * D, table=int(table.shape[0]) * int(table.shape[1]), page=KVH * ps * D,
               **{"positions of a table": int(table.shape[1]) * ps + 63})
    if D > PAGED_ANY_MAX_D:
        raise NotImplementedError(f"{node.op_type}: head_dim {D} is over {PAGED_ANY_MAX_D}")
    qv = _rows_view(low, q.name)
    kv, vv = (low.contiguous(t.name) for t in (kp, vp))
    out = low.new_storage(node.outputs[0].name, q.shape, q.dtype)
    low.views[node.outputs[0].name] = out
    if N == 0:
        return
    B, M, P = int(kv_len.shape[0]), int(table.shape[1]), int(kp.shape[0])
    tiled = paged_tiles(N, B, M, P, H, KVH, D, ps, q.dtype)
    if tiled:
        qv = _aligned_rows(low, q.name, qv)
        kv, vv = (low.aligned16(v, t.name) for t, v in ((kp, kv), (vp, vv)))
    args = dict(q=low.ref(qv), k_pages=low.ref(kv), v_pages=low.ref(vv), out=low.ref(out), part_o=None, part_ml=None,
                **_batch(low, table, q_start, kv_len), q_rs=qv.strides[0], q_hs=qv.strides[1],
                **_pool_strides(kp.shape, layout), pages=P, N=N, H=H, KVH=KVH, D=D, page_size=ps,
                scale=float(node.attrs["scale"]), dtype=DTYPE_CODE[q.dtype], page_groups=0, group_magic=0, grid_wide=0,
                grid_narrow=0, pad=0)
    params = {"rows": N, "seqs": B, "heads": H, "kv_heads": KVH, "head_dim": D}
    ins, outs = [t.name for t in node.inputs], [node.outputs[0].name]
    if tiled is None:
        low.emit(LaunchStep(kind="paged_attention", kernel="k_paged_attn_any", module="paged", arg_struct="PagedAttnArgs",
                            args=args, grid=(N, H, 1), block=(64, 1, 1), inputs=ins, outputs=outs, params=params))
        return
    params["pieces16"] = ["q", "k_pages", "v_pages"]
    groups = ps // 16
    part_rows = 2 * tiled["grid_narrow"] * PT_NARROW + tiled["wide_slots"] * PT_WIDE
    args.update(part_o=low.scratch(outs[0] + ".part_o", 4 * part_rows * D),
                part_ml=low.scratch(outs[0] + ".part_ml", 8 * part_rows), page_groups=groups,
                group_magic=0 if groups == 1 else -(-2 ** 32 // groups), grid_wide=tiled["grid_wide"],
                grid_narrow=tiled["grid_narrow"])
    name = f"{'bf16' if q.dtype == 'bfloat16' else 'f16'}_d{D}"
    low.emit(LaunchStep(
        kind="paged_attention", kernel="k_paged_attn_" + name, module="paged", arg_struct="PagedAttnArgs", args=dict(args),
        grid=(tiled["grid_wide"] + tiled["grid_narrow"], 1, 1), inputs=ins, outputs=outs, params={**params, "mfma": True}))
    low.emit(LaunchStep(
        kind="paged_attention", kernel="k_paged_combine_" + name, module="paged", arg_struct="PagedAttnArgs",
        args=dict(args), grid=(min(1024, -(-N * H // 4)), 1, 1), inputs=ins, outputs=outs, params=params))


def lower_sample(low, node: OpNode) -> None:
    x, temperature, top_k, top_p, min_p, u = node.inputs
    check_sample(x, temperature, top_k, top_p, min_p, u)
    B, V = (int(s) for s in x.shape)
    if V > (SAMPLE_MAX_PIECES - 1) * (16 // ELEM_SIZE[x.dtype]) or B > 65535:
        raise NotImplementedError(f"{node.op_type}: {B} rows of {V}: over 65,535 rows, or over the kernel's {SAMPLE_MAX_PIECES} "
                                  f"pieces of the vocabulary")
    xv = low.aligned16(low.contiguous(x.name), x.name)
    out = low.new_storage(node.outputs[0].name, [B], "int64")
    low.views[node.outputs[0].name] = out
    if B == 0:
        return
    width = 16 // ELEM_SIZE[x.dtype]
    pieces = (V + width - 2) // width + 1   # most that a row, wherever it starts, can touch
    # Pieces a thread: few, so that few rows take many workgroups, but not over 32 parts, whose bins one workgroup adds
    # up. The first three launches for one row of 151,936 in bf16: 10 + 9 + 17 us in 10 parts of 8, 6 + 9 + 10 in 19 of
    # 4, 5 + 11 + 7 in 38 of 2 (but call after call 45 us rather than 43), 5 + 14 + 6 in 75 of 1. 256 rows of float32:
    # 39 + 10 + 57 by 8, 41 + 17 + 63 by 2.
    def parts_of(per):
        return -(-pieces // (256 * per))
    per = next((p for p in (1, 2, 4) if parts_of(p) <= 32 and B * parts_of(p) <= 1024), 8)
    parts, groups = parts_of(per), -(-pieces // 64)
    binned = pieces > SAMPLE_PICK_PIECES
    name = node.outputs[0].name
    ws = (lambda what, nbytes: low.scratch(f"{name}.{what}", nbytes)) if binned else (lambda what, nbytes: None)
    args = dict(logits=low.ref(xv), temperature=low.ref(low.contiguous(temperature.name)),
                top_k=low.ref(low.contiguous(top_k.name)), top_p=low.ref(low.contiguous(top_p.name)),
                min_p=low.ref(low.contiguous(min_p.name)), u=low.ref(low.contiguous(u.name)), out=low.ref(out),
                best=ws("best", 8 * B * parts), bins=ws("bins", 8 * B * parts * SAMPLE_BINS), row=ws("row", 40 * B),
                groups=ws("groups", 8 * B * groups), sums=ws("sums", 16 * B),
                listed=ws("listed", 4 * B), list=ws("list", 8 * B * SAMPLE_LIST), rows=B, vocab=V,
                dtype=DTYPE_CODE[x.dtype], shift=min(44, 62 - V.bit_length()), parts=parts, ngroups=groups, per=per)
    dt = {"float32": "f32", "float16": "f16", "bfloat16": "bf16"}[x.dtype]
    launches = [("k_sample_pick_" + dt, (B, 1, 1), 1024)]
    if binned:
        launches = [("k_sample_hist_" + dt, (parts, B, 1), 256), ("k_sample_merge", (B, 1, 1), 1024),
                    ("k_sample_collect_" + dt, (parts, B, 1), 256)] + launches
    for kernel, grid, threads in launches:
        low.emit(LaunchStep(kind="sample", kernel=kernel, module="sample", arg_struct="SampleArgs", args=dict(args),
                            grid=grid, block=(threads, 1, 1), inputs=[t.name for t in node.inputs], outputs=[name],
                            params={"rows": B, "vocab": V}))


LOWERINGS = {"serving.paged_append.default": lower_paged_append,
             "serving.paged_attention.default": lower_paged_attention, "serving.sample.default": lower_sample}
