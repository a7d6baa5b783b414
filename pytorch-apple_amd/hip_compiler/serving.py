"""Lowering of the serving operators (``npu_runtime.serving_ops``) to the kernels of csrc/kernels/paged.hip and
sample.hip. No counterpart in the reference.
"""

from __future__ import annotations

from hip_compiler.program import DTYPE_CODE, ELEM_SIZE, LaunchStep, TView
from npu_compiler.ir_reader import OpNode
from npu_runtime.serving_ops import check_paged_append, check_paged_attention, check_sample

PAGED_ANY_MAX_D = 256          # paged.hip PG_ANY_D
SAMPLE_MAX_PIECES = 4096 * 64  # sample.hip SM_GROUPS groups of 64 pieces of 16 bytes


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
    pools = [low.inplace_or_copy(t, o) for t, o in ((kp, node.outputs[1]), (vp, node.outputs[2]))]
    if N == 0:
        return
    low.emit(LaunchStep(
        kind="paged_append", kernel="k_paged_append_any", module="paged", arg_struct="PagedAppendArgs",
        args=dict(q=low.ref(qv), k=low.ref(kv), v=low.ref(vv), k_pages=low.ref(pools[0]), v_pages=low.ref(pools[1]),
                  q_out=low.ref(q_out), **_batch(low, table, q_start, kv_len),
                  inv_freq=low.ref(low.contiguous(inv.name)), q_rs=qv.strides[0], q_hs=qv.strides[1], k_rs=kv.strides[0],
                  k_hs=kv.strides[1], v_rs=vv.strides[0], v_hs=vv.strides[1], **_pool_strides(kp.shape, layout),
                  pages=int(kp.shape[0]), N=N, H=H, KVH=KVH, D=D, R=2 * int(inv.shape[0]), page_size=ps,
                  scaling=float(node.attrs.get("attention_scaling", 1.0)), dtype=DTYPE_CODE[q.dtype]),
        grid=(N, 1, 1), inputs=[t.name for t in node.inputs], outputs=[o.name for o in node.outputs],
        params={"rows": N, "seqs": int(kv_len.shape[0]), "heads": H, "kv_heads": KVH, "head_dim": D}))


def lower_paged_attention(low, node: OpNode) -> None:
    q, kp, vp, table, q_start, kv_len = node.inputs
    layout = node.attrs.get("page_layout", "hnd")
    check_paged_attention(q, kp, vp, table, q_start, kv_len, layout)
    N, H, D = (int(s) for s in q.shape)
    KVH, ps = _pool_dims(kp.shape, layout)
    _check_i32(node.op_type, rows=N * H * D, table=int(table.shape[0]) * int(table.shape[1]), page=KVH * ps * D)
    if D > PAGED_ANY_MAX_D:
        raise NotImplementedError(f"{node.op_type}: head_dim {D} is over {PAGED_ANY_MAX_D}")
    qv = _rows_view(low, q.name)
    kv, vv = (low.contiguous(t.name) for t in (kp, vp))
    out = low.new_storage(node.outputs[0].name, q.shape, q.dtype)
    low.views[node.outputs[0].name] = out
    if N == 0:
        return
    low.emit(LaunchStep(
        kind="paged_attention", kernel="k_paged_attn_any", module="paged", arg_struct="PagedAttnArgs",
        args=dict(q=low.ref(qv), k_pages=low.ref(kv), v_pages=low.ref(vv), out=low.ref(out),
                  **_batch(low, table, q_start, kv_len), q_rs=qv.strides[0], q_hs=qv.strides[1],
                  **_pool_strides(kp.shape, layout), pages=int(kp.shape[0]), N=N, H=H, KVH=KVH, D=D, page_size=ps,
                  scale=float(node.attrs["scale"]), dtype=DTYPE_CODE[q.dtype], pad=0),
        grid=(N, H, 1), block=(64, 1, 1), inputs=[t.name for t in node.inputs], outputs=[node.outputs[0].name],
        params={"rows": N, "seqs": int(kv_len.shape[0]), "heads": H, "kv_heads": KVH, "head_dim": D}))


def lower_sample(low, node: OpNode) -> None:
    x, temperature, top_k, top_p, min_p, u = node.inputs
    check_sample(x, temperature, top_k, top_p, min_p, u)
    B, V = (int(s) for s in x.shape)
    if V > (SAMPLE_MAX_PIECES - 1) * (16 // ELEM_SIZE[x.dtype]):
        raise NotImplementedError(f"{node.op_type}: a vocabulary of {V} is over the kernel's {SAMPLE_MAX_PIECES} pieces")
    xv = low.aligned16(low.contiguous(x.name), x.name)
    out = low.new_storage(node.outputs[0].name, [B], "int64")
    low.views[node.outputs[0].name] = out
    if B == 0:
        return
    low.emit(LaunchStep(
        kind="sample", kernel={"float32": "k_sample_f32", "float16": "k_sample_f16",
                               "bfloat16": "k_sample_bf16"}[x.dtype], module="sample", arg_struct="SampleArgs",
        args=dict(logits=low.ref(xv), temperature=low.ref(low.contiguous(temperature.name)),
                  top_k=low.ref(low.contiguous(top_k.name)), top_p=low.ref(low.contiguous(top_p.name)),
                  min_p=low.ref(low.contiguous(min_p.name)), u=low.ref(low.contiguous(u.name)), out=low.ref(out), rows=B,
                  vocab=V, dtype=DTYPE_CODE[x.dtype], shift=min(44, 62 - V.bit_length())),
        grid=(B, 1, 1), block=(1024, 1, 1), inputs=[t.name for t in node.inputs], outputs=[node.outputs[0].name],
        params={"rows": B, "vocab": V}))


LOWERINGS = {"serving.paged_append.default": lower_paged_append,
             "serving.paged_attention.default": lower_paged_attention, "serving.sample.default": lower_sample}
