"""Expanded latent attention on gfx950, the form of a prefill where nothing is selected: the keys and values of every head
from the cached latent rows, and ragged causal attention over them.

    expand(kv_cache, kv_scale, table, cu_len, total, page_size, w)   k, k_rope, v of the sequences' cached tokens
    attend(q, k, k_rope, v, cu_q, cu_k, scale)                       o, lse of the queries

Per pair of tokens and head this costs 192 + 128 multiply-adds where the absorbed form (dsa_dense.attend) costs 576 + 512,
so it is the form for many queries a sequence; for one or a few, whose time is the cache's stream, it is dsa_dense.attend.
The two are the same attention: with w = [W_UK; W_UV] of each head, attend(q) equals dsa_dense.attend of the absorbed
queries (q_nope W_UK, q_rope) times W_UV^T, to rounding. The softmax weights are bf16 in their product with the values,
whatever out_dtype (off by 2^-8 of each at most); sums, maxima and the lse are fp32. A query that sees a NaN score has lse
NaN. The HIP kernels are in csrc/dsa_expand.hip.
"""

from __future__ import annotations

import torch

from .. import _lib
from . import _common as C
from .dsa_decode import DQK_WIDTHS, DV

NEG_INF = -1e30
DH = 128  # a head's key width without rope, and its value width
ROPE = 64


def expand(kv_cache: torch.Tensor, kv_scale: torch.Tensor | None, table: torch.Tensor, cu_len: torch.Tensor, total: int,
           page_size: int, w: torch.Tensor, *,
           out: tuple[torch.Tensor, torch.Tensor | None, torch.Tensor] | None = None
           ) -> tuple[torch.Tensor, torch.Tensor | None, torch.Tensor]:
    """(k [total, H, 128], k_rope [total, 64] or None, v [total, H, 128]) bf16 of the cached tokens of B sequences, one
    sequence after another: sequence b's first cu_len[b + 1] - cu_len[b] tokens are rows cu_len[b] .. (cu_len [B + 1]
    int32 on the device; total: the rows of the outputs, known to the host). kv_cache [slots, 576 or 512] e4m3fn with
    kv_scale [slots] fp32 or None, table [B, max_pages] int32, w [H, 256, 512] bf16: each head's key rows, then its value
    rows. k_rope is the rows' last 64 columns (None at width 512). out: the three outputs to write; rows from cu_len[B] on
    are left as they were."""
    dev = C.on_gpu(kv_cache, kv_scale, table, cu_len, w, *(out or ()))
    D = kv_cache.shape[-1]
    if D not in DQK_WIDTHS:
        raise ValueError(f"dsa_expand: cache rows of {D}, expected 576 or 512")
    kv = C.rows_of(C.fp8_bytes(kv_cache, "kv cache"), D)
    slots = kv.shape[0]
    if page_size < 1 or slots < 1 or slots % page_size:
        raise ValueError(f"dsa_expand: {slots} cache slots are not whole pages of {page_size}")
    if kv_scale is not None:
        kv_scale = C.need(C.flat(C.as_f32(kv_scale)), "kv_scale", torch.float32, (slots,))
    if w.dim() != 3 or w.shape[0] < 1:
        raise ValueError(f"dsa_expand: w {tuple(w.shape)}, expected [H, {2 * DH}, {DV}]")
    H = w.shape[0]
    w = C.aligned(C.need(w, "w", torch.bfloat16, (H, 2 * DH, DV)))
    tb = C.as_i32(table)
    if tb.dim() != 2 or tb.shape[1] < 1:
        raise ValueError(f"dsa_expand: page table {tuple(table.shape)}, expected [B, max_pages]")
    B, total = tb.shape[0], int(total)
    if total < 0:
        raise ValueError(f"dsa_expand: {total} rows")
    cu = C.need(C.as_i32(cu_len), "cu_len", torch.int32, (B + 1,))
    if out is None:
        k, v = w.new_empty((total, H, DH)), w.new_empty((total, H, DH))
        r = w.new_empty((total, ROPE)) if D > DV else None
    else:
        k, r, v = out
        C.need(k, "k", torch.bfloat16, (total, H, DH))
        C.need(v, "v", torch.bfloat16, (total, H, DH))
        if (r is None) != (D == DV):
            raise ValueError(f"dsa_expand: a rope output for cache rows of {D}" if r is not None else
                             "dsa_expand: no rope output")
        if r is not None:
            C.need(r, "k_rope", torch.bfloat16, (total, ROPE))
    st = C.call(dev, _lib.lib().dsa_expand_latent, C.ptr(kv), C.ptr(kv_scale), C.ptr(tb), C.ptr(cu), C.ptr(w), C.ptr(k),
                C.ptr(v), C.ptr(r), B, total, H, D, tb.shape[1], int(page_size), slots // page_size)
    _lib.check(st, "dsa_expand.expand")
    return k, r, v


def attend(q: torch.Tensor, k: torch.Tensor, k_rope: torch.Tensor | None, v: torch.Tensor, cu_q: torch.Tensor,
           cu_k: torch.Tensor, scale: float, *, causal: bool = True, lse: bool = True, out_dtype=torch.bfloat16,
           out: torch.Tensor | None = None, workspace: torch.Tensor | None = None):
    """o [Tq, H, 128] in out_dtype (bf16 or fp32) and lse [Tq, H] fp32 (o alone without lse) of ragged sequences: q
    [Tq, H, 192] bf16 with k_rope [Tk, 64] bf16 shared by the heads, or [Tq, H, 128] without (k_rope None); k, v
    [Tk, H, 128] bf16; cu_q, cu_k [B + 1] int32 on the device: sequence b's queries are rows cu_q[b] .. cu_q[b + 1] - 1,
    its keys rows cu_k[b] .. . causal: query i of nq sees the first nk - nq + i + 1 of the nk keys (the last sees all);
    otherwise every key. A query that sees no key has o = 0 and lse NEG_INF; rows of q in no sequence are not written.
    workspace: dsa_expanded_workspace_bytes(B, Tq, Tk, H) bytes, or None for one kept per stream and host thread (a
    captured graph has its own)."""
    dev = C.on_gpu(q, k, k_rope, v, cu_q, cu_k, out, workspace)
    dq = DH if k_rope is None else DH + ROPE
    if q.dim() != 3 or q.shape[1] < 1 or q.shape[2] != dq:
        raise ValueError(f"dsa_expand: q {tuple(q.shape)}, expected [Tq, H, {dq}]")
    Tq, H = q.shape[:2]
    q = C.aligned(C.as_bf16(q))
    if k.dim() != 3:
        raise ValueError(f"dsa_expand: k {tuple(k.shape)}, expected [Tk, {H}, {DH}]")
    Tk = k.shape[0]
    k = C.aligned(C.need(C.as_bf16(k), "k", torch.bfloat16, (Tk, H, DH)))
    v = C.aligned(C.need(C.as_bf16(v), "v", torch.bfloat16, (Tk, H, DH)))
    r = None if k_rope is None else C.aligned(C.need(C.as_bf16(k_rope), "k_rope", torch.bfloat16, (Tk, ROPE)))
    if cu_q.dim() != 1 or cu_q.shape != cu_k.shape or cu_q.numel() < 1:
        raise ValueError(f"dsa_expand: cu_q {tuple(cu_q.shape)} and cu_k {tuple(cu_k.shape)}, expected [B + 1]")
    cq, ck = C.as_i32(cu_q), C.as_i32(cu_k)
    if out is None:
        out = q.new_empty((Tq, H, DH), dtype=out_dtype)
    C.need(out, "out", (torch.bfloat16, torch.float32), (Tq, H, DH))
    ls = q.new_empty((Tq, H), dtype=torch.float32) if lse else None
    bf = out.dtype == torch.bfloat16
    lib, B = _lib.lib(), cu_q.numel() - 1
    if workspace is not None:
        ws = C.given(workspace, "dsa_expand")
    else:
        need = int(lib.dsa_expanded_workspace_bytes(B, Tq, Tk, H))
        ws = C.scratch(dev, need, "expanded") if need else None
    st = C.call(dev, lib.dsa_expanded_mla, C.ptr(q), C.ptr(k), C.ptr(r), C.ptr(v), C.ptr(cq), C.ptr(ck),
                C.ptr(out) if bf else None, None if bf else C.ptr(out), C.ptr(ls), C.ptr(ws),
                0 if ws is None else ws.numel() * ws.element_size(), B, Tq, Tk, H,
                int(bool(causal)), float(scale))
    _lib.check(st, "dsa_expand.attend")
    return (out, ls) if lse else out
