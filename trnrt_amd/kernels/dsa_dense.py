"""Absorbed latent attention over every cached token on gfx950: the layer's attention where nothing is selected (contexts
up to the selection's size, layers without an indexer), for decode batches and for the few new tokens of a speculative step.

What it computes, per sequence b, new token i < S and head h, over the tokens t < ctx_len[b] - S + i + 1 (ctx_len counts
the S new tokens, whose rows are in the cache):
    s[t] = scale q[b, i, h] . K[t],  p = softmax(s),  o[b, i, h] = sum_t p[t] V[t],  lse = log sum_t exp(s[t])
with K[t] the cached FP8 latent row times its per-token scale, 576 wide (512 latent + 64 rope) or 512 (NoPE), and V[t] its
first 512 columns: dsa_decode.attend_tokens with every token selected. A query that sees no token has o = 0 and lse NEG_INF;
one that sees a NaN score has lse NaN. The weights p times the tokens' scales are bf16 in their product with the rows,
whatever out_dtype: off by 2^-8 of each at most where S * H > 32, and by 2^-16, in two bf16 terms, where S * H <= 32. Sums,
maxima and the lse are fp32.

The HIP kernel (csrc/dsa_dense.hip) shares the chunks of all sequences evenly among the GPU's workgroups, whatever the
lengths, so nothing about them is needed on the host.
"""

from __future__ import annotations

import torch

from .. import _lib
from . import _common as C
from .dsa_decode import DQK_WIDTHS, DV

NEG_INF = -1e30


def attend(q: torch.Tensor, kv_cache: torch.Tensor, kv_scale: torch.Tensor | None, table: torch.Tensor,
           ctx_len: torch.Tensor, page_size: int, scale: float, *, lse: bool = True, out_dtype=torch.bfloat16,
           out: torch.Tensor | None = None, workspace: torch.Tensor | None = None):
    """o [B, S, H, 512] in out_dtype (bf16 or fp32) and lse [B, S, H] fp32 (o alone without lse) of q [B, S, H, 576 or
    512] bf16; q [B, H, D] is one new token a sequence, its outputs [B, H, 512] and [B, H]. kv_cache [slots, D] e4m3fn (or
    its bits) with kv_scale [slots] fp32, or None for the unscaled cache; table [B, max_pages] int32, ctx_len [B] int32.
    Any number of heads, any page size. workspace: dsa_dense_workspace_bytes(S, H) bytes, or None for one kept per
    stream and host thread (a captured graph has its own)."""
    dev = C.on_gpu(q, kv_cache, kv_scale, table, ctx_len, out, workspace)
    rows = q.shape[:-1]  # B, (S,) H
    if len(rows) not in (2, 3) or q.shape[-1] not in DQK_WIDTHS or min(rows[1:]) < 1:
        raise ValueError(f"dsa_dense: q {tuple(q.shape)}, expected [B, H, 576 or 512] or [B, S, H, 576 or 512]")
    B, H, dqk = rows[0], rows[-1], q.shape[-1]
    S = rows[1] if len(rows) == 3 else 1
    q = C.aligned(C.as_bf16(q))
    if kv_cache.shape[-1] != dqk:
        raise ValueError(f"dsa_dense: cache rows of {kv_cache.shape[-1]} for q of {dqk}")
    kv = C.rows_of(C.fp8_bytes(kv_cache, "kv cache"), dqk)
    slots = kv.shape[0]
    if page_size < 1 or slots < 1 or slots % page_size:
        raise ValueError(f"dsa_dense: {slots} cache slots are not whole pages of {page_size}")
    if kv_scale is not None:
        kv_scale = C.need(C.flat(C.as_f32(kv_scale)), "kv_scale", torch.float32, (slots,))
    tb, lens = C.as_i32(table), C.need(C.as_i32(ctx_len), "ctx_len", torch.int32, (B,))
    if tb.dim() != 2 or tb.shape[0] != B or tb.shape[1] < 1:
        raise ValueError(f"dsa_dense: page table {tuple(table.shape)} for {B} sequences")
    if out is None:
        out = q.new_empty((*rows, DV), dtype=out_dtype)
    bf = C.need(out, "out", (torch.bfloat16, torch.float32), (*rows, DV)).dtype is torch.bfloat16
    ls = q.new_empty(rows, dtype=torch.float32) if lse else None
    lib = _lib.lib()
    if workspace is not None:
        ws = C.given(workspace, "dsa_dense")
    else:  # the partials of the row tiles that workgroups share
        ws = C.scratch(dev, int(lib.dsa_dense_workspace_bytes(S, H)), "dense")
    st = C.call(dev, lib.dsa_dense_mla, C.ptr(q), C.ptr(kv), C.ptr(kv_scale), C.ptr(tb), C.ptr(lens),
                C.ptr(out) if bf else None, None if bf else C.ptr(out), C.ptr(ls), C.ptr(ws),
                ws.numel() * ws.element_size(), B, S, H, dqk, tb.shape[1], int(page_size), slots // page_size,
                float(scale))
    _lib.check(st, "dsa_dense.attend")
    return (out, ls) if lse else out
