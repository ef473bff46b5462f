"""Quantise-on-write into the paged FP8 caches on gfx950: the cache-store step before the DSA path (the operator of
trnrt/models/decoder.py:481-486 `_store`, which trnrt/models/mla.py:445-446 calls for the latent rows and the
indexer-key rows at the step's slot_mapping).

    store(cache, slots, x, fp8_max)             the reference's form: cache[slot] = e4m3fn(clamp(x, +-fp8_max))
    store(cache, slots, x, fp8_max, scale=s)    this build's format: per-token s = max(absmax(row), 1e-30) / 448,
                                                cache[slot] = e4m3fn(clamp(x / s, +-fp8_max)), s[slot] = s

The HIP kernel (csrc/dsa_cache.hip) converts each row in one wave: fp32 arithmetic with a correctly rounded
division and round-to-nearest-even into e4m3fn, which is torch's float -> float8_e4m3fn cast.

append takes a step's rows as the projections leave them, norms and rotates them on the way, finds their slots through the
page table and writes all kinds of them (latent rows, indexer keys) in one launch (csrc/dsa_append.hip).

write_pool_keys is the pooled (GLM) indexer's key write of the same step (trnrt/models/mla.py:1277-1296): each written
token's pool key, a softmax-gated mean of the pool's cached indexer keys, into the pool-key cache.
"""

from __future__ import annotations

import ctypes
import struct
from collections.abc import Sequence

import torch

from .. import _lib
from . import _common as C
from .dsa_rope import axis_map

_FORMAT = "".join(t._type_ for _, t in _lib.AppendRows._fields_)  # (packed in 0.4 us, where ctypes fills one in 1.3)
_KIND = struct.Struct(f"{_FORMAT}{ctypes.sizeof(_lib.AppendRows) - struct.calcsize(_FORMAT)}x")
_SIZES = {torch.bfloat16: 2, torch.float32: 4}
FP8_MAX = 448.0  # the e4m3fn maximum (trnrt/engine/model_runner.py:62-70 off Neuron)


def slots_of(positions: torch.Tensor, table: torch.Tensor, page_size: int) -> torch.Tensor:
    """Cache slots of token positions [T] through one sequence's table [P] or per-row tables [T, P]
    (trnrt/models/decoder.py:658-667 `_slots` for one position per row): table[pos // ps] * ps + pos % ps, int64."""
    pos = positions.to(torch.int64)
    tb = table.to(torch.int64)
    pages = tb[pos // page_size] if tb.dim() == 1 else tb.gather(1, (pos // page_size).view(-1, 1)).view(-1)
    return pages * page_size + pos % page_size


def store(cache: torch.Tensor, slots: torch.Tensor, x: torch.Tensor, fp8_max: float = FP8_MAX, *,
          scale: torch.Tensor | None = None) -> None:
    """Writes the rows x [T, W] (or [T, 1, W]; bf16 or fp32) into cache [slots, W] (or [slots, 1, W]; e4m3fn or its
    uint8 bits) at slots [T] int64, in place, on the current stream. With scale [slots] fp32 (this build's format)
    each row gets its own scale; without, the rows are clamped and cast as the reference does (KV scale 1.0). Rows
    whose slot is outside the cache are not written."""
    dev = C.on_gpu(cache, slots, x, scale)
    if cache.dtype not in (C.FP8, torch.uint8):
        raise NotImplementedError(f"dsa_cache.store: a {cache.dtype} cache; the kernel writes float8_e4m3fn caches")
    if not cache.is_contiguous():
        raise ValueError("dsa_cache.store: the cache must be contiguous")
    W = cache.shape[-1]
    num_slots = cache.numel() // W
    if x.shape[-1] != W or x.numel() % W:
        raise ValueError(f"dsa_cache.store: rows {tuple(x.shape)} for a cache of width {W}")
    T = x.numel() // W
    if x.dtype == torch.bfloat16:
        x_fp32 = 0
    elif x.dtype == torch.float32:
        x_fp32 = 1
    else:
        raise ValueError(f"dsa_cache.store: rows of dtype {x.dtype}, expected bfloat16 or float32")
    x = x.contiguous()
    # a step's two stores of a few us each are bound by this function: no tensor operation that changes nothing
    if slots.dim() != 1 or slots.dtype != torch.int64 or not slots.is_contiguous():
        slots = slots.reshape(-1).to(torch.int64).contiguous()
    C.need(slots, "slots", torch.int64, (T,))
    if scale is not None:
        scale = C.need(scale if scale.dim() == 1 else scale.reshape(-1), "scale", torch.float32, (num_slots,))
    if not 0.0 < fp8_max <= FP8_MAX:
        raise ValueError(f"dsa_cache.store: fp8_max {fp8_max} outside (0, {FP8_MAX}]")
    st = _lib.lib().dsa_cache_write(C.ptr(x), x_fp32, C.ptr(slots), C.ptr(cache), C.ptr(scale), T, W, num_slots,
                                    int(scale is not None), float(fp8_max), C.stream_ptr(dev))
    _lib.check(st, "dsa_cache.store")


class Rows:
    """One kind of rows for append: x [T, W] (bf16 or fp32; a view of a wider projection's columns will do) into cache
    [slots, W] (or [slots, 1, W]; e4m3fn or its uint8 bits, with scale [slots] fp32 or unscaled; or bf16).

    rope_at: the first of the 2R columns that are rotated (None: none), interleaved: their pairs as in dsa_rope.rotate.
    norm: a weight [n] for the root-mean-square norm of the first n columns, or (weight, bias) for their layer norm (bf16 or
    fp32), with eps."""

    __slots__ = ("x", "cache", "scale", "rope_at", "interleaved", "norm", "eps", "fp8_max")

    def __init__(self, x: torch.Tensor, cache: torch.Tensor, scale: torch.Tensor | None = None, *,
                 rope_at: int | None = None, interleaved: bool = True,
                 norm: torch.Tensor | tuple[torch.Tensor, torch.Tensor] | None = None, eps: float = 1e-6,
                 fp8_max: float = FP8_MAX):
        self.x, self.cache, self.scale, self.rope_at, self.interleaved = x, cache, scale, rope_at, interleaved
        self.norm, self.eps, self.fp8_max = norm, eps, fp8_max


def _norm(norm, width: int):
    """(weight, bias) of one type, starting at multiples of 16 bytes."""
    w, b = norm if isinstance(norm, (tuple, list)) else (norm, None)
    if b is not None and (b.shape != w.shape or b.device != w.device):
        raise ValueError(f"dsa_cache.append: norm weight {tuple(w.shape)} and bias {tuple(b.shape)}")
    if w.dim() != 1 or not 1 <= w.shape[0] <= width:
        raise ValueError(f"dsa_cache.append: norm weight {tuple(w.shape)} for rows of {width}")
    if w.dtype not in (torch.bfloat16, torch.float32) or (b is not None and b.dtype is not w.dtype):
        w, b = w.float(), None if b is None else b.float()
    return C.aligned(w.contiguous()), None if b is None else C.aligned(b.contiguous())


def append(rows: Rows | Sequence[Rows], table: torch.Tensor, ctx_len: torch.Tensor, page_size: int, *,
           cu_new: torch.Tensor | None = None, positions: torch.Tensor | None = None, inv_freq: torch.Tensor | None = None,
           axes: Sequence[int] | None = None, factor: float = 1.0) -> None:
    """The rows of T new tokens of B sequences into the paged caches, in place, on the current stream: sequence b's are rows
    cu_new[b] .. cu_new[b + 1] - 1 of every x (cu_new [B + 1] int32; None: T / B each) and the last of its ctx_len[b] tokens
    (ctx_len [B] int32 counts the new ones), through table [B, max_pages] int32. The columns that a kind names are rotated
    by positions ([T], or [axes, T] with axes, as in dsa_rope.rotate; None: the token's place in its sequence) x inv_freq
    [R] fp32 x factor (without inv_freq no kind is rotated, and positions and axes are not used). Everything is in fp32 and
    rounded once, as store rounds. A token whose place is outside the table, or whose page is the null page or outside the
    pool, is not written, nor are rows in no sequence. No two tokens of a call may have one slot. (table, ctx_len and cu_new
    may be int64: values past int32's ends are these.)"""
    rows = (rows,) if isinstance(rows, Rows) else rows
    if not rows:
        raise ValueError("dsa_cache.append: no rows")
    dev = C.on_gpu(table, ctx_len, cu_new, positions, inv_freq)
    if table.dim() != 2 or table.shape[1] < 1 or page_size < 1:
        raise ValueError(f"dsa_cache.append: table {tuple(table.shape)} with pages of {page_size}")
    B, max_pages = table.shape
    tb, lens = C.whole(table, "table"), C.need(C.whole(ctx_len, "ctx_len"), "ctx_len", torch.int32, (B,))
    cu = None if cu_new is None else C.need(C.whole(cu_new, "cu_new"), "cu_new", torch.int32, (B + 1,))
    R = 0
    if inv_freq is not None:
        R = C.need(inv_freq, "inv_freq", torch.float32, (None,)).shape[0]
    T = slots = None
    kinds = b""  # (a step's call of a few us is bound by this function: packed, with few tensor attributes asked twice)
    held = []  # what tensors were copied to, until the launch
    on = table.get_device()
    for r in rows:
        x, cache, scale, norm, at = r.x, r.cache, r.scale, r.norm, r.rope_at
        if x.get_device() != on or cache.get_device() != on or (scale is not None and scale.get_device() != on):
            C.on_gpu(table, x, cache, scale)
        size = _SIZES.get(x.dtype)
        if size is None:
            raise ValueError(f"dsa_cache.append: rows of {x.dtype}, expected bfloat16 or float32")
        if x.dim() != 2:  # (a copy, where the strides do not merge)
            x = x.reshape(-1, x.shape[-1])
            held.append(x)
        t, W = x.shape
        if cache.shape[-1] != W or W == 0:
            raise ValueError(f"dsa_cache.append: rows {tuple(x.shape)} for a cache of width {cache.shape[-1]}")
        bf = cache.dtype is torch.bfloat16
        if not bf and cache.dtype is not C.FP8 and cache.dtype is not torch.uint8:
            raise NotImplementedError(f"dsa_cache.append: a {cache.dtype} cache; it is float8_e4m3fn or bfloat16")
        to = cache.data_ptr()
        if not cache.is_contiguous() or to % 16:
            raise ValueError("dsa_cache.append: the cache must be contiguous and start at a multiple of 16 bytes")
        n = cache.shape[0] if cache.dim() == 2 else cache.numel() // W
        if T is None:
            T, slots = t, n
        if t != T or n != slots or n < 1 or n % page_size:
            raise ValueError(f"dsa_cache.append: {t} rows of {T}, {n} cache slots of {slots} in pages of {page_size}")
        row, col = x.stride()
        if col != 1 or x.data_ptr() % 16 or (T > 1 and (row * size % 16 or row < W)):
            x = x.clone(memory_format=torch.contiguous_format)
            held.append(x)
            row = W
        elif T <= 1:  # (a single row's stride says nothing)
            row = W
        if at is None:
            at = -1
        elif not (R and 0 <= at <= W - 2 * R):
            raise ValueError(f"dsa_cache.append: {2 * R} rotated columns from {at} on in rows of {W}")
        if scale is not None:  # (written in place: no copy of one that is not contiguous)
            scale = C.need(C.flat(C.need(scale, "scale", torch.float32)), "scale", torch.float32, (slots,)).data_ptr()
        w = b = norm_fp32 = norm_width = 0
        if norm is not None:
            norm = _norm(norm, W)
            C.on_gpu(table, *norm)
            held.append(norm)
            w, b = norm[0].data_ptr(), 0 if norm[1] is None else norm[1].data_ptr()
            norm_fp32, norm_width = norm[0].dtype is torch.float32, norm[0].shape[0]
        kinds += _KIND.pack(x.data_ptr(), row, w, b, to, scale or 0, size == 4, W, at, bool(r.interleaved), norm_fp32,
                            norm_width, bf, r.eps, r.fp8_max)
    if cu is None and T and (not B or T % B):
        raise ValueError(f"dsa_cache.append: {T} rows for {B} sequences without cu_new")
    pos, n_axes, which = axis_map(axes, positions, R, T, "dsa_cache.append") if R else (None, 1, None)
    st = C.call(dev, _lib.lib().dsa_cache_append, kinds, len(rows), tb.data_ptr(), lens.data_ptr(), C.ptr(cu), C.ptr(pos),
                C.ptr(inv_freq), which, T, B, R, n_axes, factor, max_pages, page_size, slots // page_size)
    _lib.check(st, "dsa_cache.append")


def write_pool_keys(pool_key: torch.Tensor, rows: torch.Tensor, positions: torch.Tensor, table: torch.Tensor,
                    slot_mapping: torch.Tensor, ape: torch.Tensor, page_size: int, kp: int, *,
                    rows_scale: torch.Tensor | None = None) -> None:
    """Recomputes the pool key of every written token's pool and writes it to pool_key [slots, 128 / kp] bf16 as kp
    pieces, one per slot of the pool (trnrt/models/mla.py:1277-1296 `write_pool_keys`, glm5_next.py:151-160
    `pool_keys`): rows the cached indexer rows [slots, W >= 256] ([key 128 | gate logits 128], e4m3fn with optional
    per-token rows_scale, or bf16), positions [T], table [T, Pp] or one [Pp], slot_mapping [T] (a padded row, in the
    null page, writes only its own slot), ape [kp, 128] (the pool-position bias, idx_pool_ape)."""
    dev = C.on_gpu(pool_key, rows, positions, table, slot_mapping, ape, rows_scale)
    if pool_key.dtype != torch.bfloat16 or not pool_key.is_contiguous():
        raise ValueError("dsa_cache.write_pool_keys: pool_key must be a contiguous bf16 cache")
    W = rows.shape[-1]
    num_slots = rows.numel() // W
    if pool_key.numel() != num_slots * (128 // kp):
        raise ValueError(f"dsa_cache.write_pool_keys: pool_key {tuple(pool_key.shape)} for {num_slots} slots, kp {kp}")
    fp8 = rows.dtype in (C.FP8, torch.uint8)
    if not fp8 and rows.dtype != torch.bfloat16:
        raise ValueError(f"dsa_cache.write_pool_keys: rows of dtype {rows.dtype}")
    if not rows.is_contiguous():
        raise ValueError("dsa_cache.write_pool_keys: rows must be contiguous")
    T = positions.numel()
    pos = C.need(C.as_i32(positions.reshape(-1)), "positions", torch.int32, (T,))
    sm = C.need(slot_mapping.reshape(-1).to(torch.int64).contiguous(), "slot_mapping", torch.int64, (T,))
    tb = C.as_i32(table)
    if tb.dim() not in (1, 2) or (tb.dim() == 2 and tb.shape[0] != T):
        raise ValueError(f"dsa_cache.write_pool_keys: table {tuple(table.shape)} for {T} rows")
    ap = C.need(C.as_f32(ape), "ape", torch.float32, (kp, 128))
    rs = None if rows_scale is None else C.need(C.as_f32(rows_scale).reshape(-1), "rows_scale", torch.float32,
                                                 (num_slots,))
    st = _lib.lib().dsa_pool_keys_write(C.ptr(rows), int(fp8), C.ptr(rs), W, C.ptr(ap), C.ptr(pos), C.ptr(tb),
                                        int(tb.dim() == 1), tb.shape[-1], C.ptr(sm), C.ptr(pool_key), T, kp,
                                        page_size, num_slots, C.stream_ptr(dev))
    _lib.check(st, "dsa_cache.write_pool_keys")
