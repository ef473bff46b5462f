"""Pages of the paged caches on gfx950: copying, forking, releasing and compacting them, in every cache at once.

The pool is a use count per page on the device, ref [num_pages] int32 (0: free; page 0 is the null page, never given
out, counted or moved), beside the page tables [rows, max_pages] and the caches that they index (latent rows, indexer
keys, scales, pool keys, of one layer or of all: any contiguous tensor whose first dimension is the pool's slots):

    fork(ref, table, ctx_len, parents, caches, page_size)    n new sequences that share their parents' full pages
    release(ref, table, ctx_len, page_size)                  sequences that ended
    compact(ref, table, caches, page_size)                   the pages in use moved to the pool's front
    copy(caches, src, dst, page_size)                        pages src[i] -> dst[i]

The reference keeps its page pool on the host (trnrt/engine/kv_pool.py:1-50). Here nothing comes back to the host, so a
step with forks in it can be captured in a graph; choices are in ascending order and do not vary from run to run. The HIP
kernels (csrc/dsa_pages.hip) move a page of all caches in one launch.
"""

from __future__ import annotations

import ctypes

import torch

from .. import _lib
from . import _common as C


def _caches(caches, page_size: int, num_pages: int | None, what: str):
    """(device pointers, bytes per page, count, pages of the pool) of the caches; num_pages None: the first cache's."""
    caches = list(caches)
    if page_size < 1:
        raise ValueError(f"{what}: pages of {page_size}")
    for c in caches:
        if not c.is_contiguous() or c.dim() < 1:
            raise ValueError(f"{what}: a cache must be contiguous, its first dimension the pool's slots")
        if num_pages is None:
            num_pages = c.shape[0] // page_size
        if c.shape[0] != num_pages * page_size or c.numel() == 0:
            raise ValueError(f"{what}: a cache of {tuple(c.shape)} for {num_pages} pages of {page_size}")
    n = len(caches)
    ptrs = (ctypes.c_void_p * max(n, 1))(*[c.data_ptr() for c in caches])
    size = (ctypes.c_longlong * max(n, 1))(*[c.numel() // num_pages * c.element_size() for c in caches])
    return ptrs, size, n, num_pages


def _ref(ref: torch.Tensor, what: str) -> torch.Tensor:
    if ref.dim() != 1 or ref.numel() < 1:
        raise ValueError(f"{what}: ref {tuple(ref.shape)}, expected [num_pages]")
    return C.need(ref, "ref", torch.int32)


def copy(caches, src: torch.Tensor, dst: torch.Tensor, page_size: int) -> None:
    """Page src[i] -> page dst[i] of every cache, in place, on the current stream. A pair with an id outside the pool,
    with dst the null page or with src == dst is skipped; no dst may be a src or another pair's dst."""
    caches = list(caches)
    if not caches:
        raise ValueError("dsa_pages.copy: no caches")
    dev = C.on_gpu(*caches, src, dst)
    ptrs, size, n_caches, num_pages = _caches(caches, page_size, None, "dsa_pages.copy")
    if src.dim() != 1 or src.shape != dst.shape:
        raise ValueError(f"dsa_pages.copy: src {tuple(src.shape)}, dst {tuple(dst.shape)}")
    src, dst = C.as_i32(src), C.as_i32(dst)
    st = C.call(dev, _lib.lib().dsa_pages_copy, ptrs, size, n_caches, C.ptr(src), C.ptr(dst), src.numel(), num_pages)
    _lib.check(st, "dsa_pages.copy")


def fork(ref: torch.Tensor, table: torch.Tensor, ctx_len: torch.Tensor, parents: torch.Tensor, caches,
         page_size: int, *, workspace: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """n new sequences, child i of row parents[i] of table [B, max_pages] int32 with ctx_len [B] tokens: (child_table
    [n, max_pages] int32, pages [n] int32). The parent's full pages are shared (ref, in place, rises by one), a partial
    last page is copied into the lowest free page of every cache; pages[i] is that page, 0 where there is no partial page,
    -1 where the pool had none left or parents[i] is no row (the child's table row is then 0 and counts nothing).
    workspace: dsa_pages_workspace_bytes(num_pages, n) bytes, or None for one kept per stream and host
    thread (a captured graph has its own)."""
    caches = list(caches)
    dev = C.on_gpu(ref, table, ctx_len, parents, workspace, *caches)
    _ref(ref, "dsa_pages.fork")
    ptrs, size, n_caches, num_pages = _caches(caches, page_size, ref.numel(), "dsa_pages.fork")
    if table.dim() != 2 or table.shape[1] < 1:
        raise ValueError(f"dsa_pages.fork: table {tuple(table.shape)}, expected [B, max_pages]")
    B, max_pages = table.shape
    if parents.dim() != 1:
        raise ValueError(f"dsa_pages.fork: parents {tuple(parents.shape)}, expected [n]")
    n = parents.numel()
    tb, par = C.as_i32(table), C.as_i32(parents)
    lens = C.need(C.as_i32(ctx_len), "ctx_len", torch.int32, (B,))
    child, pages = tb.new_empty((n, max_pages)), tb.new_empty((n,))
    lib = _lib.lib()
    if workspace is not None:
        ws = C.given(workspace, "dsa_pages")
    else:
        ws = C.scratch(dev, int(lib.dsa_pages_workspace_bytes(num_pages, n)), "pages")
    st = C.call(dev, lib.dsa_pages_fork, C.ptr(ref), C.ptr(tb), C.ptr(lens), C.ptr(par), C.ptr(child), C.ptr(pages),
                ptrs, size, n_caches, C.ptr(ws), ws.numel() * ws.element_size(), B, n, max_pages, int(page_size),
                num_pages)
    _lib.check(st, "dsa_pages.fork")
    return child, pages


def release(ref: torch.Tensor, table: torch.Tensor, ctx_len: torch.Tensor, page_size: int) -> None:
    """The rows of table [n, max_pages] int32 give up the pages of their ctx_len [n] tokens: ref, in place, falls by one
    for each, never below 0."""
    dev = C.on_gpu(ref, table, ctx_len)
    _ref(ref, "dsa_pages.release")
    if table.dim() != 2 or table.shape[1] < 1:
        raise ValueError(f"dsa_pages.release: table {tuple(table.shape)}, expected [n, max_pages]")
    n, max_pages = table.shape
    tb, lens = C.as_i32(table), C.need(C.as_i32(ctx_len), "ctx_len", torch.int32, (n,))
    st = C.call(dev, _lib.lib().dsa_pages_release, C.ptr(ref), C.ptr(tb), C.ptr(lens), n, max_pages, int(page_size),
                ref.numel())
    _lib.check(st, "dsa_pages.release")


def compact(ref: torch.Tensor, table: torch.Tensor, caches, page_size: int, *,
            workspace: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The L pages in use moved to pages 1 .. L of every cache: (table, ref, remap), the table [B, max_pages] and the
    counts in the new places and each page's new place [num_pages] (0: a free page), all int32. Pages already up to L
    stay; the k-th one past L goes to the k-th free page. ref and table are not changed, the caches are, in place (pages
    past L keep their bytes). Table entries of free pages become 0. workspace: dsa_pages_workspace_bytes(num_pages, 0)
    bytes, or None for one kept per stream and host thread (a captured graph has its own)."""
    caches = list(caches)
    dev = C.on_gpu(ref, table, workspace, *caches)
    _ref(ref, "dsa_pages.compact")
    ptrs, size, n_caches, num_pages = _caches(caches, page_size, ref.numel(), "dsa_pages.compact")
    if table.dim() != 2 or table.shape[1] < 1:
        raise ValueError(f"dsa_pages.compact: table {tuple(table.shape)}, expected [B, max_pages]")
    B, max_pages = table.shape
    tb = C.as_i32(table)
    new_table = tb.new_empty((B, max_pages))
    new_ref, remap = torch.empty_like(ref), torch.empty_like(ref)
    lib = _lib.lib()
    if workspace is not None:
        ws = C.given(workspace, "dsa_pages")
    else:
        ws = C.scratch(dev, int(lib.dsa_pages_workspace_bytes(num_pages, 0)), "pages")
    st = C.call(dev, lib.dsa_pages_compact, C.ptr(ref), C.ptr(tb), C.ptr(new_ref), C.ptr(new_table), C.ptr(remap), ptrs,
                size, n_caches, C.ptr(ws), ws.numel() * ws.element_size(), B, max_pages, num_pages)
    _lib.check(st, "dsa_pages.compact")
    return new_table, new_ref, remap
