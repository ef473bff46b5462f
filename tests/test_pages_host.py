"""The page operations' refusals (include/dsa_gfx950.h dsa_pages_*, trnrt_amd/kernels/dsa_pages.py): every one is made on
the host, before any HIP call, so these run without a GPU."""

import ctypes

import pytest
import torch

from trnrt_amd import _lib
from trnrt_amd.kernels import dsa_pages

P = ctypes.c_void_p(256)  # never dereferenced


def _set(n=1, ptr=256, size=64):
    return (ctypes.c_void_p * n)(*[ptr] * n), (ctypes.c_longlong * n)(*[size] * n), n


def test_copy_refusals():
    lib = _lib.lib()
    c, s, n = _set()
    assert lib.dsa_pages_copy(c, s, n, P, P, -1, 4, None) == _lib.DSA_EINVAL
    assert lib.dsa_pages_copy(c, s, n, P, P, 1, 0, None) == _lib.DSA_EINVAL
    assert lib.dsa_pages_copy(None, None, 1, P, P, 1, 4, None) == _lib.DSA_EINVAL
    assert lib.dsa_pages_copy(c, s, -1, P, P, 1, 4, None) == _lib.DSA_EINVAL
    assert lib.dsa_pages_copy(*_set(ptr=0), P, P, 1, 4, None) == _lib.DSA_EINVAL  # a null cache
    assert lib.dsa_pages_copy(*_set(size=0), P, P, 1, 4, None) == _lib.DSA_EINVAL  # pages of no bytes
    assert lib.dsa_pages_copy(c, s, n, None, P, 1, 4, None) == _lib.DSA_EINVAL
    assert lib.dsa_pages_copy(*_set(size=1 << 40), P, P, 1, 4, None) == _lib.DSA_EUNSUPPORTED  # too many pieces
    assert lib.dsa_pages_copy(c, s, n, None, None, 0, 4, None) == _lib.DSA_OK  # nothing to do
    assert lib.dsa_pages_copy(None, None, 0, P, P, 1, 4, None) == _lib.DSA_OK


def test_fork_release_compact_refusals():
    lib = _lib.lib()
    c, s, k = _set()
    ws = lib.dsa_pages_workspace_bytes(100, 7)
    assert ws >= 7 * 4 and lib.dsa_pages_workspace_bytes(0, 1) == 0 and lib.dsa_pages_workspace_bytes(1, -1) == 0

    def fork(ref=P, table=P, wsp=P, size=ws, B=2, n=7, mp=4, ps=64, pages=100):
        return lib.dsa_pages_fork(ref, table, P, P, P, P, c, s, k, wsp, size, B, n, mp, ps, pages, None)

    assert fork(ref=None) == _lib.DSA_EINVAL and fork(table=None) == _lib.DSA_EINVAL
    assert fork(B=-1) == _lib.DSA_EINVAL and fork(n=-1) == _lib.DSA_EINVAL and fork(mp=0) == _lib.DSA_EINVAL
    assert fork(ps=0) == _lib.DSA_EINVAL and fork(pages=0) == _lib.DSA_EINVAL
    assert fork(wsp=None) == _lib.DSA_EWORKSPACE and fork(size=7 * 4 - 1) == _lib.DSA_EWORKSPACE
    assert fork(n=0) == _lib.DSA_OK
    assert lib.dsa_pages_release(None, P, P, 1, 4, 64, 100, None) == _lib.DSA_EINVAL
    assert lib.dsa_pages_release(P, P, P, -1, 4, 64, 100, None) == _lib.DSA_EINVAL
    assert lib.dsa_pages_release(P, P, P, 1, 4, 0, 100, None) == _lib.DSA_EINVAL
    assert lib.dsa_pages_release(None, None, None, 0, 4, 64, 100, None) == _lib.DSA_OK
    q, r, t, u = (ctypes.c_void_p(256 * i) for i in range(2, 6))

    def compact(ref=P, table=q, new_ref=r, new_table=t, remap=u, wsp=P, size=ws, B=2, mp=4, pages=100):
        return lib.dsa_pages_compact(ref, table, new_ref, new_table, remap, c, s, k, wsp, size, B, mp, pages, None)

    assert compact(ref=None) == _lib.DSA_EINVAL and compact(remap=None) == _lib.DSA_EINVAL
    assert compact(new_ref=P) == _lib.DSA_EINVAL and compact(new_table=q) == _lib.DSA_EINVAL  # in place
    assert compact(pages=0) == _lib.DSA_EINVAL and compact(mp=0) == _lib.DSA_EINVAL
    assert compact(pages=1 << 30) == _lib.DSA_EUNSUPPORTED
    assert compact(size=64) == _lib.DSA_EWORKSPACE


def test_host_tensors_and_shapes_raise():
    ref = torch.zeros(4, dtype=torch.int32)
    table, one = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    cache = torch.zeros(4 * 16, 8, dtype=torch.uint8)
    for call in (lambda: dsa_pages.fork(ref, table, one, one, [cache], 16),
                 lambda: dsa_pages.release(ref, table, one, 16),
                 lambda: dsa_pages.compact(ref, table, [cache], 16),
                 lambda: dsa_pages.copy([cache], one, one, 16)):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()
    with pytest.raises(ValueError, match="no caches"):
        dsa_pages.copy([], one, one, 16)
    with pytest.raises(ValueError, match="for 4 pages of 16"):
        dsa_pages._caches([torch.zeros(63, 8)], 16, 4, "x")
    with pytest.raises(ValueError, match="contiguous"):
        dsa_pages._caches([torch.zeros(64, 8).t()], 16, 4, "x")
    with pytest.raises(ValueError, match="pages of 0"):
        dsa_pages._caches([torch.zeros(64, 8)], 0, 4, "x")
    with pytest.raises(ValueError, match="ref"):
        dsa_pages._ref(torch.zeros(2, 2, dtype=torch.int32), "x")


def test_fork_refuses_pools_at_the_end_of_32_bits():
    """The search for free pages goes in steps of 4,096: past 2^31 - 4,096 pages its index would turn negative."""
    lib = _lib.lib()
    c, s, k = _set()
    for pages in (0x7fff0001, 0x7fffffff):
        assert lib.dsa_pages_fork(P, P, P, P, P, P, c, s, k, P, 1 << 20, 2, 7, 4, 64, pages, None) == _lib.DSA_EUNSUPPORTED


def test_fork_of_an_empty_table():
    """A table without rows has no parent: nothing of it is read, so it may be null."""
    lib = _lib.lib()
    c, s, k = _set()
    assert lib.dsa_pages_fork(P, P, P, P, P, P, c, s, k, None, 0, 0, 7, 4, 64, 100, None) == _lib.DSA_EWORKSPACE
    assert lib.dsa_pages_fork(P, None, None, P, P, P, c, s, k, None, 0, 0, 7, 4, 64, 100, None) == _lib.DSA_EWORKSPACE
    assert lib.dsa_pages_fork(P, None, None, P, P, P, c, s, k, P, 1 << 20, 1, 7, 4, 64, 100, None) == _lib.DSA_EINVAL
