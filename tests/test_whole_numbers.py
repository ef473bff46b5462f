"""Index arguments of other types than int32 (trnrt_amd/kernels/_common.py whole): wider ones do not wrap, others are refused."""

import pytest
import torch

from tests._helpers import say
from trnrt_amd.kernels import _common as C
from trnrt_amd.kernels import dsa_cache, dsa_expand, dsa_verify


def test_whole():
    top, low = 2 ** 31 - 1, -2 ** 31
    wide = torch.tensor([2 ** 63 - 1, -2 ** 63, 2 ** 32 + 5, -2 ** 32, top, low, 0, -1, 2 ** 31])
    got = C.whole(wide, "x")
    assert got.dtype is torch.int32 and got.tolist() == [top, low, top, low, top, low, 0, -1, top]
    assert C.whole(torch.tensor([2 ** 32 - 1, 7], dtype=torch.uint32), "x").tolist() == [top, 7]
    same = torch.arange(4, dtype=torch.int32)
    assert C.whole(same, "x") is same and C.whole(same[::2], "x").is_contiguous()
    for t in (torch.int16, torch.int8, torch.uint8):
        assert C.whole(same.to(t), "x").tolist() == [0, 1, 2, 3]
    for t in (torch.float32, torch.float64, torch.bfloat16, torch.bool, torch.complex64, torch.uint64):
        with pytest.raises(ValueError, match="x: dtype"):
            C.whole(torch.ones(2).to(t), "x")


@pytest.mark.gpu
def test_ranges_without_an_end():
    """last = 2^63 - 1 (no limit) and first = -2^63 leave everything to be seen, past the keys' number nothing."""
    say("int64 ranges")
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(n, 2, 128, generator=g).to(torch.bfloat16).cuda() for n in (40, 90, 90))
    cq, ck = (torch.tensor([0, n], dtype=torch.int32).cuda() for n in (40, 90))
    whole = dsa_expand.attend(q, k, None, v, cq, ck, 0.1, first=torch.zeros(40, dtype=torch.int32).cuda())
    for kw in (dict(last=torch.full((40,), 2 ** 63 - 1).cuda()), dict(first=torch.full((40,), -2 ** 63).cuda()),
               dict(last=torch.full((40,), 2 ** 32).cuda(), first=torch.full((40,), -2 ** 32 + 1).cuda())):
        got = dsa_expand.attend(q, k, None, v, cq, ck, 0.1, **kw)
        assert torch.equal(got[0], whole[0]) and torch.equal(got[1], whole[1])
    out, lse = dsa_expand.attend(q, k, None, v, cq, ck, 0.1, first=torch.full((40,), 2 ** 32).cuda())
    assert (out == 0).all() and (lse == -1e30).all()
    for kw in (dict(first=torch.zeros(40).cuda()), dict(last=torch.full((40,), float("inf")).cuda())):
        with pytest.raises(ValueError, match="dtype"):
            dsa_expand.attend(q, k, None, v, cq, ck, 0.1, **kw)


@pytest.mark.gpu
def test_drafts_and_ends():
    """A draft of 2^32 + 5 is no token (and not token 5); ends past the rows are their number; floats are refused."""
    say("int64 drafts")
    logits = torch.zeros(2, 50, device="cuda")
    logits[:, 5] = 9.0
    one = torch.ones(1, device="cuda")
    args = (torch.full((2,), 1e-3).cuda(), 0.5 * one, one)
    cu = torch.tensor([0, 2]).cuda()
    for draft, taken in ((5, 1), (2 ** 32 + 5, 0), (5 - 2 ** 32, 0)):
        tokens, accepted, _ = dsa_verify.verify(logits, torch.tensor([draft, 0]).cuda(), cu, *args)
        assert accepted.tolist() == [taken] and tokens.tolist() == [5, 5 if taken else -1]
    tokens, accepted, _ = dsa_verify.verify(logits, torch.tensor([5, 0]).cuda(), torch.tensor([-2 ** 40, 2 ** 40]).cuda(), *args)
    assert accepted.tolist() == [1] and tokens.tolist() == [5, 5]
    with pytest.raises(ValueError, match="dtype"):
        dsa_verify.verify(logits, torch.tensor([5.0, 0.0]).cuda(), cu, *args)
    with pytest.raises(ValueError, match="dtype"):
        dsa_verify.verify(logits, torch.tensor([5, 0]).cuda(), cu.float(), *args)


@pytest.mark.gpu
def test_pages_and_lengths():
    """A page or a length of 2^32 + 1 is outside the pool or the table (and not page 1 or a length of 1): nothing is written."""
    say("int64 pages")
    x = torch.ones(1, 64, device="cuda")
    for page, n, written in ((1, 1, True), (2 ** 32 + 1, 1, False), (1 - 2 ** 32, 1, False), (1, 2 ** 32 + 1, False),
                             (1, -2 ** 32 + 1, False)):
        cache = torch.zeros(32, 64, dtype=torch.bfloat16, device="cuda")
        table, ctx = torch.tensor([[page, 0]]).cuda(), torch.tensor([n]).cuda()
        dsa_cache.append(dsa_cache.Rows(x, cache), table, ctx, 16, cu_new=torch.tensor([0, 1]).cuda())
        assert bool((cache[16] == 1).all()) == written and (cache.sum() == 64 * written).all()
    for kw in (dict(table=table.float()), dict(ctx_len=ctx.float()), dict(cu_new=torch.tensor([0.0, 1.0]).cuda())):
        with pytest.raises(ValueError, match="dtype"):
            dsa_cache.append(dsa_cache.Rows(x, cache), **{**dict(table=table, ctx_len=ctx, page_size=16), **kw})
