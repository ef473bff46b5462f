"""Appends to the paged caches (dsa_cache.append) against their definition in float64, and bit for bit against dsa_cache.store
where nothing happens on the way.

Tolerances, from the arithmetic. A normed or rotated value is off by less than 4e-6 of the row's largest size: the norm's
sum of squares is 16 sums in a lane and 6 across lanes, all of one sign (22 2^-24 of it, half of that in the root), the root,
the quotient, the difference and two products another 6 2^-24, so 17 2^-24 = 1e-6; the rotation 1e-6 of |x0| + |x1| (as in
the rotation's own tests) in fp32; a layer norm's mean is off by 22 2^-24 of the mean size, which eps and the spread keep
below 1e-6 of the largest for these inputs. The scale has the same error relative to itself; a code, up to 448, is then
off by less than 448 x 6e-6 before it is rounded to e4m3: by at most 2^-4 of itself, or 2^-10 below the least normal."""

import pytest
import torch

from tests._helpers import say
from tests.test_gpu_rope import freqs, reference as rotated
from trnrt_amd.kernels import dsa_cache, dsa_rope
from trnrt_amd.kernels.dsa_cache import Rows

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


def setup(new, old, ps, seed, spare=2, shuffle=True):
    """Page tables of sequences with new[b] new tokens behind old[b]: (cu, ctx_len, table, slots, token's slot, its place)."""
    g = torch.Generator().manual_seed(seed)
    ctx = [a + b for a, b in zip(new, old)]
    npg = [-(-n // ps) for n in ctx]
    pages = 1 + sum(npg) + spare
    perm = torch.randperm(pages - 1, generator=g) + 1 if shuffle else torch.arange(1, pages)
    table = torch.zeros(len(new), max(max(npg), 1), dtype=torch.int32)
    slot, place, at = [], [], 0
    for b, n in enumerate(npg):
        table[b, :n] = perm[at:at + n]
        at += n
        p = torch.arange(ctx[b] - new[b], ctx[b])
        slot.append(table[b][p // ps].long() * ps + p % ps)
        place.append(p)
    cu = torch.tensor([0] + new).cumsum(0).to(torch.int32)
    return cu.cuda(), torch.tensor(ctx, dtype=torch.int32).cuda(), table.cuda(), pages * ps, torch.cat(slot), torch.cat(place)


def normed(x, norm, eps):
    if norm is None:
        return x
    w, b = norm if isinstance(norm, tuple) else (norm, None)
    n = w.shape[0]
    y = x[:, :n]
    if b is None:
        y = y / (y.square().mean(1, keepdim=True) + eps).sqrt() * w.cpu().double()
    else:
        y = y - y.mean(1, keepdim=True)
        y = y / (y.square().mean(1, keepdim=True) + eps).sqrt() * w.cpu().double() + b.cpu().double()
    return torch.cat([y, x[:, n:]], 1)


def expected(x, pos, freq, axes, rope_at, half, norm, eps=1e-6, factor=1.0):
    y = normed(x.cpu().double(), norm, eps)
    if rope_at is not None:
        R = freq.shape[0]
        part = rotated(y[:, None, rope_at:rope_at + 2 * R], pos, freq, axes, half, factor)[0][:, 0]
        y = torch.cat([y[:, :rope_at], part, y[:, rope_at + 2 * R:]], 1)
    return y


def check(cache, scale, before, slot, y):
    """The written rows, and that nothing else was."""
    rest = torch.ones(cache.shape[0], dtype=torch.bool)
    rest[slot] = False
    assert torch.equal(cache.view(torch.uint8).cpu()[rest], before.view(torch.uint8).cpu()[rest])
    if cache.dtype == torch.bfloat16:
        tol = 2.0 ** -8 * y.abs() + 6e-6 * y.abs().amax(1, keepdim=True)
        assert ((cache.cpu()[slot].double() - y).abs() <= tol).all()
        return
    s = y.abs().amax(1).clamp(min=1e-30) / 448
    if scale is not None:
        assert (scale.cpu()[rest] == 7).all()
        assert ((scale.cpu()[slot].double() - s).abs() <= 6e-6 * s).all()
        code = y / s[:, None]
    else:
        code = y.clamp(-448, 448)
    tol = (code.abs() * 2.0 ** -4).clamp(min=2.0 ** -10) + 448 * 6e-6
    err = (cache.view(FP8).cpu()[slot].double() - code).abs()
    assert (err <= tol).all(), f"codes off by {float((err / tol).max())} of the tolerance"


@pytest.mark.parametrize("new,old,ps", [
    ([1], [0], 64), ([1] * 8, [31, 64, 0, 4095, 63, 1, 128, 700], 64), ([5] * 13, [60] * 13, 64), ([0, 3, 0, 200, 1, 0], [9] * 6, 16),
    ([333, 1000], [0, 77], 64), ([1] * 300, list(range(300)), 1), ([0] * 70 + [9] + [0] * 5000 + [4, 70] + [0] * 3, [3] * 5076, 33),
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("norm", [False, True])
def test_append(new, old, ps, dtype, norm):
    """Latent rows (views of a projection's wider rows) and indexer keys, each with its own rotation and norm."""
    say("append", len(new), sum(new), ps, dtype, norm)
    cu, ctx, table, slots, slot, place = setup(new, old, ps, len(new))
    g = torch.Generator().manual_seed(sum(new))
    T, spare = sum(new), 3
    wide = torch.randn(T + spare, 64 + 576, generator=g) * torch.exp(torch.randn(T + spare, 1, generator=g))
    x = wide.to(dtype).cuda()[:, 64:]
    key = (torch.randn(T + spare, 128, generator=g) + 0.5).to(dtype).cuda()
    kv, k = (torch.randint(0, 120, (slots, w), dtype=torch.uint8, generator=g).cuda() for w in (576, 128))
    before = kv.clone(), k.clone()
    ks, kks = torch.full((slots,), 7.0).cuda(), torch.full((slots,), 7.0).cuda()
    freq = freqs(32)
    w = (1 + 0.3 * torch.randn(512, generator=g)).to(dtype).cuda() if norm else None
    wb = tuple((m + 0.3 * torch.randn(128, generator=g)).cuda() for m in (1, 0)) if norm else None
    dsa_cache.append([Rows(x, kv, ks, rope_at=512, norm=w), Rows(key, k, kks, rope_at=0, interleaved=False, norm=wb, eps=1e-5)],
                     table, ctx, ps, cu_new=cu, inv_freq=freq, factor=1.1)
    check(kv, ks, before[0], slot, expected(x[:T], place, freq, None, 512, False, w, factor=1.1))
    check(k, kks, before[1], slot, expected(key[:T], place, freq, None, 0, True, wb, 1e-5, factor=1.1))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_equals_store(dtype):
    """Nothing on the way: store's bytes at the token's slots, scaled and unscaled, and rotate's values between them."""
    say("append equals store", dtype)
    new, old = [7, 1, 90], [100, 0, 63]
    cu, ctx, table, slots, slot, _ = setup(new, old, 64, 3)
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(98, 576, generator=g) * 100).to(dtype).cuda()
    for scaled in (True, False):
        a, b = (torch.zeros(slots, 576, dtype=FP8, device="cuda") for _ in range(2))
        sa, sb = (torch.zeros(slots, device="cuda") if scaled else None for _ in range(2))
        dsa_cache.append(Rows(x, a, sa, fp8_max=448.0 if scaled else 240.0), table, ctx, 64, cu_new=cu)
        dsa_cache.store(b, slot.cuda(), x, 448.0 if scaled else 240.0, scale=sb)
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        assert not scaled or torch.equal(sa, sb)
    if dtype == torch.float32:
        pos = torch.randint(0, 9999, (3, 98), generator=g).to(torch.int32).cuda()
        axes = [i % 3 for i in range(32)]
        dsa_cache.append(Rows(x, a, None, rope_at=64), table, ctx, 64, cu_new=cu, positions=pos, inv_freq=freqs(32), axes=axes)
        y = x.clone()
        dsa_rope.rotate(y[:, None, 64:128], pos, freqs(32), axes=axes, out=y[:, None, 64:128])
        dsa_cache.store(b, slot.cuda(), y)
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("W,at,R,half,n", [(8, None, 0, False, None), (1024, 0, 256, True, 1024), (1024, 504, 8, True, 504),
                                            (640, 496, 32, True, 8), (512, None, 0, False, 512), (576, 512, 32, False, 576),
                                            (128, 64, 32, True, 128), (256, 0, 4, False, 16)])
@pytest.mark.parametrize("kind", ["e4m3", "unscaled", "bf16"])
def test_widths(W, at, R, half, n, kind):
    say("append widths", W, at, R, half, n, kind)
    cu, ctx, table, slots, slot, place = setup([4, 30], [70, 2], 64, W)
    g = torch.Generator().manual_seed(W)
    x = torch.randn(34, W, generator=g).bfloat16().cuda()
    cache = torch.zeros(slots, W, dtype=torch.bfloat16 if kind == "bf16" else FP8, device="cuda")
    scale = torch.full((slots,), 7.0, device="cuda") if kind == "e4m3" else None
    freq = freqs(R) if R else None
    w = (1 + 0.2 * torch.randn(n, generator=g)).cuda() if n else None
    dsa_cache.append(Rows(x, cache, scale, rope_at=at, interleaved=not half, norm=w), table, ctx, 64, cu_new=cu, inv_freq=freq)
    check(cache, scale, torch.zeros_like(cache), slot, expected(x, place, freq, None, at, half, w))


def test_four_kinds_even_batches_and_axes():
    """Four kinds in one call, T / B tokens each, several axes; copies where rows start between 16 bytes; an int64 table."""
    say("append four kinds")
    B, S = 5, 3
    cu, ctx, table, slots, slot, place = setup([S] * B, [64, 1, 0, 200, 63], 64, 9)
    g = torch.Generator().manual_seed(2)
    T = B * S
    pos = torch.randint(0, 1 << 20, (4, T), generator=g).to(torch.int32).cuda()
    axes = [3 - i % 4 for i in range(16)]
    kinds, want = [], []
    for i, W in enumerate((576, 128, 256, 40)):
        x = torch.randn(T, W + 3, generator=g).cuda()[:, 3:] if i % 2 else torch.randn(T, W, generator=g).bfloat16().cuda()
        c, s = torch.zeros(slots, 1, W, dtype=FP8, device="cuda"), torch.full((slots, 1), 7.0, device="cuda")
        kinds.append(Rows(x, c, s, rope_at=8, interleaved=i < 2))
        want.append((c.view(slots, W), s.view(-1), expected(x, pos, freqs(16), axes, 8, i >= 2, None)))
    dsa_cache.append(kinds, table.long(), ctx, 64, positions=pos, inv_freq=freqs(16), axes=axes)
    for c, s, y in want:
        check(c, s, torch.zeros_like(c), slot, y)


def test_rows_of_batches_that_do_not_merge():
    """x [B, S, W] out of [B, S + 1, W], several kinds of one size: each kind's copy lives until the launch."""
    say("append, batches that do not merge")
    cu, ctx, table, slots, slot, place = setup([3] * 5, [40] * 5, 64, 4)
    g = torch.Generator().manual_seed(8)
    x = [torch.randn(5, 4, 128, generator=g).bfloat16().cuda() for _ in range(3)]
    a, b = [[torch.zeros(slots, 128, dtype=torch.bfloat16).cuda() for _ in x] for _ in range(2)]
    dsa_cache.append([Rows(y[:, :3], c) for y, c in zip(x, a)], table, ctx, 64, cu_new=cu)
    dsa_cache.append([Rows(y[:, :3].reshape(15, 128).contiguous(), c) for y, c in zip(x, b)], table, ctx, 64, cu_new=cu)
    for y, c, d in zip(x, a, b):
        assert torch.equal(c, d) and torch.equal(c.cpu()[slot], y[:, :3].reshape(15, 128).cpu())


@pytest.mark.parametrize("stride", [0, 8, 577, 580])
def test_one_row_of_any_stride(stride):
    say("append, a row of stride", stride)
    cu, ctx, table, slots, slot, place = setup([1], [70], 64, 4)
    x = torch.randn(600, generator=torch.Generator().manual_seed(8)).bfloat16().cuda()
    cache = torch.zeros(slots, 576, dtype=torch.bfloat16).cuda()
    dsa_cache.append(Rows(x.as_strided((1, 576), (stride, 1)), cache), table, ctx, 64)
    assert torch.equal(cache.cpu()[slot], x[None, :576].cpu())


def test_no_rotation_beside_positions_and_axes():
    """Rows without rotated columns in a program that has positions of three axes for its other layers."""
    say("append, axes without frequencies")
    cu, ctx, table, slots, slot, place = setup([3, 40], [40, 7], 64, 4)
    x = torch.randn(43, 512, generator=torch.Generator().manual_seed(8)).bfloat16().cuda()
    cache = torch.zeros(slots, 512, dtype=torch.bfloat16).cuda()
    pos = torch.zeros(3, 43, dtype=torch.int32).cuda()
    dsa_cache.append(Rows(x, cache), table, ctx, 64, cu_new=cu, positions=pos, axes=[i % 3 for i in range(32)], factor=1.1)
    assert torch.equal(cache.cpu()[slot], x.cpu())


def test_what_is_not_written():
    """Places outside the table, the null page, pages outside the pool, a length shorter than the new tokens, no sequence."""
    say("append not written")
    ps, pages = 4, 6
    table = torch.tensor([[1, 2], [3, 0], [9, -1], [4, 5]], dtype=torch.int32).cuda()
    ctx = torch.tensor([9, 6, 8, 2], dtype=torch.int32).cuda()  # the first's last token is outside its table
    cu = torch.tensor([1, 4, 8, 10, 15], dtype=torch.int32).cuda()  # row 0 and rows 15, 16 in no sequence
    x = torch.arange(1, 18).float()[:, None].expand(17, 8).contiguous().cuda()
    cache, scale = torch.zeros(pages * ps, 8, dtype=FP8, device="cuda"), torch.zeros(pages * ps, device="cuda")
    dsa_cache.append(Rows(x, cache, scale), table, ctx, ps, cu_new=cu)
    want = torch.zeros(pages * ps)
    # b 0: rows 1 .. 3 at places 6, 7, 8; b 1: rows 4 .. 7 at 2 .. 5 (page 0 from 4 on); b 2: pages 9 and -1; b 3: rows
    # 10 .. 14 at -3 .. 1
    for row, s in ((1, 2 * ps + 2), (2, 2 * ps + 3), (4, 3 * ps + 2), (5, 3 * ps + 3), (13, 4 * ps), (14, 4 * ps + 1)):
        want[s] = row + 1.0
    assert torch.equal((scale * 448).round().cpu(), want) and torch.equal((cache[:, 0].float().cpu() != 0), want != 0)


def test_rows_of_zeros_and_infinities():
    """A row of zeros has the least scale and codes 0, a row with an infinity what store makes of it."""
    say("append zeros")
    cu, ctx, table, slots, slot, _ = setup([3], [0], 64, 1)
    x = torch.zeros(3, 128, device="cuda")
    x[1, 5], x[2, 7] = float("inf"), float("nan")
    a, b = (torch.ones(slots, 128, device="cuda").to(FP8) for _ in range(2))
    sa, sb = torch.zeros(slots, device="cuda"), torch.zeros(slots, device="cuda")
    dsa_cache.append(Rows(x, a, sa), table, ctx, 64, cu_new=cu)
    dsa_cache.store(b, slot.cuda(), x, scale=sb)
    assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)) and torch.equal(sa, sb)
    w = torch.ones(128, device="cuda")
    dsa_cache.append(Rows(x[:1], a, sa, norm=(w, w)), table, ctx[:1] - 2, 64)
    assert (a[slot[0]].float() == 448).all() and sa[slot[0]] == torch.tensor(1.0 / 448)


def test_large_cache():
    """Slots whose rows lie past 2^32 bytes, and rows of x past 2^31 values."""
    say("append large cache")
    pages = 130_000
    cache, scale = torch.zeros(pages * 64, 576, dtype=FP8, device="cuda"), torch.zeros(pages * 64, device="cuda")
    table = torch.tensor([[pages - 1, 3], [7, pages - 2]], dtype=torch.int32).cuda()
    ctx, row = torch.tensor([64, 70], dtype=torch.int32).cuda(), 800_000_000
    big = torch.empty(3 * row + 576, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(big, (4, 576), (row, 1))
    x.copy_(torch.randn(4, 576, generator=torch.Generator().manual_seed(5)))
    dsa_cache.append(Rows(x, cache, scale), table, ctx, 64)
    slot = torch.tensor([(pages - 1) * 64 + 62, (pages - 1) * 64 + 63, (pages - 2) * 64 + 4, (pages - 2) * 64 + 5]).cuda()
    y = x.cpu().double()
    s = y.abs().amax(1) / 448
    assert ((scale[slot].cpu().double() - s).abs() <= 6e-6 * s).all() and int((scale != 0).sum()) == 4
    code = y / s[:, None]
    assert ((cache[slot].cpu().double() - code).abs() <= (code.abs() * 2.0 ** -4).clamp(min=2.0 ** -10) + 448 * 6e-6).all()


def test_streams_and_graph():
    say("append graph")
    cu, ctx, table, slots, slot, _ = setup([2, 2], [70, 5], 64, 4)
    g = torch.Generator().manual_seed(8)
    x = torch.randn(4, 576, generator=g).cuda()
    kv, s = torch.zeros(slots, 576, dtype=FP8, device="cuda"), torch.zeros(slots, device="cuda")
    kv2, s2 = kv.clone(), s.clone()
    call = lambda c, z: dsa_cache.append(Rows(x, c, z, rope_at=512), table, ctx, 64, inv_freq=freqs32)  # noqa: E731
    freqs32 = freqs(32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(kv, s)
    side.synchronize()
    call(kv2, s2)
    assert torch.equal(kv.view(torch.uint8), kv2.view(torch.uint8)) and torch.equal(s, s2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(kv, s)
    for _ in range(3):
        x.copy_(torch.randn(4, 576, generator=g))
        ctx.sub_(1)
        graph.replay()
        torch.cuda.synchronize()
        call(kv2, s2)
        assert torch.equal(kv.view(torch.uint8), kv2.view(torch.uint8)) and torch.equal(s, s2)


def test_refusals():
    cu, ctx, table, slots, _, _ = setup([2, 2], [70, 5], 64, 4)
    x = torch.zeros(4, 128, device="cuda")
    kv, s, f = torch.zeros(slots, 128, dtype=FP8, device="cuda"), torch.zeros(slots, device="cuda"), freqs(32)
    i32 = dict(dtype=torch.int32, device="cuda")

    def call(rows=None, table=table, ctx=ctx, ps=64, **kw):
        dsa_cache.append(Rows(x, kv, s, rope_at=0) if rows is None else rows, table, ctx, ps, **{**dict(cu_new=cu, inv_freq=f), **kw})

    call()
    for kw in (dict(rows=[]), dict(table=table[0]), dict(ctx=ctx[:1]), dict(ps=0), dict(ps=63), dict(cu_new=cu[:2]),
               dict(inv_freq=None), dict(inv_freq=freqs(65)), dict(positions=torch.zeros(3, **i32)),
               dict(positions=torch.zeros(2, 4, **i32)), dict(axes=[1] * 32), dict(rows=Rows(x, kv, s[1:])), dict(rows=Rows(x, kv, s.repeat(2)[::2][:, None])),
               dict(rows=Rows(x[:, :120], kv, s)), dict(rows=Rows(x.half(), kv, s)), dict(rows=Rows(x, kv, s, rope_at=72)),
               dict(rows=[Rows(x, kv, s), Rows(x[:3], kv, s)]), dict(rows=Rows(x, kv, s, norm=f[None])),
               dict(rows=Rows(x, kv, s, norm=torch.ones(136, device="cuda"))), dict(rows=Rows(x, kv, s, norm=(f, f[:8]))),
               dict(rows=Rows(x, kv, s, fp8_max=500.0)), dict(rows=Rows(x, kv.to(torch.bfloat16), s)),
               dict(rows=Rows(x, kv.T.contiguous().T, s)), dict(cu_new=None, rows=Rows(x[:3], kv, s))):
        with pytest.raises(ValueError):
            call(**kw)
    for kw in (dict(rows=Rows(x, kv.half(), None)), dict(rows=[Rows(x, kv, s)] * 5), dict(rows=Rows(x, kv, s, rope_at=4)),
               dict(rows=Rows(x, kv, s, norm=torch.ones(12, device="cuda")))):
        with pytest.raises(NotImplementedError):
            call(**kw)
    with pytest.raises(RuntimeError, match="GPU only"):
        call(rows=Rows(x.cpu(), kv, s))
    call(rows=Rows(x[:0], kv, s), cu_new=torch.zeros(3, **i32))  # no tokens


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fp8_max", [448.0, 240.0])
@pytest.mark.parametrize("W", [128, 576])
def test_infinities_without_a_scale(dtype, fp8_max, W):
    """+infinity is clamped to the largest code, -infinity and NaN to the least: store's bytes, from rows and out of a norm."""
    say("append infinities, unscaled", dtype, fp8_max, W)
    cu, ctx, table, slots, slot, _ = setup([5], [60], 64, 2)
    x = torch.randn(5, W, generator=torch.Generator().manual_seed(W)).to(dtype).cuda()
    x[0, 5], x[1, 7], x[2, 0], x[3, W - 1], x[3, 1] = torch.inf, -torch.inf, torch.nan, torch.inf, -torch.inf
    x[4, 3], x[4, 9] = 3e38, -3e38
    a, b = (torch.ones(slots, W, device="cuda").to(FP8) for _ in range(2))
    dsa_cache.append(Rows(x, a, fp8_max=fp8_max), table, ctx, 64, cu_new=cu)
    dsa_cache.store(b, slot.cuda(), x, fp8_max)
    assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    got = a[slot.cuda()].float()
    assert got[0, 5] == got[3, W - 1] == got[4, 3] == fp8_max and got[1, 7] == got[3, 1] == got[4, 9] == -fp8_max
    w = torch.full((W,), 1e38, device="cuda")  # (normed values of 2 and more overflow)
    y = torch.zeros(1, W, device="cuda")
    y[0, 0], y[0, 1] = 1.0, -1.0
    dsa_cache.append(Rows(y, a, norm=w, fp8_max=fp8_max), table, ctx, 64)
    assert a[slot[4].cuda(), :2].float().tolist() == [fp8_max, -fp8_max] and (a[slot[4].cuda(), 2:].float() == 0).all()
