"""Rotary positions (trnrt_amd/kernels/dsa_rope.py) against their definition in float64.

Tolerance, from the arithmetic: the reduced angle is rounded once to fp32 in turns (at most 2^-26 of them, 1e-7 radians),
the series for cos and sin are good to 2^-23 (1.2e-7), so these are off by less than 2.3e-7 each, times the factor's roundings;
a result is one product and one fma of them (2^-23 of the sizes): less than 6e-7 factor (|x0| + |x1|) in all, for which 1e-6 is
taken, then the output's rounding (2^-8 or 2^-24 of the value)."""

import pytest
import torch

from tests._helpers import say
from trnrt_amd.kernels import dsa_rope

pytestmark = pytest.mark.gpu


def pairs(x, half):
    R = x.shape[-1] // 2
    return (x[..., :R], x[..., R:]) if half else (x[..., 0::2], x[..., 1::2])


def unpaired(a, b, half):
    return torch.cat([a, b], -1) if half else torch.stack([a, b], -1).flatten(-2)


def reference(x, pos, freq, axes, half, factor=1.0, turn=1.0):
    """x [T, H, 2R] rotated in float64 on the CPU, and the sizes that the tolerance goes by."""
    p = pos.cpu().double().view(-1, x.shape[0])
    which = [0] * freq.shape[0] if axes is None else list(axes)
    phi = turn * torch.stack([p[a] for a in which], 1) * freq.cpu().double()
    c, s = phi.cos()[:, None] * factor, phi.sin()[:, None] * factor
    a, b = pairs(x.cpu().double(), half)
    size = unpaired(a.abs() + b.abs(), a.abs() + b.abs(), half) * abs(factor)
    return unpaired(a * c - b * s, b * c + a * s, half), size


def close(got, ref, size):
    half_step = torch.finfo(got.dtype).eps / 2
    tol = 1e-6 * size + half_step * (ref.abs() + 1e-6 * size)
    err = (got.cpu().double() - ref).abs()
    assert (err <= tol).all(), f"off by {float((err / tol.clamp(min=1e-300)).max())} of the tolerance"


def freqs(R):
    return (10000.0 ** (-torch.arange(R, dtype=torch.float64) / R)).float().cuda()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,H,R,n,pad", [
    (1, 1, 32, 1, 0), (8, 64, 32, 1, 512), (3, 5, 1, 1, 0), (7, 3, 20, 3, 4), (1000, 16, 32, 3, 128), (33, 2, 256, 4, 0),
    (2, 128, 64, 2, 0), (5, 7, 13, 2, 3), (2500, 1, 32, 1, 64), (300, 65, 24, 3, 1), (20000, 1, 4, 1, 8),
])
def test_rotate(T, H, R, n, pad, dtype, half):
    """New outputs, outputs into a view of wider rows, and in place; what lies beside is left as it was."""
    say("rotate", T, H, R, n, pad, dtype, half)
    g = torch.Generator().manual_seed(T * 7 + R)
    wide = torch.randn(T, H, pad + 2 * R, generator=g).to(dtype).cuda()
    x = wide[..., pad:]
    pos = torch.randint(0, 1 << 20, (n, T) if n > 1 else (T,), generator=g).to(torch.int32).cuda()
    axes = [i * 5 % n for i in range(R)] if n > 1 else None
    freq = freqs(R)
    ref, size = reference(x, pos, freq, axes, half, 1.25)
    y = dsa_rope.rotate(x, pos, freq, axes=axes, interleaved=not half, factor=1.25)
    close(y, ref, size)
    into = torch.full((T, H, 2 * R + 3), 7.0, dtype=dtype, device="cuda")
    z = dsa_rope.rotate(x, pos, freq, axes=axes, interleaved=not half, factor=1.25, out=into[..., :2 * R])
    assert torch.equal(z, y) and (into[..., 2 * R:] == 7).all()
    beside = wide[..., :pad].clone()
    dsa_rope.rotate(x, pos, freq, axes=axes, interleaved=not half, factor=1.25, out=x)
    assert torch.equal(x, y) and torch.equal(wide[..., :pad], beside)


@pytest.mark.parametrize("half", [False, True])
def test_far_and_negative_positions(half):
    say("rotate far", half)
    pos = torch.tensor([0, 1, -1, 123456789, -2147483648, 2147483647, 1 << 24, (1 << 24) + 1], dtype=torch.int32).cuda()
    x = torch.randn(8, 4, 64, generator=torch.Generator().manual_seed(1)).cuda()
    ref, size = reference(x, pos, freqs(32), None, half)
    close(dsa_rope.rotate(x, pos, freqs(32), interleaved=not half), ref, size)


def test_other_layouts():
    """Rows without heads, strided columns, transposed heads, int64 positions, broadcast heads, no tokens."""
    say("rotate layouts")
    g = torch.Generator().manual_seed(3)
    x = torch.randn(64, 6, 50, generator=g).cuda()
    pos = torch.randint(0, 5000, (50,), generator=g).cuda()
    freq = freqs(32)
    rows = x.permute(2, 1, 0)  # [50, 6, 64], columns 300 apart
    ref, size = reference(rows, pos, freq, None, False)
    close(dsa_rope.rotate(rows, pos, freq), ref, size)
    heads = torch.randn(6, 50, 64, generator=g).cuda().transpose(0, 1)
    out = torch.empty(6, 50, 64, device="cuda").transpose(0, 1)
    ref, size = reference(heads, pos, freq, None, False)
    close(dsa_rope.rotate(heads, pos, freq, out=out), ref, size)
    flat = torch.randn(50, 64, generator=g).cuda()
    ref, size = reference(flat[:, None], pos, freq, None, True)
    close(dsa_rope.rotate(flat, pos, freq, interleaved=False)[:, None], ref, size)
    wide = flat[:, None].expand(50, 9, 64)
    ref, size = reference(wide, pos, freq, None, False)
    close(dsa_rope.rotate(wide, pos, freq), ref, size)
    assert dsa_rope.rotate(flat[:0], pos[:0], freq).shape == (0, 64)


@pytest.mark.parametrize("half", [False, True])
def test_inverse_is_the_gradient(half):
    """rotate is linear: <g, rotate(x)> = <rotate(g, inverse), x>, the inverse undoes it, and differences in x of one entry
    give the gradient's entry. (Each inner product of 1,920 terms is of fp32 results off by less than 1e-6 of their sizes.)"""
    say("rotate inverse", half)
    gen = torch.Generator().manual_seed(5)
    x, g = (torch.randn(10, 3, 64, generator=gen).cuda() for _ in range(2))
    pos = torch.randint(0, 9000, (3, 10), generator=gen).to(torch.int32).cuda()
    kw = dict(axes=[i % 3 for i in range(32)], interleaved=not half)
    y = dsa_rope.rotate(x, pos, freqs(32), factor=0.7, **kw)
    gx = dsa_rope.rotate(g, pos, freqs(32), factor=0.7, inverse=True, **kw)
    a, b = (g.double() * y.double()).sum(), (gx.double() * x.double()).sum()
    assert abs(a - b) <= 2e-6 * 2 * (g.double().abs().sum() * x.double().abs().max())
    back = dsa_rope.rotate(dsa_rope.rotate(x, pos, freqs(32), **kw), pos, freqs(32), inverse=True, **kw)
    size = reference(x, pos, freqs(32), kw["axes"], half)[1]
    big = unpaired(*[pairs(size, half)[0] * 2] * 2, half)  # (of the rotated values)
    assert ((back.cpu().double() - x.cpu().double()).abs() <= 2e-6 * big + 1e-12).all()
    for t, h, c in ((0, 0, 0), (9, 2, 63), (4, 1, 31), (3, 0, 32)):
        d = torch.zeros_like(x)
        d[t, h, c] = 1.0  # (linear: the difference is exact)
        change = (g.double() * dsa_rope.rotate(d, pos, freqs(32), factor=0.7, **kw).double()).sum()
        assert abs(change - gx[t, h, c].double()) <= 4e-6 * g.double().abs().max()


def test_rows_far_apart():
    """Rows whose offsets pass 2^31 values and 2^32 bytes, read and written."""
    say("rotate far apart")
    row = 1_200_000_000
    big = torch.empty(2 * row + 300, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(big, (3, 2, 64), (row, 64, 1))
    x.copy_(torch.randn(3, 2, 64, generator=torch.Generator().manual_seed(4)))
    pos = torch.tensor([5, 70, 900], dtype=torch.int32).cuda()
    ref, size = reference(x, pos, freqs(32), None, False)
    close(dsa_rope.rotate(x, pos, freqs(32)), ref, size)
    dsa_rope.rotate(x, pos, freqs(32), out=x)
    close(x, ref, size)


def test_streams_and_graph():
    """On a side stream, and captured and replayed with other inputs between eager calls."""
    say("rotate graph")
    gen = torch.Generator().manual_seed(6)
    x, pos = torch.randn(20, 8, 64, generator=gen).cuda(), torch.arange(20, dtype=torch.int32).cuda()
    freq = freqs(32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = dsa_rope.rotate(x, pos, freq)
    side.synchronize()
    assert torch.equal(y, dsa_rope.rotate(x, pos, freq))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z = dsa_rope.rotate(x, pos, freq)
    for k in range(3):
        x.copy_(torch.randn(20, 8, 64, generator=gen))
        pos.add_(1000 * k)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(z, dsa_rope.rotate(x, pos, freq))


def test_refusals():
    x, pos, freq = torch.zeros(4, 2, 64, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda"), freqs(32)
    for kw in (dict(x=x.half()), dict(x=x[..., :62]), dict(x=x[None]), dict(positions=pos[:3]), dict(positions=pos.float()),
               dict(inv_freq=freq.double()), dict(inv_freq=freq[::2]), dict(axes=[0] * 31), dict(axes=[1] * 32),
               dict(positions=pos.expand(3, 4)), dict(out=x[:3]), dict(out=x.bfloat16()),
               dict(out=torch.zeros(1, 2, 64, device="cuda").expand(4, 2, 64)),
               dict(out=torch.zeros(4, 2, 128, device="cuda")[..., ::2])):
        with pytest.raises(ValueError):
            dsa_rope.rotate(**{**dict(x=x, positions=pos, inv_freq=freq), **kw})
    with pytest.raises(NotImplementedError):
        dsa_rope.rotate(torch.zeros(1, 600, device="cuda"), pos[:1], freqs(300))
    with pytest.raises(RuntimeError, match="GPU only"):
        dsa_rope.rotate(x, pos.cpu(), freq)


def test_outputs_whose_rows_overlap_are_refused():
    """Rows 32 of 64 values apart, heads that run into the next token's; rows between each other's are taken."""
    say("rotate overlap")
    x, pos, freq = torch.randn(6, 3, 64, device="cuda"), torch.arange(6, dtype=torch.int32, device="cuda"), freqs(32)
    big = torch.zeros(4096, device="cuda")
    for strides in ((192, 32, 1), (128, 64, 1), (96, 576, 1), (0, 64, 1)):
        if strides == (96, 576, 1):  # (apart)
            dsa_rope.rotate(x, pos, freq, out=big.as_strided((6, 3, 64), strides))
            assert torch.equal(big.as_strided((6, 3, 64), strides), dsa_rope.rotate(x, pos, freq))
            continue
        with pytest.raises(ValueError, match="no row over another"):
            dsa_rope.rotate(x, pos, freq, out=big.as_strided((6, 3, 64), strides))
    with pytest.raises(ValueError, match="no row over another"):
        dsa_rope.rotate(x[:, 0], pos, freq, out=big.as_strided((6, 64), (60, 1)))
    y = big.as_strided((1, 3, 64), (1, 64, 1))  # (one token: its stride says nothing)
    dsa_rope.rotate(x[:1], pos[:1], freq, out=y)
    assert torch.equal(y, dsa_rope.rotate(x[:1], pos[:1], freq))
