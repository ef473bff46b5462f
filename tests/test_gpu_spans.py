"""The expanded attention with a range of keys for each query, capped scores and a bias by distance (dsa_expand.attend's first,
last, softcap, slopes) against its definition in float64.

Tolerances, from the arithmetic. A score's error e[t]: the products' fp32 sum, D 2^-24 times the sum of |q k|; with a cap the
tanh's, less than cap 2^-20 (the exponent's argument y = 2 s / cap is off by 2^-23 of itself, which moves tanh by at most y (1 -
tanh^2) 2^-23 < 2^-23; exp2 and the reciprocal are good to 2^-22 each of a term of at most 2; the last product and sum 2^-23:
together below 2^-20); the bias, the running maximum and the factor of log2 e each 2^-23 of the sizes that they are added to (the bias of a tile of 64 keys is
one sum of two, off by 64 of them). A
weight moves by e[t] relative, so an output by sum p e |v| + (sum p e) sum p |v|, and lse by sum p e, to first order (1.01 for
the rest). Weights are rounded to bf16 in their product (2^-8 of sum p |v|), sums are fp32 (2^-20), a bf16 output is rounded
once more (2^-8)."""

import pytest
import torch

from tests._helpers import launched_kernels, say
from tests.test_gpu_expand import cu_of
from trnrt_amd.kernels import dsa_expand

pytestmark = pytest.mark.gpu


def reference(q, k, r, v, lq, lk, scale, causal, first, last, cap, slopes):
    Tq, H, D = q.shape
    out = torch.zeros(Tq, H, 128, dtype=torch.float64, device="cuda")
    lse = torch.full((Tq, H), -1e30, dtype=torch.float64, device="cuda")
    A, PE, PEV = torch.zeros_like(out), torch.zeros_like(lse), torch.zeros_like(out)
    q, k, v = q.double(), k.double(), v.double()
    q0 = k0 = 0
    for nq, nk in zip(lq, lk):
        t = torch.arange(nk, device="cuda")
        place = (nk - nq + torch.arange(nq, device="cuda"))[:, None]
        see = torch.ones(nq, nk, dtype=torch.bool, device="cuda")
        if causal:
            see &= t <= place
        if first is not None:
            see &= t >= first[q0:q0 + nq, None]
        if last is not None:
            see &= t < last[q0:q0 + nq, None]
        for h in range(H):
            key = k[k0:k0 + nk, h]
            if r is not None:
                key = torch.cat([key, r[k0:k0 + nk].double()], 1)
            x = q[q0:q0 + nq, h]
            s = x @ key.T.contiguous() * scale
            e = (x.abs() @ key.abs().T.contiguous()) * scale * D * 2.0 ** -24
            if cap:
                s = cap * torch.tanh(s / cap)
                e = e + cap * 2.0 ** -20
            if slopes is not None:
                s = s - slopes[h].double() * (place - t).abs()
                e = e + slopes[h].double().abs() * ((place - t).abs() + 64) * 2.0 ** -22
            e = e + s.abs() * 2.0 ** -22
            ok = see.any(1)
            if nk == 0 or not ok.any():
                continue
            s = s.masked_fill(~see, -torch.inf)[ok]
            p = torch.softmax(s, -1)
            pe = p * e[ok]
            rows = torch.arange(q0, q0 + nq, device="cuda")[ok]
            value = v[k0:k0 + nk, h].contiguous()
            out[rows, h], A[rows, h] = p @ value, p @ value.abs()
            PE[rows, h], PEV[rows, h] = pe.sum(-1), pe @ value.abs()
            lse[rows, h] = torch.logsumexp(s, -1)
        q0 += nq
        k0 += nk
    return out, lse, A, PE, PEV


def compare(out, lse, refs):
    ref, lref, A, PE, PEV = refs
    tol = A * (2.0 ** -8 + 2.0 ** -20) + 1.01 * (PEV + PE[..., None] * A)
    tol = tol + (2.0 ** -8 * (ref.abs() + tol) if out.dtype == torch.bfloat16 else 0) + 1e-30
    err = (out.double() - ref).abs()
    assert (err <= tol).all(), f"{int((~(err <= tol)).sum())} outputs off, the worst {float((err / tol).max())} of the tolerance"
    assert ((lse == -1e30) == (lref == -1e30)).all()
    ltol = 1.01 * PE + 2.0 ** -20 + 2.0 ** -21 * lref.abs()
    err = (lse.double() - lref).abs()
    assert (err <= ltol).all(), f"lse off by {float((err / ltol).max())} of the tolerance"


def inputs(lq, lk, H, rope, seed, gain=1.5):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(sum(lq), H, 192 if rope else 128, generator=g) * gain).to(torch.bfloat16).cuda()
    k, v = (torch.randn(sum(lk), H, 128, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    r = torch.randn(sum(lk), 64, generator=g).to(torch.bfloat16).cuda() if rope else None
    return q, k, r, v


def masks(kind, lq, lk, seed):
    """(causal, first, last) of a kind, int32 [Tq] on the GPU or None."""
    g = torch.Generator().manual_seed(seed)
    first, last = [], []
    for nq, nk in zip(lq, lk):
        p = nk - nq + torch.arange(nq)
        if kind == "prefix":
            first.append(torch.zeros(nq)), last.append((p + 1).clamp(min=nk * 2 // 5))
        elif kind == "documents":
            at, starts = 0, torch.zeros(max(nk, 1), dtype=torch.int64)
            while at < nk:
                n = int(torch.randint(1, max(2, nk // 3), (1,), generator=g))
                starts[at:at + n] = at
                at += n
            first.append(starts[p.clamp(min=0)] if nk else torch.zeros(nq)), last.append(p + 1)
        elif kind == "window":
            first.append(p - 69), last.append(p + 1)
        elif kind == "images":  # blocks of 100 tokens that see each other both ways, and text before them
            first.append(torch.zeros(nq)), last.append((p // 100 + 1) * 100)
        else:  # any ranges, empty ones and ones past the ends among them
            a = torch.randint(-20, nk + 20, (nq,), generator=g)
            first.append(a), last.append(a + torch.randint(-10, max(nk // 2, 2), (nq,), generator=g))
    first, last = (torch.cat(x).to(torch.int32).cuda() for x in (first, last))
    if kind == "prefix" or kind == "images":
        return False, None, last
    if kind in ("documents", "window"):
        return True, first, None
    return False, first, last


SHAPES = [([1], [1], 1), ([64], [64], 8), ([300, 1, 0, 257], [300, 65, 4, 600], 3), ([700], [1400], 16), ([10, 3, 2], [4, 0, 1], 2),
          ([1] * 40, [77] * 40, 2), ([900], [900], 5)]


@pytest.mark.parametrize("kind", ["prefix", "documents", "window", "images", "any"])
@pytest.mark.parametrize("rope", [True, False])
@pytest.mark.parametrize("lq,lk,H", SHAPES)
def test_ranges(lq, lk, H, rope, kind):
    say("spans", len(lq), sum(lq), sum(lk), H, rope, kind)
    q, k, r, v = inputs(lq, lk, H, rope, H)
    causal, first, last = masks(kind, lq, lk, H)
    out, lse = dsa_expand.attend(q, k, r, v, cu_of(lq).cuda(), cu_of(lk).cuda(), 192 ** -0.5, causal=causal, first=first, last=last)
    compare(out, lse, reference(q, k, r, v, lq, lk, 192 ** -0.5, causal, first, last, 0.0, None))


@pytest.mark.parametrize("cap,bias", [(20.0, False), (0.0, True), (5.0, True), (0.5, False), (50.0, False), (1e6, False)])
@pytest.mark.parametrize("kind", ["causal", "prefix", "any"])
@pytest.mark.parametrize("rope", [True, False])
@pytest.mark.parametrize("lq,lk,H", SHAPES)
def test_scores(lq, lk, H, rope, kind, cap, bias):
    say("spans scores", len(lq), sum(lq), sum(lk), H, rope, kind, cap, bias)
    if cap == 1e6 and (rope or kind != "causal"):
        pytest.skip("a cap that leaves the scores as they are, once")
    q, k, r, v = inputs(lq, lk, H, rope, H + 1, gain=4.0)
    slopes = torch.exp2(-8.0 * torch.arange(1, H + 1) / H).cuda() if bias else None
    if bias and H > 2:
        slopes[0], slopes[1] = 0.0, -0.01  # (none, and one that favours what is far)
    causal, first, last = (True, None, None) if kind == "causal" else masks(kind, lq, lk, H)
    for dtype in (torch.bfloat16, torch.float32):
        out, lse = dsa_expand.attend(q, k, r, v, cu_of(lq).cuda(), cu_of(lk).cuda(), 192 ** -0.5, causal=causal, first=first,
                                     last=last, softcap=cap, slopes=slopes, out_dtype=dtype)
        compare(out, lse, reference(q, k, r, v, lq, lk, 192 ** -0.5, causal, first, last, cap, slopes))


@pytest.mark.parametrize("lq,lk,H", [([20], [9000], 2), ([300], [5000], 4), ([256, 256], [4000, 64], 8)])
def test_splits(lq, lk, H):
    """Few queries over many keys: the keys of a range in splits, of which some hold no key of a query."""
    q, k, r, v = inputs(lq, lk, H, True, 3)
    slopes = torch.full((H,), 0.002).cuda()
    for kind in ("window", "any", "prefix"):
        say("spans splits", lq, lk, H, kind)
        causal, first, last = masks(kind, lq, lk, 5)
        args = (q, k, r, v, cu_of(lq).cuda(), cu_of(lk).cuda(), 192 ** -0.5)
        kw = dict(causal=causal, first=first, last=last, softcap=30.0, slopes=slopes)
        assert "expanded_combine_kernel" in launched_kernels(lambda: dsa_expand.attend(*args, **kw))
        out, lse = dsa_expand.attend(*args, **kw)
        compare(out, lse, reference(q, k, r, v, lq, lk, 192 ** -0.5, causal, first, last, 30.0, slopes))


def test_growing_and_large_scores():
    """Scores that grow along the keys past 2^60 again and again, and ranges that begin where the maximum would be far off."""
    say("spans large scores")
    lq, lk, H = [400], [800], 4
    q, k, r, v = inputs(lq, lk, H, False, 9, gain=1.0)
    k = (k.float() * torch.linspace(0.1, 60, 800, device="cuda")[:, None, None]).to(torch.bfloat16)
    for kind in ("any", "window"):
        causal, first, last = masks(kind, lq, lk, 2)
        out, lse = dsa_expand.attend(q, k, None, v, cu_of(lq).cuda(), cu_of(lk).cuda(), 1.0, causal=causal, first=first, last=last)
        refs = reference(q, k, None, v, lq, lk, 1.0, causal, first, last, 0.0, None)
        compare(out, lse, refs)


def test_whole_ranges_equal_the_causal_form():
    """Ranges that leave everything causal, and nothing changed of the scores: the same bytes as without them."""
    say("spans whole")
    lq, lk, H = [300, 5], [300, 700], 4
    q, k, r, v = inputs(lq, lk, H, True, 4)
    a = dsa_expand.attend(q, k, r, v, cu_of(lq).cuda(), cu_of(lk).cuda(), 0.07)
    b = dsa_expand.attend(q, k, r, v, cu_of(lq).cuda(), cu_of(lk).cuda(), 0.07, first=torch.zeros(305, dtype=torch.int32).cuda())
    c = dsa_expand.attend(q, k, r, v, cu_of(lq).cuda(), cu_of(lk).cuda(), 0.07, last=torch.full((305,), 2 ** 31 - 1).cuda())
    for x in (b, c):
        assert torch.equal(a[0], x[0]) and torch.equal(a[1], x[1])


def test_strange_values_in_hidden_keys():
    """Scores of hidden keys may be NaN or infinite: no query that cannot see them changes where their values are finite; a
    query that sees a NaN score has lse NaN."""
    say("spans hidden NaN")
    lq = lk = [500]
    q, k, r, v = inputs(lq, lk, 2, True, 6)
    first = torch.where(torch.arange(500) < 250, 0, 250).to(torch.int32).cuda()  # two documents
    clean = dsa_expand.attend(q, k, r, v, cu_of(lq).cuda(), cu_of(lk).cuda(), 0.07, first=first)
    k[240, 0, 3], k[245, :, 9], r[247] = torch.nan, torch.inf, -torch.inf
    out, lse = dsa_expand.attend(q, k, r, v, cu_of(lq).cuda(), cu_of(lk).cuda(), 0.07, first=first)
    assert torch.equal(out[250:], clean[0][250:]) and torch.equal(lse[250:], clean[1][250:])
    assert torch.equal(out[:240], clean[0][:240]) and lse[240:250, 0].isnan().all()


@pytest.mark.parametrize("cap,bias", [(50.0, False), (0.5, False), (0.0, True), (50.0, True)])
def test_strange_values_in_hidden_keys_beside_caps_and_distances(cap, bias):
    """The same where scores are changed. A hidden score may decide how its neighbours' caps are computed, within what those are
    off by (cap 2^-20 on both sides, 2^-13 of a weight at most here): the outputs then move by that, by two roundings of each
    weight and by the outputs' own, so by less than 2^-7 + 2^-8 + 2^-12 of the largest value; the lse by 2^-13 and 2^-23 of it."""
    say("spans hidden NaN, scores", cap, bias)
    lq = lk = [500]
    q, k, r, v = inputs(lq, lk, 2, True, 6)
    first = torch.where(torch.arange(500) < 250, 0, 250).to(torch.int32).cuda()
    kw = dict(first=first, softcap=cap, slopes=torch.tensor([0.01, 0.5]).cuda() if bias else None)
    clean = dsa_expand.attend(q, k, r, v, cu_of(lq).cuda(), cu_of(lk).cuda(), 0.07, **kw)
    k[240, 0, 3], k[245, :, 9], r[247] = torch.nan, torch.inf, -torch.inf
    out, lse = dsa_expand.attend(q, k, r, v, cu_of(lq).cuda(), cu_of(lk).cuda(), 0.07, **kw)
    for a, b in ((250, 500), (0, 240)):
        assert ((out - clean[0])[a:b].abs() <= (2.0 ** -7 + 2.0 ** -8 + 2.0 ** -12) * v.abs().max()).all()
        assert ((lse - clean[1])[a:b].abs() <= 2.0 ** -13 + 2.0 ** -23 * lse[a:b].abs()).all()
    assert lse[240:250, 0].isnan().all()


def test_graph():
    say("spans graph")
    lq, lk, H = [40, 100], [3000, 100], 2
    q, k, r, v = inputs(lq, lk, H, True, 8)
    causal, first, last = masks("any", lq, lk, 1)
    cq, ck, slopes = cu_of(lq).cuda(), cu_of(lk).cuda(), torch.full((H,), 0.01).cuda()
    run = lambda: dsa_expand.attend(q, k, r, v, cq, ck, 0.07, causal=causal, first=first, last=last, softcap=9.0, slopes=slopes)  # noqa: E731
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for _ in range(3):
        first.sub_(7), slopes.mul_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        eager = run()
        assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1])


def test_refusals():
    q, k, r, v = inputs([4], [4], 2, True, 1)
    cu, i = cu_of([4]).cuda(), torch.zeros(4, dtype=torch.int32, device="cuda")
    for kw in (dict(first=i[:3]), dict(last=i[None]), dict(slopes=torch.ones(3, device="cuda")), dict(softcap=-1.0),
               dict(softcap=float("inf")), dict(softcap=float("nan"))):
        with pytest.raises(ValueError):
            dsa_expand.attend(q, k, r, v, cu, cu, 0.1, **kw)
    with pytest.raises(RuntimeError, match="GPU only"):
        dsa_expand.attend(q, k, r, v, cu, cu, 0.1, first=i.cpu())


@pytest.mark.parametrize("cached", [0, 3000])
@pytest.mark.parametrize("H,bias", [(2, False), (3, True)])
def test_how_far_a_hidden_value_reaches(cached, H, bias):
    """A value's NaN stays with the queries whose 32 go through its tile of 64 keys: every other one is as it was, bit for bit,
    and those that see it are NaN. Ranges at random places, some empty, in blocks of 32 that lie far apart."""
    say("spans hidden values", cached, H, bias)
    lq, lk = [700, 65], [700 + cached, 65]
    q, k, r, v = inputs(lq, lk, H, True, 7)
    g = torch.Generator().manual_seed(cached + H)
    block = torch.randint(0, lk[0], (22,), generator=g).repeat_interleave(32)[:700]
    first = torch.cat([block + torch.randint(0, 40, (700,), generator=g), torch.zeros(65, dtype=torch.int64)])
    last = first + torch.randint(-3, 200, (765,), generator=g)
    last[700:] = torch.arange(1, 66)
    a, z = first.to(torch.int32).cuda(), last.to(torch.int32).cuda()
    kw = dict(causal=False, first=a, last=z, slopes=torch.full((H,), 0.01).cuda() if bias else None)
    clean = dsa_expand.attend(q, k, r, v, cu_of(lq).cuda(), cu_of(lk).cuda(), 0.07, **kw)
    lo, hi = first[:700].clamp(0, lk[0]), last[:700].clamp(max=lk[0])
    for key in torch.randint(0, lk[0], (6,), generator=g).tolist() + [int(block[40])]:
        w = v.clone()
        w[key] = torch.nan
        out, lse = dsa_expand.attend(q, k, r, w, cu_of(lq).cuda(), cu_of(lk).cuda(), 0.07, **kw)
        reached = torch.zeros(765, dtype=torch.bool)
        for i in range(0, 700, 32):
            some = lo[i:i + 32] < hi[i:i + 32]
            if some.any():
                begin, end = int(lo[i:i + 32][some].min()) // 64 * 64, -(-int(hi[i:i + 32][some].max()) // 64) * 64
                reached[i:min(i + 32, 700)] = begin <= key < end
        assert torch.equal(out.cpu()[~reached], clean[0].cpu()[~reached]) and torch.equal(lse, clean[1])
        sees = torch.zeros(765, dtype=torch.bool)
        sees[:700] = (lo <= key) & (key < hi)
        assert out.cpu()[sees].isnan().all()


@pytest.mark.parametrize("rope", [True, False])
@pytest.mark.parametrize("lq,lk,H", [([700], [1400], 4), ([300, 1, 0, 257], [300, 65, 4, 600], 3), ([20], [9000], 2)])
def test_steep_distances(lq, lk, H, rope):
    """Slopes of up to 16 a token, at which a bias is off by more than 2^-22 of itself: by slope (|p - t| + 64) 2^-22 at most."""
    say("spans steep", len(lq), sum(lq), sum(lk), H, rope)
    q, k, r, v = inputs(lq, lk, H, rope, H + 5)
    for slopes in (torch.linspace(2.0, 16.0, H).cuda(), torch.linspace(-0.5, -4.0, H).cuda()):
        for cap in (0.0, 30.0):
            out, lse = dsa_expand.attend(q, k, r, v, cu_of(lq).cuda(), cu_of(lk).cuda(), 192 ** -0.5, softcap=cap, slopes=slopes,
                                         out_dtype=torch.float32)
            compare(out, lse, reference(q, k, r, v, lq, lk, 192 ** -0.5, True, None, None, cap, slopes))
