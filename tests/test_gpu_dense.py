"""Absorbed latent attention without a selection (trnrt_amd/kernels/dsa_dense.py) against the definition in float64, with
the caches' unused slots full of NaN.

Tolerances, from the arithmetic: the kernel rounds each softmax weight (times its token's scale) to bf16, off by at most
2^-8 of it, so an output by at most 2^-8 of A = sum_t p[t] |V[t]|; a bf16 output is rounded once more, 2^-8 of its size;
scores are fp32 sums of D products, off by less than D 2^-24 sum |q K| (E below, their largest over the tokens), which moves
weights by that much relative, and the log-sum-exp by that much, plus the roundings of the exponential and the logarithm
(a few 2^-23 each, and 2^-23 of the maximum)."""

import pytest
import torch

from tests._helpers import say
from trnrt_amd.kernels import dsa_decode, dsa_dense

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


def make(lens, S, H, D, ps, seed, q_gain=1.0, scaled=True, spread=0.5):
    """CPU inputs: pages in random order, every slot that holds no token NaN."""
    g = torch.Generator().manual_seed(seed)
    B = len(lens)
    npg = [-(-n // ps) for n in lens]
    mp = max(max(npg), 1) + 1
    pages = 1 + sum(npg)
    table = torch.full((B, mp), -7, dtype=torch.int32)  # entries past a row's pages are not read
    perm = (torch.randperm(pages - 1, generator=g) + 1).to(torch.int32)
    kv = torch.full((pages * ps, D), 0x7F, dtype=torch.uint8)
    sc = torch.full((pages * ps,), float("nan"))
    at = 0
    for b, n in enumerate(lens):
        table[b, :npg[b]] = perm[at:at + npg[b]]
        at += npg[b]
        t = torch.arange(n)
        slot = table[b][t // ps].long() * ps + t % ps
        x = torch.randn(n, D, generator=g) * torch.exp(spread * torch.randn(n, 1, generator=g))
        s = x.abs().amax(-1).clamp(min=1e-30) / 448 if n else torch.ones(0)
        kv[slot] = (x / s[:, None]).clamp(-448, 448).to(FP8).view(torch.uint8)
        sc[slot] = s
    q = (torch.randn(B, S, H, D, generator=g) * q_gain).to(torch.bfloat16)
    return q, kv, sc if scaled else None, table, torch.tensor(lens, dtype=torch.int32)


def reference(q, kv, sc, table, lens, ps, scale):
    """(out, lse, A, E) in float64 on the GPU's float64 units."""
    B, S, H, D = q.shape
    dev = "cuda"
    out = torch.zeros(B, S, H, 512, dtype=torch.float64)
    lse = torch.full((B, S, H), -1e30, dtype=torch.float64)
    A, E = torch.zeros_like(out), torch.zeros(B, S, H, dtype=torch.float64)
    for b in range(B):
        n = min(max(int(lens[b]), 0), table.shape[1] * ps)
        t = torch.arange(n)
        slot = table[b][t // ps].long() * ps + t % ps
        K = kv[slot].view(FP8).to(torch.float64).to(dev)
        if sc is not None:
            K = K * sc[slot].to(torch.float64).to(dev)[:, None]
        for i in range(S):
            m = n - S + i + 1
            if m <= 0:
                continue
            x = q[b, i].to(torch.float64).to(dev)
            s = x @ K[:m].T.contiguous() * scale
            w = torch.softmax(s, -1)
            out[b, i] = (w @ K[:m, :512].contiguous()).cpu()
            A[b, i] = (w @ K[:m, :512].abs().contiguous()).cpu()
            lse[b, i] = torch.logsumexp(s, -1).cpu()
            E[b, i] = (x.abs() @ K[:m].abs().T.contiguous()).amax(-1).cpu() * scale * D * 2.0 ** -24
    return out, lse, A, E


def check(inp, ps, scale=192 ** -0.5, out_dtype=torch.bfloat16, squeeze=False):
    q, kv, sc, table, lens = inp
    ref, lref, A, E = reference(q, kv, sc, table, lens, ps, scale)
    g = [None if x is None else x.cuda() for x in (q[:, 0] if squeeze else q, kv, sc, table, lens)]
    out, lse = dsa_dense.attend(*g, ps, scale, out_dtype=out_dtype)
    assert out.dtype == out_dtype
    out, lse = out.double().cpu().view(ref.shape), lse.double().cpu().view(lref.shape)
    rel = 2.0 ** -8 + 2 * E[..., None] + 2.0 ** -20
    tol = A * rel + (2.0 ** -8 * (ref.abs() + A * rel) if out_dtype == torch.bfloat16 else 0) + 1e-30
    bad = ~((out - ref).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} outputs off, the worst {float(((out - ref).abs() / tol).max())} of the tolerance"
    ltol = E + 2.0 ** -21 + 2.0 ** -22 * lref.abs()
    bad = ~((lse - lref).abs() <= ltol)
    assert not bad.any(), f"lse off by {float(((lse - lref).abs() / ltol).max())} of the tolerance"
    return out, lse


@pytest.mark.parametrize("D", [576, 512])
@pytest.mark.parametrize("H,S", [(16, 1), (64, 1), (1, 1), (24, 1), (128, 1), (16, 4), (40, 3), (8, 7)])
def test_heads_and_new_tokens(H, S, D):
    say("dense", H, S, D)
    check(make([300, 1, 64, 65, 63, 0, 129, 777], S, H, D, 64, seed=H + S), 64)


@pytest.mark.parametrize("ps", [1, 16, 33, 48, 128, 1000])
def test_page_sizes(ps):
    say("dense pages of", ps)
    check(make([500, 31, 2], 2, 20, 576, ps, seed=ps), ps)


def test_one_new_token_without_its_dimension():
    say("dense [B, H, D]")
    check(make([100, 200], 1, 32, 512, 64, seed=1), 64, squeeze=True)


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scaled", [True, False])
def test_unscaled_cache_and_fp32_outputs(scaled, out_dtype):
    say("dense scaled", scaled, out_dtype)
    inp = make([700, 90], 1, 64, 576, 64, seed=3, scaled=scaled, q_gain=1.0 if scaled else 0.01)
    check(inp, 64, out_dtype=out_dtype)


@pytest.mark.parametrize("gain", [0.0, 8.0, 40.0])
def test_flat_and_steep_softmax(gain):
    """All weights alike; maxima that move far between chunks; rows whose scores all lie far below zero."""
    say("dense gain", gain)
    inp = make([1500, 640, 70], 1, 48, 576, 64, seed=5, q_gain=gain)
    check(inp, 64)
    q, kv, sc, table, lens = inp
    kv[:] = torch.where(kv == 0x7F, kv, 0x38)  # every value 1: scores - |q| scale
    check((-q.abs(), kv, sc, table, lens), 64)


def test_scales_far_apart():
    """Token scales from 2^-40 to 2^6 within a chunk, zeros among them; where every other score lies far below zero, the
    tokens of scale 0 have the largest softmax weights and add nothing."""
    say("dense scales far apart")
    q, kv, sc, table, lens = make([900, 130, 64], 1, 24, 576, 64, seed=6, spread=0.0)
    live = sc == sc
    g = torch.Generator().manual_seed(7)
    e = torch.randint(-40, 7, sc.shape, generator=g).float()
    check((q, kv, torch.where(live, torch.exp2(e) / 448, sc), table, lens), 64)
    check((q, kv, torch.where(live & (torch.arange(sc.numel()) % 3 > 0), torch.exp2(e) / 448, torch.where(live, 0.0, sc)), table, lens), 64)
    low = torch.where(kv == 0x7F, kv, 0x38)  # every value 1
    zero_late = torch.where(live, torch.where(torch.arange(sc.numel()) % 5 > 0, 1.0, 0.0), sc)
    check((-q.abs() * 8, low, zero_late, table, lens), 64)  # scores near -2,500, and 0


def test_one_token_outweighs_the_rest():
    """A first token that only its rope columns score, with 2^22 times the weight of each other and no value: the outputs
    are the others', to their own size."""
    say("dense one token outweighs the rest")
    q, kv, sc, table, lens = make([3000, 500], 1, 32, 576, 64, seed=8, spread=0.0)
    scale = 192 ** -0.5
    q[..., :512] *= 0.05
    q[..., 512:] = 1.0
    for b in range(2):
        n = int(lens[b])
        t = torch.arange(n)
        slot = table[b][t // 64].long() * 64 + t % 64
        kv[slot, 512:] = 0  # (+0)
        first = table[b][0].long() * 64
        kv[first, :512], kv[first, 512:], sc[first] = 0, 0x38, 22 * 0.6931471805599453 / (64 * scale)
    check((q, kv, sc, table, lens), 64, scale=scale)
    check((q, kv, sc, table, lens), 64, scale=scale, out_dtype=torch.float32)


@pytest.mark.parametrize("H", [16, 64])
def test_long_and_ragged(H):
    """Row tiles shared by many workgroups, several tiles in one workgroup, sequences without tokens between."""
    say("dense long", H)
    check(make([40000, 0, 3, 0, 0, 9000, 128, 20001], 1, H, 576, 64, seed=H), 64)


@pytest.mark.parametrize("H,S,lens", [(64, 11, [700, 40, 0, 130]), (128, 20, [300, 90]), (128, 70, [200]), (16, 150, [1000, 149])])
def test_many_row_tiles(H, S, lens):
    """More row tiles than an XCD has CUs, and numbers of them that do not divide its CUs; appends longer than their
    sequence's earlier tokens."""
    say("dense row tiles", H, S, lens)
    check(make(lens, S, H, 576 if S < 50 else 512, 64, seed=S), 64)


def test_many_short_sequences():
    say("dense 1,100 sequences")
    g = torch.Generator().manual_seed(0)
    lens = torch.randint(0, 130, (1100,), generator=g).tolist()
    check(make(lens, 1, 16, 512, 16, seed=2), 16)


def test_padded_batch():
    """Thousands of sequences without tokens around the few that have some."""
    say("dense padded batch")
    lens = [700] + [0] * 1500 + [65, 0, 900] + [0] * 511 + [3] + [0] * 512 + [64, 1000] + [0] * 300
    check(make(lens, 1, 16, 576, 64, seed=13), 64)


def test_all_empty_and_no_sequence():
    say("dense empty")
    out, lse = check(make([0, 0, 0], 2, 16, 576, 64, seed=2), 64)
    assert not out.any() and (lse.float() == -1e30).all()  # (as fp32, which has no -1e30 exactly)
    q, kv, sc, table, lens = (x.cuda() for x in make([4], 1, 16, 576, 64, seed=2))
    o, l = dsa_dense.attend(q[:0], kv, sc, table[:0], lens[:0], 64, 0.1)
    assert o.shape == (0, 1, 16, 512) and l.shape == (0, 1, 16)


def test_lengths_past_the_table_and_foreign_pages():
    """A length past the table is the table's; a page id outside the cache reads the null page."""
    say("dense clamps")
    q, kv, sc, table, lens = make([200, 128], 1, 16, 576, 64, seed=9)
    table[0, 4], lens[0] = 0, 10 ** 9  # five pages, the last the null page
    table[1, 1] = 10 ** 6
    kv[:64], sc[:64] = 0x30, 0.5
    want = table.clone()
    want[1, 1] = 0
    kv[table[0, 3].long() * 64 + 8:table[0, 3].long() * 64 + 64] = 0x28
    sc[table[0, 3].long() * 64 + 8:table[0, 3].long() * 64 + 64] = 0.25
    ref, lref, A, _ = reference(q, kv, sc, want, lens, 64, 0.07)
    out, lse = dsa_dense.attend(q.cuda(), kv.cuda(), sc.cuda(), table.cuda(), lens.cuda(), 64, 0.07)
    assert ((out.double().cpu() - ref).abs() <= 2.0 ** -7 * A + 1e-6).all()
    assert (lse.double().cpu() - lref).abs().max() < 1e-4


def test_selecting_every_token_agrees():
    """dsa_decode.attend_tokens over all positions is the same attention: both within two weight roundings of it."""
    say("dense against the selected form")
    q, kv, sc, table, lens = (x.cuda() for x in make([1000, 512, 77], 1, 64, 576, 64, seed=4))
    idx = torch.arange(1000, dtype=torch.int32, device="cuda").repeat(3, 1)
    out, lse = dsa_dense.attend(q[:, 0], kv, sc, table, lens, 64, 192 ** -0.5)
    o2, l2 = dsa_decode.attend_tokens(q[:, 0].contiguous(), kv, sc, idx, lens, table, 64, 192 ** -0.5)
    torch.testing.assert_close(out.float(), o2.float(), atol=2e-2, rtol=2e-2)
    torch.testing.assert_close(lse, l2, atol=1e-5, rtol=1e-6)


def test_graph_replays_and_another_stream():
    say("dense in a graph, on another stream")
    inps = [make([900, 64, 1300], 2, 16, 576, 64, seed=30 + i) for i in range(3)]
    q, kv, sc, table, lens = (x.cuda() for x in inps[0])
    ws = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        eager = dsa_dense.attend(q, kv, sc, table, lens, 64, 0.07, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = dsa_dense.attend(q, kv, sc, table, lens, 64, 0.07, workspace=ws)
    for i in (0, 1, 2):
        for a, b in zip((q, kv, sc, table, lens), inps[i]):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        want = dsa_dense.attend(q, kv, sc, table, lens, 64, 0.07)
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
        if i == 0:
            assert torch.equal(out, eager[0])


def test_views_at_odd_places():
    """Queries that start at an odd element are copied; a cache that does is refused."""
    say("dense odd places")
    q, kv, sc, table, lens = (x.cuda() for x in make([100, 5], 1, 16, 576, 64, seed=12))
    want = dsa_dense.attend(q, kv, sc, table, lens, 64, 0.1)
    flat = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")
    odd = flat[1:].view(q.shape)
    odd.copy_(q)
    got = dsa_dense.attend(odd, kv, sc, table, lens, 64, 0.1)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    cache = torch.empty(kv.numel() + 8, dtype=torch.uint8, device="cuda")[8:].view(kv.shape)
    cache.copy_(kv)
    with pytest.raises(ValueError):
        dsa_dense.attend(q, cache, sc, table, lens, 64, 0.1)


def test_refusals():
    q, kv, sc, table, lens = (x.cuda() for x in make([100, 5], 1, 16, 576, 64, seed=0))
    ok = dict(q=q, kv_cache=kv, kv_scale=sc, table=table, ctx_len=lens, page_size=64, scale=0.1)
    for bad in (dict(q=q[..., :500]), dict(q=q[0, 0]), dict(page_size=60), dict(page_size=0), dict(kv_scale=sc[:-1]),
                dict(table=table[:1]), dict(table=table[0]), dict(ctx_len=lens[:1]), dict(kv_cache=kv.float()),
                dict(kv_cache=kv.t()), dict(kv_cache=kv.view(-1, 512), kv_scale=None), dict(out=torch.empty(2, 1, 16, 500, device="cuda")),
                dict(out=torch.empty(2, 1, 16, 512, dtype=torch.float16, device="cuda")),
                dict(workspace=torch.empty(64, dtype=torch.uint8, device="cuda")),
                dict(workspace=torch.empty(1, dtype=torch.uint8, device="cuda").expand(1 << 30))):
        with pytest.raises(ValueError):
            dsa_dense.attend(**{**ok, **bad})
    with pytest.raises(RuntimeError, match="GPU only"):
        dsa_dense.attend(**{**ok, "q": q.cpu()})


@pytest.mark.parametrize("H,S,D", [(64, 11, 576), (64, 13, 512), (48, 14, 576), (96, 7, 512)])
def test_workgroups_without_a_tile(H, S, D):
    """Row tiles that are no multiple of a team's, shares of several units that begin in a sequence's last set and go on
    behind sequences without tokens: some workgroups' first step is the search for the next sequence."""
    say("dense workgroups without a tile", H, S, D)
    check(make([130, 0, 0, 70, 0, 200] * 14, S, H, D, 64, seed=H + S), 64)


@pytest.mark.parametrize("H", [8, 16, 64])
@pytest.mark.parametrize("n", [200, 60000])
def test_nan_reaches_the_lse(H, n):
    """A token's NaN (in its row or its scale) shows in the lse of the queries that see it, not as the value of a query that
    sees nothing, whether a row tile is one workgroup's or joined; the other sequences and queries have theirs."""
    say("dense NaN", H, n)
    q, kv, sc, table, lens = make([n, 3, 130, 0], 3, H, 576, 64, seed=H)
    ref, lref, _, E = reference(q, kv, sc, table, lens, 64, 0.05)
    kv[table[0, 1].long() * 64 + 5, 7] = 0x7F  # token 69 of the first sequence, which every query sees
    sc[table[2, 2].long() * 64 + 1] = float("nan")  # the last token of the third, which only its last query sees
    out, lse = dsa_dense.attend(*(x.cuda() for x in (q, kv, sc, table, lens)), 64, 0.05)
    out, lse = out.double().cpu(), lse.double().cpu()
    assert out[0].isnan().all() and lse[0].isnan().all()
    assert out[2].isnan().all() and lse[2, 2].isnan().all()
    for b, i in ((1, 0), (1, 1), (1, 2), (2, 0), (2, 1), (3, 0), (3, 2)):
        assert ((lse[b, i] - lref[b, i]).abs() <= E[b, i] + 2.0 ** -21 + 2.0 ** -22 * lref[b, i].abs()).all()
    assert not out[3].any() and (lse[3].float() == -1e30).all()


def test_two_threads_on_one_stream():
    """Calls of two host threads on one stream, whose launches come between each other's: each joins its own partials."""
    say("dense, two threads")
    import threading

    ins = [tuple(x.cuda() for x in make([5000 + 900 * i, 400], 1, 16, 576, 64, seed=40 + i)) for i in range(2)]
    want = [dsa_dense.attend(*x, 64, 0.05) for x in ins]
    torch.cuda.synchronize()
    got = [[], []]

    def run(i):
        for _ in range(200):
            got[i].append(dsa_dense.attend(*ins[i], 64, 0.05))

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(2):
        assert len(got[i]) == 200 and all(torch.equal(o, want[i][0]) and torch.equal(l, want[i][1]) for o, l in got[i])


def exact_scores(lens, S, H, D, seed, step):
    """Inputs whose scores are exact in fp32 in any order (values in halves and scales in powers of two), and with `step` higher
    by 69 of base 2 from token 128 on, past what the running maximum lets pass."""
    q, kv, sc, table, lens = make(lens, S, H, D, 64, seed)
    g = torch.Generator().manual_seed(seed + 1)
    live = sc == sc
    x = torch.tensor([-1.0, -0.5, 0.0, 0.5, 1.0, 1.5])[torch.randint(0, 6, kv.shape, generator=g)]
    for b, n in enumerate(lens.tolist()):
        t = torch.arange(n)
        slot = table[b][t // 64].long() * 64 + t % 64
        x[slot, 0] = torch.where(t >= 128, 96.0, 0.0) if step else 0.0
    kv = torch.where(live[:, None], x.to(FP8).view(torch.uint8), kv)
    sc = torch.where(live, torch.exp2(torch.randint(-1, 2, sc.shape, generator=g).float()) if not step else torch.ones_like(sc), sc)
    q = (torch.randint(-8, 9, q.shape, generator=g) / 8).to(torch.bfloat16)
    q[..., 0] = 8.0
    return q, kv, sc, table, lens


@pytest.mark.parametrize("step", [False, True])
@pytest.mark.parametrize("H,S,D,lens", [(16, 1, 576, [200, 1, 64, 300]), (32, 1, 512, [130, 300]), (8, 3, 576, [65, 280]),
                                        (16, 2, 512, [300] * 200), (16, 1, 576, [300, 290, 0] * 80)])
def test_two_terms_of_the_weights(H, S, D, lens, step):
    """Up to 32 rows a softmax weight is two bf16 terms, off by 2^-8 of 2^-8 of it. With exact scores s (base 2, at most M in size)
    the exponent's error is that of the factor's, the difference's and the maximum's roundings, 4 M 2^-24 at most, the
    exponential's 2^-23 of its value; the sums of n tokens in two terms are off by less than 3 n 2^-24 of A. One term alone
    would not pass."""
    say("dense two terms", H, S, D, len(lens), step)
    scale = 1 / 16
    q, kv, sc, table, lens = exact_scores(lens, S, H, D, 3, step)
    out = dsa_dense.attend(q.cuda(), kv.cuda(), sc.cuda(), table.cuda(), lens.cuda(), 64, scale, lse=False,
                           out_dtype=torch.float32).double()
    one_term = 0
    for b, n in enumerate(lens.tolist()):
        t = torch.arange(n)
        slot = table[b][t // 64].long() * 64 + t % 64
        K = (kv[slot].view(FP8).double() * sc[slot].double()[:, None]).cuda()
        sigma = sc[slot].double().cuda()
        for i in range(S):
            m = n - S + i + 1
            if m <= 0:
                assert not out[b, i].any()
                continue
            s = q[b, i].double().cuda() @ K[:m].T.contiguous() * scale
            p = torch.softmax(s, -1)
            V = K[:m, :512].contiguous()
            ref, A = p @ V, p @ V.abs()
            M = float(s.abs().max()) * 1.4426950408889634
            tol = A * (2.0 ** -16 + 2 * (4 * M * 2.0 ** -24 * 0.6931471805599453 + 2.0 ** -23) + 3 * n * 2.0 ** -24) + 1e-30
            err = (out[b, i] - ref).abs()
            assert (err <= tol).all(), f"sequence {b}: the worst {float((err / tol).max())} of the tolerance"
            w = torch.exp(s - s.amax(-1, keepdim=True)) * sigma[:m]  # the oracle with one bf16 term
            planted = (w.float().bfloat16().double() / sigma[:m] / torch.exp(s - s.amax(-1, keepdim=True)).sum(-1, keepdim=True)) @ V
            one_term += int(((planted - ref).abs() > tol).sum())
    assert one_term > 0


@pytest.mark.parametrize("H,S,D,lens", [(64, 1, 576, [1, 2, 0, 5, 64, 33] * 4), (128, 1, 512, [3, 1, 17]), (40, 2, 576, [64, 1, 9]),
                                        (128, 4, 576, [1, 6, 50]), (64, 1, 576, [300, 64, 1000, 129])])
@pytest.mark.parametrize("gain", [0.25, 1.0])
def test_the_heaviest_weight_is_exact(H, S, D, lens, gain):
    """Past 32 rows a softmax weight times its token's scale is one bf16 term, off by 2^-8 of it; in a stretch of one chunk the
    token with the largest score plus its scale's log2 without the whole part has a power of two there, which is off by
    nothing. With exact products in the scores s (base 2, at most M in size; values in halves, any scales), the exponent's error
    is 4 M 2^-24 at most, with the logarithm's 2^-21, the exponential's 2^-23; sums of n tokens are off by n 2^-24 of A."""
    say("dense heaviest weight", H, S, D, lens, gain)
    q, kv, sc, table, lens_t = exact_scores(lens, S, H, D, 5, False)
    g = torch.Generator().manual_seed(6)
    sc = torch.where(sc == sc, torch.exp2(torch.rand(sc.shape, generator=g) - 7), sc)
    q = (q.float() * gain * 64).to(torch.bfloat16)  # (an exact factor)
    scale = 1 / 32
    out = dsa_dense.attend(q.cuda(), kv.cuda(), sc.cuda(), table.cuda(), lens_t.cuda(), 64, scale, lse=False,
                           out_dtype=torch.float32).double()
    for b, n in enumerate(lens):
        t = torch.arange(n)
        slot = table[b][t // 64].long() * 64 + t % 64
        sigma = sc[slot].double().cuda()
        K = kv[slot].view(FP8).double().cuda() * sigma[:, None]
        frac = torch.log2(sigma) - torch.log2(sigma).round()
        for i in range(S):
            m = n - S + i + 1
            if m <= 0:
                assert not out[b, i].any()
                continue
            s = q[b, i].double().cuda() @ K[:m].T.contiguous() * scale
            p = torch.softmax(s, -1)
            V = K[:m, :512].contiguous()
            ref, A = p @ V, p @ V.abs()
            rest = p.clone()
            key = s * 1.4426950408889634 + frac[:m]
            for c0 in range(0, m, 64):
                rest[:, c0:c0 + 64].scatter_(1, key[:, c0:c0 + 64].argmax(-1, keepdim=True), 0.0)
            M = float(s.abs().max()) * 1.4426950408889634
            tol = 2.0 ** -8 * (rest @ V.abs()) + A * (2 * (4 * M * 2.0 ** -24 + 2.0 ** -21) + (n + 8) * 2.0 ** -24) + 1e-30
            err = (out[b, i] - ref).abs()
            assert (err <= tol).all(), f"sequence {b}: the worst {float((err / tol).max())} of the tolerance"
