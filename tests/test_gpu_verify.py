"""Verification of drafts (trnrt_amd/kernels/dsa_verify.py) against a loop over rows in numpy's float64: tokens and counts
equal, the log probabilities within 2^-24 of themselves (they are rounded once) and 2^-17: a row's sum is of 32-bit exponentials
whose exponents are off by 1.5 x 2^-23 of themselves, 20 at the weights' mean at most (20 x 1.5 x 2^-23 ln 2 = 2.5e-6), exp2 by
2^-23 twice (a logit's and its wave's), a term goes through 16 roundings on its way into the sum (1e-6) and the sum through two
more: 3.9e-6, less than 2^-17 = 7.6e-6."""

import math

import numpy as np
import pytest
import torch

from tests._helpers import say
from trnrt_amd.kernels import dsa_verify

pytestmark = pytest.mark.gpu


def softmax(logits, temperature):
    x = logits.astype(np.float64)
    x = np.where(x > -np.inf, x, -np.inf)  # (NaN too)
    m = x.max()
    if m == -np.inf:
        return np.zeros_like(x), np.full_like(x, -np.inf)
    t = float(temperature) if temperature > 0 else 1.0
    with np.errstate(invalid="ignore"):  # (-infinity over an infinite temperature)
        e = np.where(x == m, 0.0, -np.inf if m == np.inf else np.where(x > -np.inf, (x - m) / t, -np.inf))
    p = np.exp(e)
    return p / p.sum(), e - math.log(p.sum())


def first_max(logits):
    x = np.where(logits > -np.inf, logits, -np.inf)
    return int(np.argmax(x)) if x.max() > -np.inf else -1


def reference(logits, draft, cu, u, v, temperature, probs):
    N, V = logits.shape
    tokens, logp, accepted = np.full(N, -1), np.zeros(N), np.zeros(len(cu) - 1, dtype=int)
    for b in range(len(cu) - 1):
        warm = temperature[b] > 0
        for j in range(cu[b], cu[b + 1]):
            p, lp = softmax(logits[j], temperature[b])
            x, last = int(draft[j]), j == cu[b + 1] - 1
            if not last:
                known = 0 <= x < V
                if warm:
                    q = 1.0 if probs is None else float(probs[j, x]) if known else 0.0
                    taken = known and float(u[j]) * q < p[x]
                else:
                    taken = known and x == first_max(logits[j])
                if taken:
                    tokens[j], logp[j] = x, lp[x]
                    accepted[b] += 1
                    continue
            if not warm:
                y = first_max(logits[j])
            else:
                r = p.copy()
                if not last and probs is None and 0 <= x < V:
                    r[x] = 0
                elif not last and probs is not None:
                    r = np.maximum(p - probs[j].astype(np.float64), 0)
                if not r.sum() > 0:
                    r = p
                c = np.cumsum(r)
                over = np.nonzero(c > float(v[b]) * c[-1])[0]
                y = int(over[0]) if len(over) else -1
            tokens[j] = y
            logp[j] = lp[y] if y >= 0 else 0.0
            break
    return tokens, accepted, logp


def numbers(t):
    return None if t is None else t.float().cpu().numpy()


def check(logits, draft, cu, u, v, temperature, probs=None, got=None):
    N = logits.shape[0]
    args = [t.cuda() for t in (draft, cu, u, v, temperature)]
    tokens, accepted, logp = dsa_verify.verify(logits, *args, draft_probs=probs) if got is None else got
    rt, ra, rl = reference(numbers(logits), draft.numpy(), cu.numpy(), u.numpy(), v.numpy(), temperature.numpy(), numbers(probs))
    assert (accepted.cpu().numpy() == ra).all(), (accepted.cpu().numpy(), ra)
    a, z = int(cu[0]), int(cu[-1])
    assert (tokens.cpu().numpy()[a:z] == rt[a:z]).all(), (tokens.cpu().numpy()[a:z], rt[a:z])
    err = np.abs(logp.double().cpu().numpy()[a:z] - rl[a:z])
    assert (err <= 2.0 ** -24 * np.abs(rl[a:z]) + 2.0 ** -17).all()
    assert tokens.shape == logp.shape == (N,)
    return tokens, accepted, logp


def make(rows, V, dtype, probs, seed, near=0.5):
    g = torch.Generator().manual_seed(seed)
    N, B = sum(rows), len(rows)
    target = torch.randn(N, V, generator=g) * 3
    logits = target.to(dtype).cuda()
    temperature = torch.tensor([0.0 if b % 4 == 2 else 0.5 + 0.3 * (b % 3) for b in range(B)])
    seq = torch.repeat_interleave(torch.arange(B), torch.tensor(rows))
    q = torch.softmax((target + near * torch.randn(N, V, generator=g)) / temperature.clamp(min=0.3)[seq][:, None], -1)
    draft = torch.multinomial(q, 1, generator=g)[:, 0].to(torch.int32) if N else torch.zeros(0, dtype=torch.int32)
    cu = torch.tensor([0] + rows).cumsum(0).to(torch.int32)
    u, v = torch.rand(N, generator=g), torch.rand(B, generator=g)
    return logits, draft, cu, u, v, temperature, None if probs is None else q.to(probs).cuda()


@pytest.mark.parametrize("rows,V", [
    ([1], 1), ([4], 2), ([2, 1, 5, 0, 3], 7), ([5] * 13, 1000), ([1, 8, 2, 9], 8191), ([3, 3], 8192), ([2, 4, 1], 8193),
    ([5, 5, 2], 65537), ([3] * 200, 33), ([300, 2], 64), ([2, 3], 600001),
    ([4, 1, 0, 9] * 11, 65537), ([70] * 3, 70000),
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("probs", [None, torch.float32, torch.bfloat16])
def test_verify(rows, V, dtype, probs):
    say("verify", len(rows), sum(rows), V, dtype, probs)
    check(*make(rows, V, dtype, probs, V + len(rows)))


def test_everything_taken_and_nothing():
    say("verify taken")
    logits, draft, cu, u, v, temperature, q = make([6] * 9, 500, torch.float32, torch.float32, 3)
    _, accepted, _ = check(logits, draft, cu, torch.zeros_like(u), v, temperature.clamp(min=0.4), q)
    assert (accepted == 5).all()
    far = (draft + 250) % 500
    z = torch.zeros(54, 500)
    z.scatter_(1, draft.long()[:, None], 1.0)  # the draft is certain of what the target holds unlikely
    hard = logits.clone()
    hard[torch.arange(54), draft.long().cuda()] = -40.0
    _, accepted, _ = check(hard, draft, cu, u.clamp(min=0.01), v, temperature, z.cuda())
    assert (accepted == 0).all()
    check(logits, far, cu, u, v, temperature, q)


def test_masks_ties_and_strange_logits():
    """-infinity, NaN, +infinity (one and several), rows with nothing left, equal logits, and their greedy forms."""
    say("verify strange")
    V = 9000
    logits, draft, cu, u, v, temperature, q = make([3] * 12, V, torch.float32, torch.float32, 11)
    logits[:, 5000:] = -torch.inf
    logits[0:6] = 1.5  # all equal
    logits[7, 8191:8194] = torch.inf
    logits[9, 100] = torch.inf
    logits[12, ::3] = torch.nan
    logits[15:18] = -torch.inf  # nothing can come
    logits[19] = torch.nan
    logits[21:24] = torch.tensor(float(torch.finfo(torch.float32).min))
    logits[24, 1:] = -torch.inf
    for heat in (temperature, torch.zeros(12), torch.full((12,), 1e-3), torch.full((12,), 1e30), torch.full((12,), torch.nan)):
        check(logits, draft, cu, u, v, heat, q)
        check(logits, draft, cu, u, v, heat)
    low = logits.bfloat16()
    check(low, draft, cu, u, v, temperature, q.bfloat16())


@pytest.mark.parametrize("V", [300, 40000])
def test_strange_temperatures(V):
    """Infinite ones (all tokens that can come alike), the least and the largest, beside masked and infinite logits."""
    say("verify, strange temperatures", V)
    temperature = torch.tensor([math.inf, 1e30, 1e-30, 1e-45, 3e38, math.nan, -1.0, math.inf])
    logits, draft, cu, u, v, _, q = make([4] * 8, V, torch.float32, torch.float32, 5)
    logits[:, V // 3:V // 2] = -math.inf
    logits[29:, 7] = math.inf
    check(logits, draft, cu, u, v, temperature, q)
    check(logits, draft, cu, u, v, temperature)


def test_edges_of_the_random_numbers():
    """u and v at 0 and just under 1; drafts that are no tokens; a draft that leaves nothing over."""
    say("verify edges")
    most = 1 - 2.0 ** -24
    for probs in (None, torch.float32):
        logits, draft, cu, u, v, temperature, q = make([4] * 10, 20000, torch.bfloat16, probs, 21)
        for a in (0.0, most):
            check(logits, draft, cu, torch.full_like(u, a), torch.full_like(v, a), temperature, q)
        odd = draft.clone()
        odd[::5], odd[3::7] = -1, 20000
        check(logits, odd, cu, u, v, temperature, q)
    # q above p everywhere: a draft is refused with r = 0, and the token comes from p
    q = torch.full((40, 20000), 2.0, device="cuda")
    check(logits, draft, cu, u.clamp(min=0.5), v, temperature, q)
    # one token holds everything; its draft is taken, another's is refused
    sure = torch.full((40, 20000), -torch.inf, device="cuda")
    sure[:, 12345] = 3.0
    check(sure, torch.full_like(draft, 12345), cu, u, v, temperature)
    check(sure, torch.full_like(draft, 12344), cu, u, v, temperature)


@pytest.mark.parametrize("V", [3, 700, 40000, 100000])  # (the last with the stop rows in a launch of their own)
def test_decisions_that_32_bits_do_not_make(V):
    """u q within an fp32 rounding of p, on either side; and a draft whose probabilities are the target's own, rounded, refused
    all the same: what is left over is roundings, and the token is the one that they give in 64 bits."""
    say("verify close", V)
    for dtype in (torch.bfloat16, torch.float32):
        logits, draft, cu, u, v, temperature, _ = make([3] * 40, V, dtype, None, V)
        temperature = temperature.clamp(min=0.7)
        seq = torch.arange(40).repeat_interleave(3)
        p = torch.softmax(logits.cpu().double() / temperature.double()[seq][:, None], -1)
        q = p.float()
        px = p.gather(1, draft.long()[:, None])[:, 0]
        half = q.clone()
        half.scatter_(1, draft.long()[:, None], (2 * px).float()[:, None])
        _, accepted, _ = check(logits, draft, cu, torch.full_like(u, 0.5), v, temperature, half.cuda())
        assert (accepted > 0).any() and (accepted < 2).any()
        above = q.clone()  # q just above p at the drafted token, so that u just under 1 refuses it
        above.scatter_(1, draft.long()[:, None], (px * (1 + 2.0 ** -20)).float()[:, None])
        _, accepted, _ = check(logits, draft, cu, torch.full_like(u, 1 - 2.0 ** -24), v, temperature, above.cuda())
        assert (accepted < 2).any()
        check(logits, draft, cu, torch.full_like(u, 1 - 2.0 ** -24), v, temperature, (q * (1 + 3e-6)).cuda())


def test_views_and_rows_outside():
    """Rows of padded matrices that start between 16 bytes; rows before the first and behind the last sequence."""
    say("verify views")
    for dtype, at in ((torch.bfloat16, 1), (torch.bfloat16, 3), (torch.float32, 1), (torch.float32, 2)):
        logits, draft, cu, u, v, temperature, q = make([3, 0, 4, 2], 10007, dtype, torch.bfloat16, at)
        wide, qw = (torch.full((9, 10007 + 5), 50.0, dtype=t.dtype, device="cuda") for t in (logits, q))
        wide[:, at:at + 10007], qw[:, at + 1:at + 10008] = logits, q
        check(wide[:, at:at + 10007], draft, cu, u, v, temperature, qw[:, at + 1:at + 10008])
        check(logits.T.contiguous().T, draft, cu, u, v, temperature, q)
    inner = torch.tensor([1, 3, 3, 7], dtype=torch.int32)
    check(logits, draft, inner, u, v[:3], temperature[:3], q)


def test_rows_of_any_stride():
    """A single row whose stride is below its width, a vocabulary of one token, one row for all, columns apart."""
    say("verify, strides")
    x, q = torch.randn(904, generator=torch.Generator().manual_seed(3)).cuda(), torch.full((904,), 0.01).cuda()
    for N, V, strides in [(1, 700, (0, 1)), (1, 700, (5, 1)), (1, 1, (1, 7)), (4, 1, (3, 7)), (4, 300, (0, 1)),
                          (4, 300, (2, 3))]:
        logits, probs = x.as_strided((N, V), strides), q.as_strided((N, V), strides)
        rand = torch.Generator().manual_seed(N + V)
        check(logits, torch.randint(0, V, (N,), generator=rand, dtype=torch.int32), torch.tensor([0, N], dtype=torch.int32),
              torch.rand(N, generator=rand), torch.rand(1, generator=rand), torch.ones(1), probs)


def test_rows_far_apart():
    """Rows of logits and probabilities whose offsets pass 2^31 values."""
    say("verify far apart")
    logits, draft, cu, u, v, temperature, q = make([3, 1], 5000, torch.bfloat16, torch.bfloat16, 8)
    row = 900_000_000
    far, qf = (torch.as_strided(torch.empty(3 * row + 5000, dtype=torch.bfloat16, device="cuda"), (4, 5000), (row, 1)) for _ in "ab")
    far.copy_(logits), qf.copy_(q)
    check(far, draft, cu, u, v, temperature, qf)


def test_no_rows():
    say("verify no rows")
    z = torch.zeros(0, device="cuda")
    i = torch.zeros(0, dtype=torch.int32, device="cuda")
    tokens, accepted, logp = dsa_verify.verify(torch.zeros(0, 100, device="cuda"), i, torch.zeros(4, **dict(dtype=torch.int32,
                                               device="cuda")), z, torch.zeros(3, device="cuda"), torch.ones(3, device="cuda"))
    assert tokens.numel() == 0 and logp.numel() == 0 and (accepted == 0).all()
    out = dsa_verify.verify(torch.zeros(0, 100, device="cuda"), i, torch.zeros(1, dtype=torch.int32, device="cuda"), z, z, z)
    assert [t.numel() for t in out] == [0, 0, 0]


def test_distribution():
    """What comes out first is distributed as the target's samples, whatever the draft: 40,000 sequences of one draft over 12
    tokens; a count off by 5 of its standard deviations comes once in two million."""
    say("verify distribution")
    g = torch.Generator().manual_seed(77)
    B, V = 40000, 12
    row = torch.randn(V, generator=g) * 1.5
    q = torch.softmax(row + torch.randn(V, generator=g), -1)
    p = torch.softmax(row.double() / 0.9, -1)
    draft = torch.multinomial(q, 2 * B, replacement=True, generator=g).to(torch.int32)
    cu = torch.arange(0, 2 * B + 1, 2, dtype=torch.int32)
    u, v = torch.rand(2 * B, generator=g), torch.rand(B, generator=g)
    tokens, accepted, _ = dsa_verify.verify(row.cuda().expand(2 * B, V).contiguous(), draft.cuda(), cu.cuda(), u.cuda(), v.cuda(),
                                            torch.full((B,), 0.9).cuda(), draft_probs=q.cuda().expand(2 * B, V).contiguous())
    count = torch.bincount(tokens[0::2].cpu().long(), minlength=V).double()
    assert ((count - B * p).abs() <= 5 * (B * p * (1 - p)).sqrt()).all()
    share = torch.minimum(p, q.double()).sum()
    assert abs(accepted.double().mean().cpu() - share) <= 5 * (share * (1 - share) / B).sqrt()


def test_streams_threads_and_graphs():
    """A side stream, two host threads on one stream, two captured graphs replayed in turn with eager calls between."""
    import threading

    say("verify graphs")
    sets = [make([3, 5, 1], 9001, torch.bfloat16, torch.float32, 31), make([2] * 40, 30011, torch.float32, None, 32)]
    on = [tuple(None if t is None else t.cuda() for t in s) for s in sets]

    def run(s):
        return dsa_verify.verify(*s[:6], draft_probs=s[6])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [run(s) for s in on]
    side.synchronize()
    for s, o in zip(sets, got):
        check(*s, got=o)
    found = {}

    def many(k):
        found[k] = [run(on[k]) for _ in range(20)]

    threads = [threading.Thread(target=many, args=(k,)) for k in (0, 1)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.synchronize()
    for k in (0, 1):
        for o in found[k]:
            check(*sets[k], got=o)
    graphs, outs = [], []
    for s in on:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(run(s))
    g = torch.Generator().manual_seed(9)
    for _ in range(3):
        for k in (0, 1):
            sets[k][3].copy_(torch.rand(sets[k][3].shape, generator=g))
            sets[k][4].copy_(torch.rand(sets[k][4].shape, generator=g))
            on[k][3].copy_(sets[k][3]), on[k][4].copy_(sets[k][4])
            graphs[k].replay()
        run(on[1])
        torch.cuda.synchronize()
        for k in (0, 1):
            check(*sets[k], got=outs[k])


def test_refusals():
    logits, draft, cu, u, v, temperature, q = [t.cuda() for t in make([3, 2], 50, torch.float32, torch.float32, 1)]
    base = dict(logits=logits, draft=draft, cu=cu, u=u, v=v, temperature=temperature, draft_probs=q)
    dsa_verify.verify(**base)
    for kw in (dict(logits=logits.half()), dict(logits=logits[0]), dict(logits=logits[:, :0]), dict(draft=draft[1:]), dict(cu=cu[None]),
               dict(u=u[1:]), dict(u=u.double()), dict(v=u), dict(temperature=u), dict(draft_probs=q[1:]), dict(draft_probs=q.half()),
               dict(workspace=torch.empty(64, dtype=torch.uint8, device="cuda"))):
        with pytest.raises(ValueError):
            dsa_verify.verify(**{**base, **kw})
    with pytest.raises(RuntimeError, match="GPU only"):
        dsa_verify.verify(**{**base, "u": u.cpu()})


@pytest.mark.parametrize("B,V", [(1, 6), (9, 3000), (3, 70000), (40, 70000)])  # (the last with a launch for the stop rows)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_weights_that_are_nothing_in_64_bits(B, V, dtype):
    """Low temperatures, at which all but few tokens' probabilities are 0 in 64 bits (e^-1000 and less): with v = 0 the first token
    whose is not comes; and where the draft's probabilities leave nothing over of those few (r = 0), it comes from p."""
    say("verify, weights that are nothing", B, V, dtype)
    g = torch.Generator().manual_seed(V)
    rows = [3] * B
    N = 3 * B
    cu = torch.tensor([0] + rows).cumsum(0).to(torch.int32)
    main = torch.randint(V // 2, V, (N,), generator=g)
    logits = torch.randint(-3, 1, (N, V), generator=g).float()
    logits[torch.arange(N), main] = 10.0
    logits = logits.to(dtype).cuda()
    q = torch.zeros(N, V)
    q[torch.arange(N), main] = 1.0
    q[:, 2], q[:, 0] = 1e-30, 1e-38  # (drafts of these are refused: their p is 0)
    u, zero, most = torch.rand(N, generator=g), torch.zeros(B), torch.full((B,), 1 - 2.0 ** -24)
    for heat in (1e-3, 1e-2):
        temperature = torch.full((B,), heat)
        for v in (zero, most):
            for draft in (torch.full((N,), -1, dtype=torch.int32), torch.full((N,), 2, dtype=torch.int32), main.to(torch.int32)):
                for probs in (None, q.cuda(), q.to(torch.bfloat16).cuda()):
                    tokens, _, _ = check(logits, draft, cu, u, v, temperature, probs)
                    drawn = tokens.cpu()[tokens.cpu() >= 0].long()
                    assert torch.isin(drawn, main).all()


def test_targets_beside_a_tokens_edge():
    """v within 2e-12 to 4e-11 of where the running sum passes a token's end: r is (1e-5 of p, so that no token is too near to
    say) and its sums are such that the 32-bit row sum's error and a 32-bit sum of q together move them by more than that. In 64
    bits they are off by less than 1e-12: r by 3e-16 of p, 3e-11 of itself, at random over 100,000 tokens. The reference is in
    80 bits. The temperature is one whose reciprocal rounds badly, so that the 32-bit sum is off by 4e-7."""
    say("verify, edges")
    V, B = 100_000, 128
    rng = np.random.default_rng(5)
    heats = np.float32(0.9) + np.arange(4000, dtype=np.float32) * np.float32(2.0 ** -16)
    k = 1.4426950408889634 / heats.astype(np.float64)
    heat = heats[np.argmax(k.astype(np.float32) / k)]
    l = (np.round(rng.standard_normal(V) * 2 * 256) / 256).astype(np.float32)  # (differences exact in 32 bits)
    e = np.exp((l.astype(np.longdouble) - l.max()) / np.longdouble(heat))
    p = e / e.sum()
    q = (p * (1 + np.longdouble(1e-5) * np.where(rng.random(V) < 0.5, 1, -1))).astype(np.float32)
    r = np.maximum(p - q, 0)
    c = np.cumsum(r)
    c /= c[-1]
    ends = c[r > 0]
    vs = []
    for v in (ends.astype(np.float32), np.nextafter(ends.astype(np.float32), np.float32(0)),
              np.nextafter(ends.astype(np.float32), np.float32(1))):
        gap = np.abs(v - ends)
        vs.append(v[(gap > 2e-12) & (gap < 4e-11) & (v > 0) & (v < 1)])
    v = np.unique(np.concatenate(vs))
    assert len(v) >= 32
    v = rng.choice(v, B)
    want = np.array([int(np.nonzero(c > np.longdouble(x))[0][0]) for x in v])
    x = int(np.argmax(np.where(q > p, p, 0)))  # (u q > p: refused)
    row, probs = torch.tensor(l).cuda(), torch.tensor(q).cuda()
    for few in (4, B):  # (the stop rows found by the pick itself, and in a launch of their own)
        tokens = []
        for at in range(0, B, few):
            n = 2 * few
            tokens.append(dsa_verify.verify(
                row.expand(n, V).contiguous(), torch.full((n,), x, dtype=torch.int32).cuda(),
                torch.arange(0, n + 1, 2, dtype=torch.int32).cuda(), torch.full((n,), 1 - 2.0 ** -24).cuda(),
                torch.tensor(v[at:at + few]).cuda(), torch.full((few,), float(heat)).cuda(),
                draft_probs=probs.expand(n, V).contiguous())[0][0::2].cpu())
        got = torch.cat(tokens).numpy()
        assert (got == want).all(), (int((got != want).sum()), got[got != want], want[got != want])


def test_long_rows():
    """Rows past 2^25 logits, nearly all of them equal and 15 below one: their exponents are 20 in the weights' mean, as large as
    they can be, and each rounds alike (at the temperature of 4,000 whose reciprocal rounds worst). The drafts' u are the two fp32
    numbers on either side of p. Their sum by hand: one weight of 1 and V - 1 of e^(-15 / T)."""
    say("verify, long rows")
    V = (1 << 25) + 5
    heats = np.float32(0.99) + np.arange(4000, dtype=np.float32) * np.float32(2.0 ** -20)
    k = 1.4426950408889634 / heats.astype(np.float64)
    heat = float(heats[np.argmax(np.abs(k.astype(np.float32) / k - 1))])
    at = 31_234_567
    row = torch.full((V,), -15.0, device="cuda")
    row[at] = 0.0
    w = math.exp(-15.0 / heat)
    z = 1 + (V - 1) * w
    p = 1 / z
    below = np.float32(p)
    if float(below) >= p:
        below = np.nextafter(below, np.float32(0))
    above = np.nextafter(below, np.float32(1))
    logits = row.expand(4, V).contiguous()
    cu = torch.tensor([0, 2, 4], dtype=torch.int32).cuda()
    u = torch.tensor([below, 0.0, above, 0.0]).cuda()
    v = torch.tensor([0.25, 0.75]).cuda()
    draft = torch.full((4,), at, dtype=torch.int32).cuda()
    tokens, accepted, logp = (t.cpu() for t in dsa_verify.verify(logits, draft, cu, u, v, torch.full((2,), heat).cuda()))
    assert accepted.tolist() == [1, 0]
    assert tokens[0] == at and tokens[3] == -1
    # the second row: the first i whose running sum of weights is above 0.25 z; the third: without the draft, above 0.75
    assert tokens[1] == math.floor(0.25 * z / w) or abs(0.25 * z / w - round(0.25 * z / w)) < 1e-6
    # 0.75 (V - 1) is a whole number n: the running sum of the first n weights (token n - 1's end) is the target itself, and whether
    # it is above it is a matter of the 64-bit sums' roundings. Those are below 1e-13 of the target, and a weight is 4e-8 of it:
    # it is that token or the next.
    n = 3 * (V - 1) // 4
    assert 4 * n == 3 * (V - 1) and n < at
    assert tokens[2] in (n - 1, n)
    want = torch.tensor([math.log(p), -15.0 / heat - math.log(z), -15.0 / heat - math.log(z), 0.0], dtype=torch.float64)
    assert ((logp.double() - want).abs() <= 2.0 ** -24 * want.abs() + 2.0 ** -17).all()
