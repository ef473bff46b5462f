"""Expanded latent attention (trnrt_amd/kernels/dsa_expand.py) against its definition in float64, and the whole family
together: expanded against absorbed (dsa_dense) attention, and attention across forks and compaction (dsa_pages).

Tolerances, from the arithmetic. expand: fp32 sums of 512 exact products, off by less than 512 2^-24 of the sum of their
sizes, then one rounding to bf16 (2^-8 of the value) after the scale's (2^-24). attend: the scores' fp32 error E (D 2^-24
times the sum of |q k|, the largest over the keys) moves weights by that much relative; each weight is rounded to bf16, off by
at most 2^-8 of it, so an output by at most 2^-8 of A = sum p |v|; a bf16 output is rounded once more."""

import pytest
import torch

from tests._helpers import say
from tests.test_gpu_dense import make, reference
from trnrt_amd.kernels import dsa_cache, dsa_dense, dsa_expand, dsa_pages

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


def cu_of(lens):
    return torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32)


def weights(H, seed):
    return (torch.randn(H, 256, 512, generator=torch.Generator().manual_seed(seed)) * 512 ** -0.5).to(torch.bfloat16)


def gather(kv, sc, table, lens, ps):
    rows = []
    for b, n in enumerate(lens):
        t = torch.arange(n)
        slot = table[b][t // ps].long() * ps + t % ps
        K = kv[slot].view(FP8).double()
        rows.append(K if sc is None else K * sc[slot].double()[:, None])
    return torch.cat(rows)


@pytest.mark.parametrize("lens,H,D,ps", [
    ([1], 1, 576, 64), ([300, 0, 5, 256], 3, 576, 64), ([257, 255], 4, 512, 16), ([700], 16, 576, 33), ([64] * 20, 5, 512, 64),
    ([0, 0, 1000, 0], 8, 576, 1), ([3] * 700, 2, 576, 64),
])
@pytest.mark.parametrize("scaled", [True, False])
def test_expand(lens, H, D, ps, scaled):
    say("expand", len(lens), sum(lens), H, D, ps, scaled)
    _, kv, sc, table, _ = make(lens, 1, 1, D, ps, seed=H, scaled=scaled)
    w = weights(H, H)
    total, spare = sum(lens), 3  # three rows behind the last sequence
    guard = [torch.full((total + spare, *s), 7.0, dtype=torch.bfloat16, device="cuda") for s in ((H, 128), (64,), (H, 128))]
    k, r, v = dsa_expand.expand(kv.cuda(), None if sc is None else sc.cuda(), table.cuda(), cu_of(lens).cuda(),
                                total + spare, ps, w.cuda(), out=(guard[0], guard[1] if D > 512 else None, guard[2]))
    c = gather(kv, sc, table, lens, ps).cuda()
    W = w.double().cuda()
    for got, part in ((k, W[:, :128]), (v, W[:, 128:])):
        ref = (c[:, :512].contiguous() @ part.reshape(H * 128, 512).T.contiguous()).view(total, H, 128)
        size = (c[:, :512].abs().contiguous() @ part.reshape(H * 128, 512).abs().T.contiguous()).view(total, H, 128)
        tol = size * (512 * 2.0 ** -24 + 2.0 ** -22) * (1 + 2.0 ** -8) + 2.0 ** -8 * ref.abs() + 1e-30
        assert ((got[:total].double() - ref).abs() <= tol).all()
        assert (got[total:] == 7).all()  # left as they were
    if D > 512:
        rope = c[:, 512:]
        assert ((r[:total].double() - rope).abs() <= (2.0 ** -8 + 2.0 ** -23) * rope.abs()).all() and (r[total:] == 7).all()
    else:
        assert r is None


def test_expand_padded_batch():
    """Thousands of sequences without tokens around the few that have some."""
    say("expand padded batch")
    test_expand([5] + [0] * 3000 + [300, 0, 1] + [0] * 700 + [40], 2, 576, 64, True)


def attend_ref(q, k, r, v, lq, lk, scale, causal):
    Tq, H, _ = q.shape
    out = torch.zeros(Tq, H, 128, dtype=torch.float64, device="cuda")
    lse = torch.full((Tq, H), -1e30, dtype=torch.float64, device="cuda")
    A, E = torch.zeros_like(out), torch.zeros_like(lse)
    q, k, v = q.double(), k.double(), v.double()
    q0 = k0 = 0
    for nq, nk in zip(lq, lk):
        for h in range(H):
            key = k[k0:k0 + nk, h]
            if r is not None:
                key = torch.cat([key, r[k0:k0 + nk].double()], 1)
            x = q[q0:q0 + nq, h]
            s = x @ key.T.contiguous() * scale
            seen = (nk - nq + 1 + torch.arange(nq, device="cuda")).clamp(max=nk) if causal else torch.full((nq,), nk, device="cuda")
            s = s.masked_fill(torch.arange(nk, device="cuda") >= seen[:, None], -torch.inf)
            ok = seen > 0
            if nk == 0 or not ok.any():
                continue
            p = torch.softmax(s[ok], -1)
            rows = torch.arange(q0, q0 + nq, device="cuda")[ok]
            out[rows, h] = p @ v[k0:k0 + nk, h].contiguous()
            A[rows, h] = p @ v[k0:k0 + nk, h].abs().contiguous()
            lse[rows, h] = torch.logsumexp(s[ok], -1)
            E[rows, h] = (x[ok].abs() @ key.abs().T.contiguous()).amax(-1) * scale * x.shape[1] * 2.0 ** -24
        q0 += nq
        k0 += nk
    return out, lse, A, E


def check_attend(lq, lk, H, rope, causal, seed=0, gain=1.5, out_dtype=torch.bfloat16, scale=192 ** -0.5, spare=2):
    g = torch.Generator().manual_seed(seed)
    Tq, Tk, D = sum(lq), sum(lk), 192 if rope else 128
    q = (torch.randn(Tq + spare, H, D, generator=g) * gain).to(torch.bfloat16).cuda()
    k, v = (torch.randn(Tk, H, 128, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    r = torch.randn(Tk, 64, generator=g).to(torch.bfloat16).cuda() if rope else None
    out = torch.full((Tq + spare, H, 128), 7.0, dtype=out_dtype, device="cuda")
    out, lse = dsa_expand.attend(q, k, r, v, cu_of(lq).cuda(), cu_of(lk).cuda(), scale, causal=causal, out=out)
    ref, lref, A, E = attend_ref(q[:Tq], k, r, v, lq, lk, scale, causal)
    assert (out[Tq:] == 7).all()  # rows of no sequence
    rel = 2.0 ** -8 + 2 * E[..., None] + 2.0 ** -20
    tol = A * rel + (2.0 ** -8 * (ref.abs() + A * rel) if out_dtype == torch.bfloat16 else 0) + 1e-30
    err = (out[:Tq].double() - ref).abs()
    assert (err <= tol).all(), f"{int((~(err <= tol)).sum())} outputs off, the worst {float((err / tol).max())} of the tolerance"
    ltol = E + 2.0 ** -21 + 2.0 ** -22 * lref.abs()
    err = (lse[:Tq].double() - lref).abs()
    assert (err <= ltol).all(), f"lse off by {float((err / ltol).max())} of the tolerance"


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("rope", [True, False])
@pytest.mark.parametrize("lq,lk,H", [
    ([1], [1], 1), ([64], [64], 8), ([300, 1, 0, 257], [300, 65, 4, 600], 3), ([5, 700], [5, 700], 16), ([256, 256], [256, 512], 5),
    ([10, 3, 2], [4, 0, 1], 2),  # queries without a key
    ([1] * 300, [7] * 300, 2), ([1000], [1900], 8),
])
def test_attend(lq, lk, H, rope, causal):
    say("expanded attend", len(lq), sum(lq), sum(lk), H, rope, causal)
    check_attend(lq, lk, H, rope, causal, seed=H)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lq,lk,H,rope", [
    ([100], [5000], 16, True), ([1], [1500], 1, False), ([300, 1, 0], [9001, 4000, 70], 3, True),
    ([256, 257], [3000, 2900], 8, False), ([40, 3], [20000, 2], 16, True), ([600], [700], 5, True), ([2, 2], [0, 9000], 24, True)])
def test_attend_splits(lq, lk, H, rope, causal):
    """Few queries over many keys: the keys of a query tile shared by several workgroups, some of them without any."""
    say("attend splits", lq, lk, H, rope, causal)
    check_attend(lq, lk, H, rope, causal)


def test_attend_graph_has_its_own_workspace():
    """Graphs captured without a workspace keep their results while eager calls and another graph use the stream's."""
    say("attend, two graphs and eager calls")
    g = torch.Generator().manual_seed(3)
    ins = []
    for nq, nk, H in ((70, 4000, 4), (130, 9000, 8)):
        t = [torch.randn(n, H, d, generator=g).bfloat16().cuda() for n, d in ((nq, 128), (nk, 128), (nk, 128))]
        ins.append((t[0], t[1], None, t[2], cu_of([nq]).cuda(), cu_of([nk]).cuda(), 0.1))
    want = [tuple(x.clone() for x in dsa_expand.attend(*a)) for a in ins]
    graphs = []
    for a in ins:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = dsa_expand.attend(*a)
        graphs.append((graph, got))
    for _ in range(3):
        for graph, got in graphs:
            for x in got:
                x.zero_()
        for i in (0, 1, 0):
            graphs[i][0].replay()
        for i in (1, 0):
            assert all(torch.equal(x, y) for x, y in zip(dsa_expand.attend(*ins[i]), want[i]))
        torch.cuda.synchronize()
        for (_, got), w in zip(graphs, want):
            assert all(torch.equal(x, y) for x, y in zip(got, w))


def test_attend_more_sequences_than_threads():
    say("expanded attend, 1,300 sequences")
    g = torch.Generator().manual_seed(1)
    lq = torch.randint(0, 4, (1300,), generator=g).tolist()
    check_attend(lq, [n + 2 for n in lq], 1, True, True)


@pytest.mark.parametrize("gain", [0.0, 20.0, 100.0])
def test_attend_flat_and_steep(gain):
    say("expanded attend gain", gain)
    check_attend([700], [900], 4, True, True, gain=gain)


def test_attend_fp32_outputs():
    say("expanded attend fp32")
    check_attend([130, 40], [130, 400], 8, True, True, out_dtype=torch.float32)


def test_attend_without_keys():
    say("expanded attend no keys")
    q = torch.ones(5, 2, 128, dtype=torch.bfloat16, device="cuda")
    k = torch.empty(0, 2, 128, dtype=torch.bfloat16, device="cuda")
    cu = torch.tensor([0, 5], dtype=torch.int32, device="cuda")
    out, lse = dsa_expand.attend(q, k, None, k, cu, torch.zeros_like(cu), 0.1, causal=False)
    assert not out.any() and (lse == -1e30).all()
    none = torch.zeros(1, dtype=torch.int32, device="cuda")  # no sequence
    out, lse = dsa_expand.attend(q[:0], k, None, k, none, none, 0.1)
    assert out.shape == (0, 2, 128)


def test_refusals():
    z = torch.zeros(4, 2, 128, dtype=torch.bfloat16, device="cuda")
    r = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
    cu = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    ok = dict(q=z, k=z, k_rope=None, v=z, cu_q=cu, cu_k=cu, scale=0.1)
    for bad in (dict(k_rope=r), dict(q=z[0]), dict(k=z[:, :1]), dict(v=z[:3]), dict(cu_q=cu[:1]), dict(cu_q=cu.view(1, 2)),
                dict(out=z[:3]), dict(out=z.half())):
        with pytest.raises(ValueError):
            dsa_expand.attend(**{**ok, **bad})
    kv = torch.zeros(64, 576, dtype=torch.uint8, device="cuda")
    w = torch.zeros(2, 256, 512, dtype=torch.bfloat16, device="cuda")
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    ok = dict(kv_cache=kv, kv_scale=None, table=table, cu_len=cu, total=4, page_size=64, w=w)
    for bad in (dict(kv_cache=kv[:, :500]), dict(page_size=48), dict(kv_scale=torch.ones(3, device="cuda")), dict(w=w[0]),
                dict(w=w[:, :128]), dict(w=w.float()), dict(table=table[0]), dict(cu_len=cu[:1]), dict(total=-1),
                dict(out=(z, None, z)), dict(out=(z, r[:2], z)), dict(out=(z[:2], r, z))):
        with pytest.raises(ValueError):
            dsa_expand.expand(**{**ok, **bad})


def test_expanded_equals_absorbed():
    """One chunk of a sequence through both forms: expand + attend, and the absorbed queries through dsa_dense.attend times
    W_UV. The one side rounds the keys to bf16, the other the absorbed queries: scores differ by at most 2 x 2^-8 of scale
    sum |q k|, at most about 8 here, so the log-sum-exps by 6e-2 at most, and the weights by twice that relative; on top the
    values', weights' and outputs' roundings, 3 x 2^-8 of sizes up to about 1."""
    say("expanded against absorbed")
    H, S, n = 8, 6, 500
    _, kv, sc, table, lens = make([n, 77], 1, 1, 576, 64, seed=3)
    w = weights(H, 5)
    g = torch.Generator().manual_seed(6)
    q = (torch.randn(2, S, H, 192, generator=g) * 0.7).to(torch.bfloat16).cuda()
    kv, sc, table, lens, w = (x.cuda() for x in (kv, sc, table, lens, w))
    scale = 192 ** -0.5
    cu_k, cu_q = cu_of([n, 77]).cuda(), cu_of([S, S]).cuda()
    k, r, v = dsa_expand.expand(kv, sc, table, cu_k, n + 77, 64, w)
    o1, l1 = dsa_expand.attend(q.view(2 * S, H, 192), k, r, v, cu_q, cu_k, scale)
    q_lat = torch.stack([q[..., h, :128].float() @ w[h, :128].float() for h in range(H)], 2)
    o_lat, l2 = dsa_dense.attend(torch.cat([q_lat, q[..., 128:].float()], -1), kv, sc, table, lens, 64, scale,
                                 out_dtype=torch.float32)
    o2 = torch.stack([o_lat[..., h, :] @ w[h, 128:].float().T.contiguous() for h in range(H)], 2)
    torch.testing.assert_close(o1.float().view(2, S, H, 128), o2, atol=0.13, rtol=2e-2)
    torch.testing.assert_close(l1.view(2, S, H), l2, atol=6e-2, rtol=0)


def test_store_fork_attend_compact():
    """A serving step's life of pages: two sequences stored, forked into samples that go on differently, attended to, a
    parent released, the pool compacted; attention reads the same bits before and after, and each sample its own tokens."""
    say("store, fork, attend, release, compact")
    ps, mp, pages, H = 16, 8, 40, 16
    g = torch.Generator().manual_seed(8)
    kv = torch.zeros(pages * ps, 576, dtype=torch.uint8, device="cuda").view(FP8)
    sc = torch.zeros(pages * ps, device="cuda")
    lens = [50, 33]
    table = torch.zeros(2, mp, dtype=torch.int32)
    table[0, :4], table[1, :3] = torch.tensor([7, 30, 12, 9]), torch.tensor([21, 3, 38])
    ref = torch.zeros(pages, dtype=torch.int32)
    ref[table[table > 0].long()] = 1
    table, ref, ln = table.cuda(), ref.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    rows = [torch.randn(n, 576, generator=g).cuda() for n in lens]
    for b in range(2):
        dsa_cache.store(kv, dsa_cache.slots_of(torch.arange(lens[b], device="cuda"), table[b], ps), rows[b], scale=sc)
    parents = torch.tensor([0, 0, 1], dtype=torch.int32, device="cuda")
    child, new = dsa_pages.fork(ref, table, ln, parents, [kv, sc], ps)
    assert (new > 0).all()
    clen = ln[parents.long()] + 1
    added = torch.randn(3, 576, generator=g).cuda()  # each sample's next token
    dsa_cache.store(kv, dsa_cache.slots_of(clen - 1, child, ps), added, scale=sc)
    dsa_pages.release(ref, table[:1], ln[:1], ps)  # the first parent ends, its shared pages live on
    every = torch.cat([table[1:], child])
    q = torch.randn(4, H, 576, generator=g).to(torch.bfloat16).cuda()
    alen = torch.cat([ln[1:], clen])
    before = dsa_dense.attend(q, kv, sc, every, alen, ps, 0.05)
    moved, ref2, remap = dsa_pages.compact(ref, every, [kv, sc], ps)
    live = int((ref > 0).sum())
    assert live == 3 + 3 + 3 and int((ref2[1:live + 1] > 0).sum()) == live and int(moved.max()) == live
    kv.view(torch.uint8)[(live + 1) * ps:] = 0x7F  # NaN in every page past the front
    after = dsa_dense.attend(q, kv, sc, moved, alen, ps, 0.05)
    assert torch.equal(before[0], after[0]) and torch.equal(before[1], after[1])
    out, lse, A, _ = reference(q.cpu()[:, None], kv.view(torch.uint8).cpu(), sc.cpu(), moved.cpu(), alen.cpu(), ps, 0.05)
    assert ((after[0].double().cpu() - out[:, 0]).abs() <= 2.0 ** -7 * A[:, 0] + 1e-6).all()
    k, r, v = dsa_expand.expand(kv, sc, moved, cu_of(alen.tolist()).cuda(), int(alen.sum()), ps, weights(2, 1).cuda())
    want = torch.cat([rows[1], rows[0], added[:1], rows[0], added[1:2], rows[1], added[2:]])[:, 512:]
    assert (r.float() - want).abs().max() <= 2.0 ** -4 * want.abs().max()  # e4m3's half step
    assert not torch.isnan(k).any() and not torch.isnan(v).any()


@pytest.mark.parametrize("lq,lk,H", [([70, 3], [70, 3], 8), ([3, 2], [9000, 40], 4)])
def test_attend_nan_reaches_the_lse(lq, lk, H):
    """A key's NaN shows in the lse of the queries that see it, with the keys in splits or not; a value's only in the
    outputs."""
    say("expanded attend NaN", lq, lk, H)
    g = torch.Generator().manual_seed(H)
    q = torch.randn(sum(lq), H, 128, generator=g).bfloat16().cuda()
    k, v = (torch.randn(sum(lk), H, 128, generator=g).bfloat16().cuda() for _ in range(2))
    cu_q, cu_k = cu_of(lq).cuda(), cu_of(lk).cuda()
    k2, v2 = k.clone(), v.clone()
    k2[lk[0] - 2, 1, 5] = float("nan")  # the first sequence's last key but one: its last two queries see it
    v2[lk[0] + 1, 0, 9] = float("nan")  # a value of the second sequence
    want, lwant = dsa_expand.attend(q, k, None, v, cu_q, cu_k, 0.1)
    out, lse = dsa_expand.attend(q, k2, None, v2, cu_q, cu_k, 0.1)
    n = lq[0]
    assert lse[n - 2:n, 1].isnan().all() and out[n - 2:n, 1].isnan().all()
    rest = torch.ones_like(lse, dtype=torch.bool)
    rest[n - 2:n, 1] = False
    assert torch.equal(lse[rest], lwant[rest])
    heads = [h for h in range(H) if h != 1]
    assert torch.equal(out[:n, heads], want[:n, heads])
    assert out[-1, 0, 9].isnan() and torch.equal(out[n:, 1:], want[n:, 1:])


@pytest.mark.parametrize("lens,H,D", [
    ([1021], 16, 576), ([1022], 16, 576),  # the last batch whose 128-token tiles run at once, and one row past it
    ([700, 1, 0, 1500, 797], 16, 576), ([4095], 16, 512), ([4097 - 3], 16, 576), ([4097], 16, 512),
    ([12000], 3, 576), ([9000, 0, 20000, 1, 999], 5, 512), ([257] * 40, 7, 576), ([2], 160, 576)])
def test_expand_shares(lens, H, D):
    """Tiles of 256 tokens, and workgroups with several units: weights that run on from part to part, stores under the next
    unit's products, shares that begin and end inside a tile and go on into the next, tiles that end early."""
    say("expand shares", len(lens), sum(lens), H, D)
    test_expand(lens, H, D, 64, True)


def test_expand_shares_plan():
    """Which form and how many units a workgroup those take (as launch_expand_latent has it, 256 CUs): both forms, shares of
    one unit and of several, some of them beginning inside a tile."""
    seen = set()
    for lens, H in (([1021], 16), ([1022], 16), ([12000], 3), ([9000, 0, 20000, 1, 999], 5), ([2], 160)):
        total = sum(lens) + 3
        tok = 128 if -(-total // 128) * 2 * H <= 256 else 256
        units = -(-total // tok) * 2 * H
        grid = min(units, 256)
        starts = [units * g // grid for g in range(grid + 1)]
        seen.add((tok, units > grid, any(u % (2 * H) and u // (2 * H) != (v - 1) // (2 * H) for u, v in zip(starts, starts[1:]))))
    assert {(128, False, False), (256, False, False), (256, True, True)} <= seen
