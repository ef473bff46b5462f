"""The page operations (trnrt_amd/kernels/dsa_pages.py) against plain host loops over the same state: every table, count
and byte equal, over odd page sizes, caches of odd widths and places, pools with no page free, empty sequences, parents that
are no rows, pages past the planning workgroups' blocks, more caches than one launch takes, a captured graph and another
stream."""

import pytest
import torch

from tests._helpers import say
from trnrt_amd.kernels import dsa_pages

pytestmark = pytest.mark.gpu


def fork_ref(ref, table, lens, parents, caches, ps):
    """The definition, one child after another."""
    ref, caches = ref.clone(), [c.clone() for c in caches]
    B, mp = table.shape
    free = iter([p for p in range(1, ref.numel()) if ref[p] <= 0])
    child, pages = torch.zeros(len(parents), mp, dtype=torch.int32), torch.zeros(len(parents), dtype=torch.int32)
    src = [c.clone() for c in caches]
    for i, p in enumerate(parents.tolist()):
        if not 0 <= p < B:
            pages[i] = -1
            continue
        n = min(max(int(lens[p]), 0), mp * ps)
        full = n // ps
        if n % ps:
            new = next(free, None)
            if new is None:
                pages[i] = -1
                continue
            pages[i] = new
            child[i, full] = new
            ref[new] += 1
            old = int(table[p, full])
            for c, s in zip(caches, src):
                c[new * ps:(new + 1) * ps] = s[old * ps:(old + 1) * ps]
        child[i, :full] = table[p, :full]
        for q in table[p, :full].tolist():
            if q:
                ref[q] += 1
    return child, pages, ref, caches


def compact_ref(ref, table, caches, ps):
    caches = [c.clone() for c in caches]
    live = [p for p in range(1, ref.numel()) if ref[p] > 0]
    L = len(live)
    remap = torch.zeros_like(ref)
    holes = [p for p in range(1, L + 1) if ref[p] <= 0]
    for p in live:
        remap[p] = p if p <= L else holes.pop(0)
    new_ref = torch.zeros_like(ref)
    for p in live:
        q = int(remap[p])
        new_ref[q] = ref[p]
        if q != p:
            for c in caches:
                c[q * ps:(q + 1) * ps] = c[p * ps:(p + 1) * ps]
    return remap[table.long()], new_ref, remap, caches


def make_caches(slots, widths, g):
    return [torch.randint(0, 256, (slots, w), dtype=torch.uint8, generator=g) for w in widths]


def make_pool(B, mp, ps, pages, seed, lens=None):
    """Sequences of random lengths with pages of their own, as many as the pool has."""
    g = torch.Generator().manual_seed(seed)
    table = torch.zeros(B, mp, dtype=torch.int32)
    ref = torch.zeros(pages, dtype=torch.int32)
    perm = (torch.randperm(pages - 1, generator=g) + 1).tolist()
    ln = torch.zeros(B, dtype=torch.int32)
    for b in range(B):
        n = int(torch.randint(0, mp * ps + 1, (1,), generator=g)) if lens is None else lens[b]
        k = min(-(-n // ps), len(perm))
        ln[b] = min(n, k * ps)
        for c in range(k):
            table[b, c] = perm.pop()
            ref[table[b, c]] += 1
    return g, ref, table, ln


def check_fork(ref, table, lens, parents, caches, ps):
    want = fork_ref(ref, table, lens, parents, caches, ps)
    gr, gc = ref.cuda(), [c.cuda() for c in caches]
    child, pages = dsa_pages.fork(gr, table.cuda(), lens.cuda(), parents.cuda(), gc, ps)
    assert torch.equal(child.cpu(), want[0])
    assert torch.equal(pages.cpu(), want[1])
    assert torch.equal(gr.cpu(), want[2])
    for i, (a, b) in enumerate(zip(gc, want[3])):
        assert torch.equal(a.cpu(), b), f"cache {i}"
    return gr, child, pages


@pytest.mark.parametrize("B,mp,ps,pages,n,widths", [
    (1, 1, 64, 3, 1, [576, 4, 128, 4]),
    (3, 5, 64, 40, 7, [512, 4, 256, 4, 64]),
    (2, 4, 1, 30, 5, [8, 3]),              # pages of one token: never a partial one; odd widths
    (4, 9, 33, 60, 20, [577, 1]),          # odd pages and widths: bytes
    (5, 40, 16, 9000, 1100, [576, 4]),     # more children than a planning workgroup's threads, pages past its block
    (2, 3, 64, 6, 9, [576]),               # the pool runs out
])
def test_fork(B, mp, ps, pages, n, widths):
    say("fork", B, mp, ps, pages, n)
    g, ref, table, lens = make_pool(B, mp, ps, pages, seed=n)
    parents = torch.randint(-1, B + 1, (n,), generator=g).to(torch.int32)  # some are no rows
    check_fork(ref, table, lens, parents, make_caches(pages * ps, widths, g), ps)


def test_fork_empty_whole_and_full_pool():
    say("fork empty / whole pages / no page free")
    g, ref, table, lens = make_pool(3, 4, 8, 20, 1, lens=[0, 16, 13])
    caches = make_caches(160, [16], g)
    _, child, pages = check_fork(ref, table, lens, torch.tensor([0, 1, 2], dtype=torch.int32), caches, 8)
    assert pages.tolist()[:2] == [0, 0] and int(pages[2]) > 0 and not child[0].any()
    ref[1:] = ref[1:].clamp(min=1)  # no page free: whole pages still fork
    _, child, pages = check_fork(ref, table, lens, torch.tensor([2, 1, 2], dtype=torch.int32), caches, 8)
    assert pages.tolist() == [-1, 0, -1] and not child[0].any()


def test_no_children_and_no_caches():
    g, ref, table, lens = make_pool(2, 3, 8, 12, 2)
    gr = ref.cuda()
    child, pages = dsa_pages.fork(gr, table.cuda(), lens.cuda(), torch.zeros(0, dtype=torch.int32).cuda(), [], 8)
    assert child.shape == (0, 3) and pages.numel() == 0 and torch.equal(gr.cpu(), ref)
    check_fork(ref, table, lens, torch.tensor([1, 0], dtype=torch.int32), [], 8)  # the tables alone


@pytest.mark.parametrize("same", [1, 3])
def test_release(same):
    """Rows given once, and given more often than their pages are held (counts end at 0)."""
    say("release", same)
    g, ref, table, lens = make_pool(4, 6, 16, 30, 5)
    table[3, 5] = 31  # no page of the pool
    gr = ref.cuda()
    rep = table.repeat(same, 1)
    dsa_pages.release(gr, rep.cuda(), lens.repeat(same).cuda(), 16)
    want = ref.clone()
    for b in range(4):
        for c in range(-(-int(lens[b]) // 16)):
            if 0 < table[b, c] < 30:
                want[table[b, c]] = max(0, int(want[table[b, c]]) - same)
    assert torch.equal(gr.cpu(), want)
    dsa_pages.release(gr, rep[:0].cuda(), lens[:0].cuda(), 16)
    assert torch.equal(gr.cpu(), want)


def check_compact(ref, table, caches, ps):
    want = compact_ref(ref, table, caches, ps)
    gc = [c.cuda() for c in caches]
    gr, gt = ref.cuda(), table.cuda()
    got = dsa_pages.compact(gr, gt, gc, ps)
    assert torch.equal(gr.cpu(), ref) and torch.equal(gt.cpu(), table)  # not changed
    for a, b in zip(got, want[:3]):
        assert torch.equal(a.cpu(), b)
    for i, (a, b) in enumerate(zip(gc, want[3])):
        assert torch.equal(a.cpu(), b), f"cache {i}"


@pytest.mark.parametrize("pages,live", [(2, 1), (2, 0), (5, 4), (65, 30), (4096, 2000), (4097, 4096), (9001, 5000),
                                        (9001, 300), (8193, 8000)])
def test_compact(pages, live):
    say("compact", pages, live)
    g = torch.Generator().manual_seed(pages + live)
    ref = torch.zeros(pages, dtype=torch.int32)
    ref[torch.randperm(pages - 1, generator=g)[:live] + 1] = torch.randint(1, 5, (live,), generator=g).to(torch.int32)
    table = torch.randint(0, pages, (3, 50), generator=g).to(torch.int32)  # free pages among them
    check_compact(ref, table, make_caches(pages * 4, [24, 4], g), 4)


def test_compact_whole_pages_and_odd_places():
    say("compact, latent pages and a cache that starts at an odd byte")
    g = torch.Generator().manual_seed(4)
    ref = (torch.rand(70, generator=g) < 0.5).to(torch.int32)
    ref[0] = 0
    table = torch.randint(0, 70, (2, 9), generator=g).to(torch.int32)
    caches = make_caches(70 * 64, [576, 512], g)
    want = compact_ref(ref, table, caches, 64)
    buf = torch.zeros(70 * 64 * 512 + 3, dtype=torch.uint8, device="cuda")
    odd = buf[3:].view(70 * 64, 512)
    odd.copy_(caches[1])
    gc = [caches[0].cuda(), odd]
    dsa_pages.compact(ref.cuda(), table.cuda(), gc, 64)
    assert torch.equal(gc[0].cpu(), want[3][0]) and torch.equal(odd.cpu(), want[3][1])
    assert not buf[:3].any()


def test_more_caches_than_a_launch_takes():
    say("150 caches: fork, compact, copy")
    g, ref, table, lens = make_pool(3, 4, 8, 30, 9)
    caches = make_caches(240, [16 + i % 5 for i in range(150)], g)
    check_fork(ref, table, lens, torch.tensor([0, 1, 2, 1], dtype=torch.int32), caches, 8)
    check_compact(ref, table, caches, 8)
    gc = [c.cuda() for c in caches]
    src, dst = torch.tensor([3, 4, 29, 5, 7, 8]), torch.tensor([10, 0, 11, 30, 7, -1])  # four pairs are skipped
    dsa_pages.copy(gc, src.cuda(), dst.cuda(), 8)
    for c, got in zip(caches, gc):
        c[80:88], c[88:96] = c[24:32].clone(), c[232:240].clone()
        assert torch.equal(got.cpu(), c)


def test_copy_refuses_shapes():
    c = torch.zeros(32, 4, device="cuda")
    i = torch.zeros(2, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        dsa_pages.copy([c], i, i[:1], 8)
    with pytest.raises(ValueError):
        dsa_pages.copy([c, c[:24]], i, i, 8)
    with pytest.raises(ValueError):
        dsa_pages.fork(i, torch.zeros(1, 2, dtype=torch.int32, device="cuda"), i, i, [], 8)  # ctx_len of another length


def test_captured_and_replayed():
    """Fork, release and compact in one graph, replayed on changed state, against the host's loops each time."""
    say("pages in a graph")
    ps, pages = 16, 200
    g, ref, table, lens = make_pool(4, 8, ps, pages, 11)
    caches = make_caches(pages * ps, [576, 4], g)
    gr, gt, gl = ref.cuda(), table.cuda(), lens.cuda()
    gp = torch.tensor([0, 3, 2], dtype=torch.int32, device="cuda")
    gc = [c.cuda() for c in caches]
    ws = torch.empty(1 << 16, dtype=torch.uint8, device="cuda")

    def step():
        child, new = dsa_pages.fork(gr, gt, gl, gp, gc, ps, workspace=ws)
        dsa_pages.release(gr, gt[1:2], gl[1:2], ps)
        return (child, new) + dsa_pages.compact(gr, gt, gc, ps, workspace=ws)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in range(3):
        _, ref, table, lens = make_pool(4, 8, ps, pages, 20 + seed)
        parents = torch.randint(0, 4, (3,), generator=g).to(torch.int32)
        gr.copy_(ref), gt.copy_(table), gl.copy_(lens), gp.copy_(parents)
        for a, b in zip(gc, caches):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        child, new, r, cs = fork_ref(ref, table, lens, parents, caches, ps)
        for c in range(-(-int(lens[1]) // ps)):
            r[table[1, c]] -= 1
        t2, r2, remap, cs = compact_ref(r, table, cs, ps)
        for a, b in zip(outs, (child, new, t2, r2, remap)):
            assert torch.equal(a.cpu(), b)
        for a, b in zip(gc, cs):
            assert torch.equal(a.cpu(), b)


def test_fork_free_counts_below_zero():
    """A count of 0 or less is free: the page that a child gets from it is counted once, and not given out again."""
    say("fork, counts below zero")
    ps = 8
    ref = torch.tensor([0, 1, 1, -2, 0, -1, 1, -7, -(2 ** 31)], dtype=torch.int32, device="cuda")
    table = torch.tensor([[1, 2, 0], [6, 0, 0]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([11, 8], dtype=torch.int32, device="cuda")  # a whole page and a part, a whole page
    parents = torch.tensor([0, 1, 0, 0], dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(2)
    cache = torch.randint(0, 256, (9 * ps, 16), dtype=torch.uint8, generator=g)
    got = cache.cuda()
    child, pages = dsa_pages.fork(ref, table, lens, parents, [got], ps)
    assert pages.tolist() == [3, 0, 4, 5] and child.tolist() == [[1, 3, 0], [6, 0, 0], [1, 4, 0], [1, 5, 0]]
    assert ref.tolist() == [0, 4, 1, 1, 1, 1, 2, -7, -(2 ** 31)]
    child, pages = dsa_pages.fork(ref, table, lens, parents, [got], ps)  # two free pages are left for three
    assert pages.tolist() == [7, 0, 8, -1] and child.tolist() == [[1, 7, 0], [6, 0, 0], [1, 8, 0], [0, 0, 0]]
    assert ref.tolist() == [0, 6, 1, 1, 1, 1, 3, 1, 1]
    for p in (3, 4, 5, 7, 8):
        cache[p * ps:(p + 1) * ps] = cache[2 * ps:3 * ps]
    assert torch.equal(got.cpu(), cache)


def test_fork_of_an_empty_table():
    """No rows: no children, or children whose parents are no rows."""
    say("fork of an empty table")
    ref = torch.tensor([0, 1, 0, 2], dtype=torch.int32, device="cuda")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    table, cache = torch.zeros(0, 3, dtype=torch.int32, device="cuda"), torch.ones(32, 4, device="cuda")
    child, pages = dsa_pages.fork(ref, table, none, none, [cache], 8)
    assert child.shape == (0, 3) and pages.shape == (0,)
    child, pages = dsa_pages.fork(ref, table, none, torch.tensor([0, -1], dtype=torch.int32, device="cuda"), [cache], 8)
    assert pages.tolist() == [-1, -1] and child.tolist() == [[0, 0, 0]] * 2
    assert ref.tolist() == [0, 1, 0, 2] and (cache == 1).all()
    with pytest.raises(ValueError):
        dsa_pages.fork(ref, table[:, :0], none, none, [cache], 8)


@pytest.mark.parametrize("pages,live", [(16384, 8200), (16385, 8192), (16385, 16384), (20481, 4095), (20481, 4096), (20481, 4097),
                                        (20481, 12288), (40000, 3), (40000, 20000), (40000, 24576), (40000, 39998)])
def test_compact_large_pools(pages, live):
    """Pools up to and past the 16,384 pages for which each planning workgroup counts all of them, with the live pages' number
    on and beside multiples of a workgroup's 4,096."""
    say("compact a large pool", pages, live)
    g = torch.Generator().manual_seed(pages + live)
    ref = torch.zeros(pages, dtype=torch.int32)
    ref[torch.randperm(pages - 1, generator=g)[:live] + 1] = torch.randint(1, 5, (live,), generator=g).to(torch.int32)
    table = torch.randint(0, pages, (5, 300), generator=g).to(torch.int32)
    check_compact(ref, table, make_caches(pages * 2, [8, 4], g), 2)
