"""Pages of a cache of states on the GPU, against the same bookkeeping in Python."""
from __future__ import annotations

import random

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def make_pools(P, seed):
    """Pools of several types and page sizes, one of them a slice of a larger tensor."""
    gen = torch.Generator().manual_seed(seed)
    wide = torch.randn(P, 2, 3, 64, generator=gen).to(DEV)
    return [torch.randn(P, 2, 64, 70, generator=gen).to(DEV), wide[:, 1],
            torch.randint(0, 255, (P, 16), generator=gen, dtype=torch.uint8).to(DEV),
            torch.randn(P, 8, generator=gen).to(torch.float16).to(DEV)]


def copies(pools):
    return [p.clone() for p in pools]


def same(pools, want):
    return all(torch.equal(a, b) for a, b in zip(pools, want))


@pytest.mark.parametrize("P,n", [(2, 1), (40, 17), (1500, 700), (2049, 5), (5000, 2300)])
def test_copy(pkg, P, n):
    pools = make_pools(P, P)
    want = copies(pools)
    order = random.Random(P).sample(range(P), 2 * n)
    src, dst = order[:n], order[n:]
    if n > 3:
        src[2], dst[3] = -1, -7      # skipped
        src[0], dst[0] = src[1], dst[0]  # one source twice
    for p in want:
        for a, b in zip(src, dst):
            if a >= 0 and b >= 0:
                p[b] = p[a]
    pkg.pages_copy(pools, i32(src), i32(dst), check=True)
    assert same(pools, want)


def test_copy_leaves_out_what_depends_on_order(pkg):
    pools = make_pools(10, 1)
    want = copies(pools)
    #      fine, twice, twice, chain, chain's source fine, outside, outside, itself, fine
    src = [0, 1, 2, 3, 4, 10, 5, 6, 0]
    dst = [9, 8, 8, 4, 7, 5, 99, 6, 3]
    # 3 -> 4 is left out (4 is a source), 0 -> 3 too (3 is a source)
    for p in want:
        p[9], p[7] = p[0].clone(), p[4].clone()
    with pytest.raises(pkg.GDNError, match="index"):
        pkg.pages_copy(pools, i32(src), i32(dst), check=True)
    assert same(pools, want)


@pytest.mark.parametrize("P,n", [(1, 0), (9, 3), (50, 30), (3000, 1300)])
def test_fork_and_alloc(pkg, P, n):
    rng = random.Random(P)
    pools = make_pools(P, P + 1)
    want = copies(pools)
    used = [rng.randrange(0, 3) % 2 for _ in range(P)]
    used[0] = 1
    alive = [p for p in range(P) if used[p]]
    src = [rng.choice(alive) if rng.random() < 0.9 else -1 for _ in range(n)]
    u, dst, full = list(used), [], False
    for s in src:
        if s < 0:
            dst.append(-1)
        elif 0 in u:
            d = u.index(0)
            u[d] = 1
            dst.append(d)
            for p in want:
                p[d] = p[s]
        else:
            dst.append(-1)
            full = True
    flags, flags_out = i32(used), torch.full((P,), -9, dtype=torch.int32, device=DEV)
    out = torch.full((n,), -9, dtype=torch.int32, device=DEV)
    call = lambda: pkg.pages_fork(pools, flags, i32(src), out=out, used_out=flags_out, check=True)  # noqa: E731
    if full:
        with pytest.raises(pkg.GDNError, match="no free page"):
            call()
    else:
        assert call() is out
    assert out.tolist() == dst and flags_out.tolist() == u and flags.tolist() == used
    assert same(pools, want)
    k = min(2, u.count(0))
    got = pkg.pages_alloc(flags_out, k, check=True)
    assert got.tolist() == [p for p in range(P) if not u[p]][:k]
    assert flags_out.sum().item() == sum(u) + k


def test_fork_reports_free_and_outside_sources(pkg):
    pools = make_pools(6, 2)
    want = copies(pools)
    used = i32([1, 0, 1, 0, 0, 0])
    with pytest.raises(pkg.GDNError, match="index"):
        pkg.pages_fork(pools, used, i32([1, 2, 6, -1, 0]), check=True)
    # only the sound entries took pages
    for p in want:
        p[1], p[3] = p[2].clone(), p[0].clone()
    assert used.tolist() == [1, 1, 1, 1, 0, 0] and same(pools, want)
    got = None
    with pytest.raises(pkg.GDNError, match="no free page"):
        got = pkg.pages_alloc(used, 3, check=True)
    assert got is None and used.tolist() == [1] * 6


def test_free(pkg):
    used = i32([1, 1, 0, 1, 1])
    out = pkg.pages_free(used, i32([3, -1, 0]), check=True)
    assert out is used and used.tolist() == [0, 1, 0, 0, 1]
    for bad in ([0], [5], [1, 1]):
        with pytest.raises(pkg.GDNError, match="index"):
            pkg.pages_free(used.clone(), i32(bad), check=True)
    keep = used.clone()
    other = pkg.pages_free(used, i32([4]), used_out=torch.empty_like(used), check=True)
    assert torch.equal(used, keep) and other.tolist() == [0, 1, 0, 0, 0]
    pkg.pages_free(used, i32([]), check=True)


@pytest.mark.parametrize("P", [1, 2, 31, 64, 1025, 5000])
@pytest.mark.parametrize("share", [0.0, 0.4, 0.9, 1.0])
def test_compact(pkg, P, share):
    rng = random.Random(P)
    used = [int(rng.random() < share) * rng.randrange(1, 5) for _ in range(P)]
    pools = make_pools(P, P)
    want = copies(pools)
    count = sum(u > 0 for u in used)
    remap = [p if u and p < count else -1 for p, u in enumerate(used)]
    holes = iter(p for p in range(count) if not used[p])
    for p in range(count, P):
        if used[p]:
            remap[p] = next(holes)
            for x in want:
                x[remap[p]] = x[p]
    rows = [p for p in range(P) if used[p]][::-1] + [-1]
    flags = i32(used)
    index = i32(rows)
    got, n, where = pkg.pages_compact(pools, flags, index=index, index_out=index, check=True)
    assert where is index and index.tolist() == [remap[p] for p in rows[:-1]] + [-1]
    assert got.tolist() == remap and n.tolist() == [count]
    assert flags.tolist() == [1] * count + [0] * (P - count)
    assert same(pools, want)


def test_compact_reports_rows_of_free_pages(pkg):
    used = i32([0, 1])
    pool = torch.randn(2, 64, device=DEV)
    with pytest.raises(pkg.GDNError, match="index"):
        pkg.pages_compact(pool, used, index=i32([0, 1, 2]), check=True)


def test_serving_turn(pkg):
    """Prompts into pages, forked, decoded, some finished, compacted, decoded as a plain batch, and as GDN states."""
    H, d, io, P = 2, 64, torch.bfloat16, 16
    gen = torch.Generator().manual_seed(3)
    rand = lambda *s: torch.randn(*s, generator=gen).to(io).to(DEV)  # noqa: E731
    pool, used = torch.zeros(P, H, d, d, device=DEV), i32([1, 0] * 8)  # other owners hold the even pages
    pages = pkg.pages_alloc(used, 2)
    T = 150
    q, k, v = rand(1, T, H, d), rand(1, T, H, d), rand(1, T, H, d)
    g = -torch.rand(1, T, H, generator=gen).to(DEV) * 0.1
    cu = i32([0, 90, 150])
    pkg.lin_prefill(q, k, v, g, cu_seqlens=cu, index=pages, final_state=pool)
    kids = pkg.pages_fork(pool, used, pages.repeat_interleave(2))
    rows = torch.cat([pages, kids])
    x = [rand(6, H, d) for _ in range(3)] + [-torch.rand(6, H, generator=gen).to(DEV)]
    plain = pool[rows.long()].clone()
    assert torch.equal(plain[[0, 0, 1, 1]], plain[2:])
    o = pkg.lin_decode(*x, pool, index=rows)
    want = pkg.lin_decode(*x, plain)
    assert torch.equal(o, want) and torch.equal(pool[rows.long()], plain)
    pkg.pages_free(used, torch.cat([i32(list(range(0, P, 2))), rows[2:3]]))
    live = torch.cat([rows[:2], rows[3:]])
    _, count, now = pkg.pages_compact(pool, used, index=live)
    assert count.tolist() == [5] and sorted(now.tolist()) == list(range(5))
    by_page = torch.empty(5, dtype=torch.long, device=DEV)
    by_page[now.long()] = torch.arange(5, device=DEV)  # the row whose state is in page p
    left = plain[[0, 1, 3, 4, 5]][by_page].clone()
    assert torch.equal(pool[:5], left)
    y = [t[:5].clone() for t in x]
    beta = torch.rand(5, H, generator=gen).to(DEV)
    o1, o2 = pkg.lin_decode(*y, pool[:5]), pkg.lin_decode(*y, left)
    assert torch.equal(o1, o2) and torch.equal(pool[:5], left)
    o1, o2 = pkg.gdn_decode(*y, beta, pool[:5]), pkg.gdn_decode(*y, beta, left)
    assert torch.equal(o1, o2) and torch.equal(pool[:5], left)
    pkg.check_device_status(torch.device(DEV))


def test_turn_in_a_graph(pkg):
    P = 40
    pools = make_pools(P, 5)
    begin = copies(pools)
    used0 = i32([1] * 30 + [0] * 10)
    used, done, src = used0.clone(), i32([0, 3, 4, 17]), i32([29, 29, 11])

    def turn():
        pkg.pages_free(used, done)
        kids = pkg.pages_fork(pools, used, src)
        return (kids, *pkg.pages_compact(pools, used, index=kids))

    want = turn()
    end, flags = copies(pools), used.clone()
    for p, b in zip(pools, begin):
        p.copy_(b)
    used.copy_(used0)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = turn()
    for _ in range(2):
        for p, b in zip(pools, begin):
            p.copy_(b)
        used.copy_(used0)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert same(pools, end) and torch.equal(used, flags)
    pkg.check_device_status(torch.device(DEV))


def test_sources_just_behind_the_pool(pkg):
    """Pools that are the front of larger ones: what lies behind is no page, and is neither moved nor needed.
    Entries of one bad source side by side, in both forms of the plan."""
    for P, n in ((10, 8), (2500, 2100)):
        whole = make_pools(P + 4, P)
        want = copies(whole)
        pools = [p[:P] for p in whole]
        src, dst = [P, P, P + 1, 0, 0] + [P] * (n - 5), [1, 2, 3, 4, 4] + list(range(5, n))
        src[5] = 0  # the one sound entry
        for p in want:
            p[5] = p[0]
        with pytest.raises(pkg.GDNError, match="index"):
            pkg.pages_copy(pools, i32(src), i32(dst), check=True)
        assert same(whole, want)
        used = i32([1, 0, 1] + [1] * (P - 4) + [0])
        with pytest.raises(pkg.GDNError, match="index"):
            pkg.pages_fork(pools, used, i32([P, P, 2, 2] + [P + 2] * (n - 4)), check=True)
        for p in want:
            p[1], p[P - 1] = p[2], p[2]
        assert same(whole, want) and used.tolist() == [1] * P


def test_copy_of_a_page_onto_itself_is_no_entry(pkg):
    pools = make_pools(8, 9)
    want = copies(pools)
    for p in want:
        p[5], p[1] = p[3].clone(), p[2].clone()
    pkg.pages_copy(pools, i32([5, 3, 2, 2, 2]), i32([5, 5, 1, 2, 2]), check=True)
    assert same(pools, want)
