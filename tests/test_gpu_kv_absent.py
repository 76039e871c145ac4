"""Eviction where table entries are no page of the cache: tokens without a page
are never kept, places without one never filled, and of the others the best that
there are places for stay, the recent ones first.  Against plain lists."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

BUFFERS = ("k", "v", "k_scale", "v_scale", "mass", "position")


@pytest.fixture(scope="module")
def kv(rans):
    import kv_cache
    return kv_cache


def make(kv, mx, page, heads, pages, seed):
    """A tracked f16 cache of random contents whose masses have many ties."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = kv.PagedCache.allocate(pages, heads, 64, page, torch.float16, mx=mx, track=True)
    for t in (c.k, c.v, c.k_scale, c.v_scale):
        if t is not None and mx:
            t.copy_(torch.randint(0, 250, t.shape, device="cuda", generator=g))
        elif t is not None:
            t.copy_(torch.randn(t.shape, device="cuda", generator=g))
    c.mass.copy_((torch.rand(c.mass.shape, device="cuda", generator=g) * 20).floor() / 4)
    c.position.copy_(torch.randint(0, 1000, c.position.shape, device="cuda", generator=g))
    return c


def moves_of(c, table, lengths, seen, budget, recent, into):
    """New lengths, and (head, page, place, page, place) for every token that
    moves."""
    mass, position, page = c.mass.cpu().numpy().astype(np.float64), c.position.cpu().numpy(), c.page_size
    table, new, moves = table.cpu().numpy(), [], []

    def of(row, j):
        p = int(row[j // page])
        return (p, j % page) if 0 <= p < c.pages else None

    for b, n in enumerate(lengths.tolist()):
        n = min(max(n, 0), table.shape[1] * page)
        tokens = [j for j in range(n) if of(table[b], j)]
        row = table[b] if into is None else into.cpu().numpy()[b]
        places = [j for j in range(min(n, budget)) if of(row, j)]
        kept = min(len(tokens), len(places))
        new.append(min(n, budget))
        if into is not None and kept < len(places):
            new[-1] = places[kept - 1] + 1 if kept else 0
        if into is None and n <= budget:
            continue
        for h in range(c.kv_heads):
            def order(j):
                p, at = of(table[b], j)
                if position[p, h, at] >= int(seen[b]) - recent:
                    return 0, 0.0, j
                m = mass[p, h, at]
                return 1, math.inf if math.isnan(m) else -m, j
            best = sorted(sorted(tokens, key=order)[:kept])
            if into is None:
                to = [j for j in places if j not in set(best)]
                best = [j for j in best if j >= budget]
                assert len(to) == len(best)
            else:
                to = places[:kept]
            moves += [(h, *of(table[b], s), *of(row, d)) for s, d in zip(best, to)]
    return new, moves


def check(c, table, lengths, seen, budget, recent, into=None):
    want = {w: getattr(c, w).clone() for w in BUFFERS if getattr(c, w) is not None}
    new, moves = moves_of(c, table, lengths, seen, budget, recent, into)
    if moves:
        h, p, s, t, d = (torch.from_numpy(x).cuda() for x in np.array(moves, dtype=np.int64).T)
        for w in want:
            want[w][t, h, d] = getattr(c, w)[p, h, s]
    got = c.evict(table, lengths, seen, budget, recent, into)
    assert got.tolist() == new
    for w in want:
        assert torch.equal(getattr(c, w).view(torch.uint8), want[w].view(torch.uint8)), w
    return got


def test_recent_tokens_outlive_an_absent_page(kv):
    """Three pages of 16 and a hole: of 64 indexes 32 are kept, 16 of them
    without a place, and the eight recent tokens are among those that stay."""
    c = make(kv, False, 16, 1, 4, 0)
    table = torch.tensor([[0, -1, 2, 3]], dtype=torch.int32, device="cuda")
    c.mass[:] = torch.tensor([0.1, 9.0, 2.0, 1.0], device="cuda")[:, None, None]
    c.position.copy_(torch.arange(64, device="cuda").view(4, 1, 16))
    n = torch.tensor([64], dtype=torch.int32, device="cuda")
    check(c, table, n, n, 32, 8)
    held = set(c.position[0, 0].tolist())
    assert set(range(56, 64)) < held and held <= set(range(32, 64))


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("other", [False, True], ids=["in place", "into"])
@pytest.mark.parametrize("page", [16, 64])
def test_holes_anywhere(kv, mx, page, other):
    """A share of the table's entries is no page, before and behind the budget,
    all of them and none; so with the table of places."""
    heads, rng = 2, np.random.default_rng(page + mx)
    lengths = [0, 1, page - 1, 5 * page, 5 * page + 3, 9 * page + 7, 20 * page, 20 * page, 20 * page, 12 * page]
    wide = 21
    for budget, recent in ((6 * page, 0), (6 * page + 5, page), (3 * page - 1, 3 * page - 1), (1, 1), (19 * page, 40)):
        c = make(kv, mx, page, heads, 2 * wide * len(lengths), budget)
        order = rng.permutation(c.pages).astype(np.int32)
        table = order[:wide * len(lengths)].reshape(len(lengths), wide).copy()
        holes = rng.random(table.shape) < 0.3
        holes[6] = False
        holes[7] = True
        holes[8, :8] = True
        table[holes] = rng.choice([-1, -9, c.pages, 2 ** 31 - 1], holes.sum())
        into = None
        if other:
            into = order[wide * len(lengths):].reshape(len(lengths), wide).copy()
            holes = rng.random(into.shape) < 0.3
            holes[4:8] = False
            holes[9] = True
            into[holes] = -1
            into = torch.from_numpy(into).cuda()
        n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        seen = torch.full_like(n, 900)
        check(c, torch.from_numpy(table).cuda(), n, seen, budget, recent, into)


@pytest.mark.parametrize("other", [False, True], ids=["in place", "into"])
def test_holes_in_long_sequences(kv, other):
    """Sequences that go through the selection in one piece and in several."""
    page, lengths = 64, [20000, 40000, 70001]
    for budget, recent in ((9000, 500), (39000, 0)):
        need = [-(-n // page) for n in lengths]
        wide, width = -(-budget // page), max(need)
        c = make(kv, True, page, 1, 3 * (width + wide), budget)
        order = torch.randperm(c.pages, generator=torch.Generator().manual_seed(budget)).int()
        table = order[:3 * width].reshape(3, width).clone()
        table[0, 3:9], table[1, ::7], table[2, 100:400] = -1, -1, c.pages
        into = None
        if other:
            into = order[3 * width:].reshape(3, wide).clone()
            into[1, 5], into[2, ::3] = -1, -1
            into = into.cuda()
        n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        check(c, table.cuda(), n, torch.full_like(n, 990), budget, recent, into)


def test_what_was_left_out_stays_out(kv):
    """Attention after an eviction into other pages reads the tokens that there
    were, and nothing that lay in those pages before."""
    c = make(kv, False, 16, 1, 8, 3)
    table = torch.tensor([[0, -1, 2]], dtype=torch.int32, device="cuda")
    into = torch.tensor([[4, 5, 6]], dtype=torch.int32, device="cuda")
    n = torch.tensor([40], dtype=torch.int32, device="cuda")
    q = torch.randn(1, 2, 64, device="cuda").half()
    want = c.attend(q, table, n, track=False)
    c.k[4:7], c.v[4:7] = math.nan, math.nan
    for budget in (40, 48):
        left = c.evict(table, n, n, budget, into=into)
        assert left.tolist() == [24]
        got = c.attend(q, into, left, track=False)
        assert torch.isfinite(got).all()
        assert (got.double() - want.double()).abs().max() <= 2 ** -10 * float(want.abs().max())
