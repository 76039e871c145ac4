"""Bounds of pages, the choice of those that a query attends to, and the attention over
them.  Bounds and choices are exact: they are compared for equality."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
KINDS = [("bf16", False), ("f16", False), ("f32", False), ("bf16", True), ("f16", True)]
GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)


@pytest.fixture(scope="module")
def kv(rans):
    import kv_cache
    return kv_cache


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make(kv, dtype, mx, dim, page, heads, pages, seed=0, track=False):
    g = gen(seed)
    c = kv.PagedCache.allocate(pages, heads, dim, page, DTYPES[dtype], mx, track, bounds=True)
    for t, s in ((c.k, c.k_scale), (c.v, c.v_scale)):
        if mx:
            t.copy_(torch.randint(0, 256, t.shape, device="cuda", generator=g))
            s.copy_(torch.randint(122, 130, s.shape, device="cuda", generator=g))
        else:
            t.copy_(torch.randn(t.shape, device="cuda", generator=g))
    return c


def keys(c):
    """Keys of a whole cache in f64 on the CPU."""
    x = c.k.cpu()
    if not c.mx:
        return x.double()
    x, s = x.numpy(), c.k_scale.cpu().numpy().astype(np.int64)
    code = np.stack((x & 15, x >> 4), -1).reshape(*x.shape[:-1], -1)
    power = np.where(s == 255, np.nan, np.ldexp(1.0, (s - 127).astype(np.int32)))
    return torch.from_numpy(np.where(code & 8, -1, 1) * GRID[code & 7] * power.repeat(32, -1))


def plain_bounds(k):
    low, high = k.amin(2), k.amax(2)
    bad = ~torch.isfinite(k).all(2)
    low[bad] = high[bad] = math.nan
    return torch.stack((low, high), 2)


@pytest.mark.parametrize("dtype,mx", KINDS)
@pytest.mark.parametrize("dim,page,heads,pages", [(64, 16, 1, 40), (96, 32, 3, 9), (128, 64, 2, 17), (192, 256, 2, 5),
                                                  (256, 128, 1, 21), (128, 16, 5, 70)])
def test_bound(kv, dtype, mx, dim, page, heads, pages):
    """Of some pages, in any order, one of them twice, among numbers that are none: the
    others keep theirs."""
    c = make(kv, dtype, mx, dim, page, heads, pages, dim)
    c.bounds.fill_(7.0)
    order = torch.randperm(pages, device="cuda", generator=gen(1)).int()[:pages - 2]
    listed = torch.cat((order, order[:1], torch.tensor([-1, pages, -2 ** 31, 2 ** 31 - 1], dtype=torch.int32,
                                                       device="cuda")))
    listed = listed[torch.randperm(len(listed), device="cuda", generator=gen(2))]
    c.bound(listed)
    want = torch.full(c.bounds.shape, 7.0, dtype=torch.float64)
    at = order.long().cpu()
    want[at] = plain_bounds(keys(c))[at]
    assert torch.equal(c.bounds.double().cpu(), want)
    again = c.bounds.clone()
    c.bound(listed.view(-1, 1).expand(-1, 3).contiguous())  # a table
    assert torch.equal(c.bounds, again)
    c.bound(listed[:0])


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_bounds_at_the_edges(kv, dtype):
    """Zeros of both signs, subnormals, the largest values, and a column with a key that
    is not finite; all places of a page count."""
    t = DTYPES[dtype]
    info = torch.finfo(t)
    c = make(kv, dtype, False, 64, 16, 2, 6)
    c.k.zero_()
    step = 2.0 ** -24 if dtype == "f16" else info.tiny
    for p in range(16):
        c.k[0, 0, p, 0] = (-1) ** p * 0.0
        c.k[0, 0, p, 1] = info.max if p == 15 else -info.max
        c.k[0, 0, p, 2] = step * (p + 1)
        c.k[0, 0, p, 3] = -step * (p + 1)
    c.k[1, 1, 3, 5], c.k[1, 1, 0, 6], c.k[1, 1, 15, 7], c.k[1, 1, 9, 8] = math.inf, -math.inf, math.nan, -math.nan
    c.bound(torch.arange(6, dtype=torch.int32, device="cuda"))
    got, want = c.bounds.double().cpu(), plain_bounds(keys(c))
    assert torch.equal(torch.nan_to_num(got, 1e300), torch.nan_to_num(want, 1e300))
    assert torch.isnan(got).sum() == 8 and torch.isnan(got[1, 1, :, 5:9]).all()


def test_4_bit_blocks_that_are_nan(kv):
    c = make(kv, "bf16", True, 64, 16, 2, 3)
    c.k_scale[1, 0, 7, 1] = 255
    c.k_scale[2, 1, 0, 0] = 0  # the smallest scale
    c.bound(torch.arange(3, dtype=torch.int32, device="cuda"))
    got = c.bounds.double().cpu()
    want = plain_bounds(keys(c))
    # what lies below bf16's smallest step rounds to it
    assert torch.isnan(got[1, 0, :, 32:]).all() and torch.isnan(got).sum() == 64
    want = want.bfloat16().double()
    assert torch.equal(torch.nan_to_num(got, 1e300), torch.nan_to_num(want, 1e300))


# --------------------------------------------------------------------- select
def plain_select(c, q, table, lengths, count, first, last):
    """One sequence, kv head and page after the other, in f64."""
    bounds, q, table = c.bounds.double().cpu().numpy(), q.double().cpu().numpy(), table.cpu().numpy()
    group, page, width = q.shape[1] // c.kv_heads, c.page_size, table.shape[1]
    count = min(count, max(width, 1))
    chosen, held = np.full((len(q), c.kv_heads, count), -1, np.int64), np.zeros((len(q), c.kv_heads), np.int64)
    for b, n in enumerate(lengths.cpu().numpy().tolist()):
        n = min(max(n, 0), width * page)
        pages = -(-n // page)
        known = (table[b, :pages] >= 0) & (table[b, :pages] < c.pages)
        rows = np.where(known, table[b, :pages], 0)
        for h in range(c.kv_heads):
            pick = np.arange(pages)
            if pages > count:
                low, high = bounds[rows, h, 0], bounds[rows, h, 1]
                with np.errstate(invalid="ignore"):
                    each = [np.maximum(x * low, x * high).sum(1) for x in q[b, h * group:(h + 1) * group]]
                score = np.max(each, 0)  # NaN where one is
                score[np.isnan(score)] = math.inf
                forced = (pick < first) | (pick >= pages - last)
                order = np.lexsort((pick, -score, ~known, ~forced))
                pick = np.sort(order[:count])
            chosen[b, h, :len(pick)] = np.where(known[pick], rows[pick] * c.kv_heads + h, -1)
            if pages:
                held[b, h] = (len(pick) - 1) * page + n - (pages - 1) * page
    return chosen.reshape(-1, count), held.reshape(-1)


def tables(lengths, page, pages, seed=0, more=0):
    order = np.random.default_rng(seed).permutation(pages)
    t = np.full((len(lengths), max(-(-max(n, 0) // page) for n in lengths) + more), -1, np.int32)
    at = 0
    for row, n in zip(t, lengths):
        need = -(-max(n, 0) // page)
        row[:need] = order[at:at + need]
        at += need
    assert at <= pages
    return torch.from_numpy(t).cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda")


def compare(c, q, table, lengths, count, first, last):
    chosen, held = c.select(q, table, lengths, count, first, last)
    want, tokens = plain_select(c, q, table, lengths, count, first, last)
    assert held.tolist() == tokens.tolist()
    assert chosen.dtype is torch.int32 and np.array_equal(chosen.cpu().numpy(), want)
    return chosen, held


SELECTIONS = [  # dim, page, heads, group, lengths, more, count, first, last
    (128, 64, 2, 6, [4000], 0, 7, 1, 2), (64, 16, 1, 1, [1, 0, 16, 17, 160, 161], 3, 4, 0, 1),
    (96, 16, 3, 2, [700, 699, 5, 0, 333], 0, 9, 2, 3), (128, 16, 2, 5, [16000, 9000], 1, 64, 1, 1),
    (256, 32, 1, 8, [3000, 2999], 0, 3, 1, 2), (192, 64, 2, 17, [5000], 0, 20, 0, 20),
    (128, 128, 4, 40, [2000, 100], 0, 6, 5, 1), (64, 256, 5, 7, [9999, 256, 257, 512], 2, 3, 0, 1),
    (64, 16, 1, 3, [140000], 0, 100, 1, 1), (64, 16, 2, 1, [8192 * 16 + 5, 40], 5, 5000, 1, 1),
    (128, 16, 2, 2, [50, 60], 0, 9, 1, 1),
    # tables around those whose pages are scored where they are chosen from
    (64, 16, 2, 7, [16 * 192, 16 * 191 - 1, 40], 0, 37, 0, 1), (64, 16, 1, 8, [16 * 193], 0, 37, 3, 4),
    (64, 16, 1, 9, [16 * 192], 0, 100, 1, 1), (96, 16, 3, 5, [16 * 96, 16 * 95], 0, 95, 1, 1),
    (128, 16, 2, 8, [16 * 97, 5], 0, 7, 2, 2), (128, 32, 2, 1, [32 * 33, 32 * 65, 32 * 9], 31, 8, 1, 7),
    (192, 16, 2, 3, [16 * 48, 16 * 33, 1], 0, 17, 0, 2), (256, 16, 1, 8, [16 * 48 - 3], 0, 47, 0, 1),
    (256, 16, 1, 2, [16 * 49], 0, 2, 1, 1),
]


@pytest.mark.parametrize("dim,page,heads,group,lengths,more,count,first,last", SELECTIONS)
@pytest.mark.parametrize("dtype,mx", [("bf16", False), ("f32", False), ("f16", True)])
def test_select(kv, dtype, mx, dim, page, heads, group, lengths, more, count, first, last):
    count = max(count, first + last)
    pages = sum(-(-n // page) for n in lengths) + 2
    c = make(kv, dtype, mx, dim, page, heads, pages, 5)
    c.bound(torch.arange(pages, dtype=torch.int32, device="cuda"))
    table, n = tables(lengths, page, pages, 1, more)
    q = torch.randn(len(lengths), heads * group, dim, device="cuda", generator=gen(3)).to(DTYPES[dtype])
    compare(c, q, table, n, count, first, last)


def test_ties_and_order(kv):
    """Whole numbers, whose scores are exact: many tie, and the lower index goes first;
    counts around where ties begin and end."""
    c = make(kv, "bf16", False, 64, 16, 2, 300)
    c.k.copy_(torch.randint(-1, 2, (300, 2, 1, 64), device="cuda", generator=gen(1)).expand(300, 2, 16, 64))
    c.k[:, :, :, 3:] = 0
    c.bound(torch.arange(300, dtype=torch.int32, device="cuda"))
    table, n = tables([16 * 290 - 3], 16, 300)
    q = torch.zeros(1, 4, 64, device="cuda", dtype=torch.bfloat16)
    q[0, :, :3] = torch.tensor([[1.0, 2, 0], [0, -1, 1], [3, 0, 0], [-1, 0, 0]], device="cuda").bfloat16()
    for count in list(range(1, 40)) + [100, 288, 289, 290, 291]:
        compare(c, q, table, n, count, 0, 1)
    q.zero_()  # all scores alike
    for count in (1, 2, 17, 289):
        compare(c, q, table, n, count, 0, 1)


def test_scores_over_the_whole_range(kv):
    """Magnitudes from f32's smallest to its largest, which sums in 32 bits lose."""
    c = make(kv, "f32", False, 64, 16, 1, 200)
    scale = torch.exp2(torch.randint(-126, 127, (200, 1, 1, 1), device="cuda", generator=gen(2)).float())
    c.k.copy_(torch.randn(200, 1, 16, 64, device="cuda", generator=gen(3)).clamp(-1.9, 1.9) * scale)
    c.bound(torch.arange(200, dtype=torch.int32, device="cuda"))
    table, n = tables([16 * 197], 16, 200)
    q = torch.randn(1, 3, 64, device="cuda", generator=gen(4)) * 2.0 ** 100
    for count in (2, 50, 150):
        compare(c, q, table, n, count, 1, 1)


def test_pages_that_are_none_and_keys_that_are_not_finite(kv):
    """Entries without a page are chosen last, pages with keys that are not finite
    first, by index; those at the ends always."""
    c = make(kv, "bf16", False, 64, 16, 2, 90)
    c.k[20, 1, 3, 7], c.k[50, 0, 0, 0], c.k[51, 0, 15, 63], c.k[52, 0, 2, 2] = math.nan, math.inf, -math.inf, math.nan
    c.bound(torch.arange(90, dtype=torch.int32, device="cuda"))
    table = torch.arange(80, dtype=torch.int32, device="cuda")[None].repeat(3, 1)
    table[0, 30:70] = -1
    table[1, ::2] = 90
    table[1, 79] = -5
    table[2, :] = -1
    n = torch.full((3,), 80 * 16 - 7, dtype=torch.int32, device="cuda")
    q = torch.randn(3, 4, 64, device="cuda", generator=gen(4)).bfloat16()
    more = torch.cat((table, torch.full((3, 200), -1, dtype=torch.int32, device="cuda")), 1)  # scored apart
    many = torch.randn(3, 2 * 11, 64, device="cuda", generator=gen(5)).bfloat16()  # by the matrix cores
    for count in (2, 3, 5, 30, 39, 41, 60, 79):
        compare(c, q, table, n, count, 1, 1)
        compare(c, q, more, n, count, 1, 1)
        compare(c, many, table, n, count, 1, 1)
    c.bounds.fill_(math.nan)  # none has been made: by index
    compare(c, q, table, n, 9, 0, 2)


def test_lengths_out_of_range(kv):
    c = make(kv, "bf16", False, 64, 16, 2, 40)
    c.bound(torch.arange(40, dtype=torch.int32, device="cuda"))
    table = torch.arange(40, dtype=torch.int32, device="cuda").view(4, 10)
    n = torch.tensor([-3, 10 ** 9, 0, -2 ** 31], dtype=torch.int32, device="cuda")
    q = torch.randn(4, 2, 64, device="cuda", generator=gen(4)).bfloat16()
    compare(c, q, table, n, 4, 1, 1)
    compare(c, q, table, n, 10, 1, 1)
    compare(c, q, table, n, 99, 1, 1)
    chosen, held = c.select(q, table[:, :0], n, 4)
    assert chosen.tolist() == [[-1]] * 8 and held.tolist() == [0] * 8
    none = c.select(q[:0], table[:0], n[:0], 4)
    assert none[0].shape == (0, 4) and none[1].shape == (0,)


# --------------------------------------------------------- attention over them
@pytest.mark.parametrize("dtype,mx", KINDS)
@pytest.mark.parametrize("dim,page,heads,group,count,track", [(64, 16, 2, 3, 5, True), (128, 64, 3, 6, 4, False),
                                                              (96, 32, 1, 20, 7, True)])
def test_attend_selected(kv, dtype, mx, dim, page, heads, group, count, track):
    """Bit for bit attention over a cache that holds the chosen pages alone, and weights
    that are added to the same tokens."""
    lengths = [1000, 0, 3, 777, page * count, page * count + 1]
    pages = sum(-(-n // page) for n in lengths) + 1
    c = make(kv, dtype, mx, dim, page, heads, pages, 7, track)
    c.bound(torch.arange(pages, dtype=torch.int32, device="cuda"))
    table, n = tables(lengths, page, pages, 2)
    table[3, 1] = -1
    wide = torch.randn(len(lengths), heads * group + 2, dim, device="cuda", generator=gen(8)).to(DTYPES[dtype])
    q = wide[:, 1:-1]  # columns of a projection
    if track:
        c.mass.fill_(0.5)
    chosen, held = compare(c, q, table, n, count, 1, 1)
    out = c.attend_selected(q, chosen, held, 0.2)
    rows = len(chosen)
    at = chosen.long().clamp(min=0).flatten()
    parts = [None if t is None else t.reshape(-1, 1, page, t.shape[3])[at].contiguous()
             for t in (c.k, c.v, c.k_scale, c.v_scale)]
    more = [None, None] if not track else [torch.zeros(len(at), 1, page, device="cuda"),
                                           torch.zeros(len(at), 1, page, dtype=torch.int32, device="cuda")]
    alone = kv.PagedCache(parts[0], parts[1], DTYPES[dtype], parts[2], parts[3], *more)
    own = torch.arange(len(at), dtype=torch.int32, device="cuda").view(rows, -1)
    own = torch.where(chosen >= 0, own, -1)
    want = alone.attend(q.reshape(rows, group, dim), own, held, 0.2).view(len(lengths), heads * group, dim)
    assert torch.equal(out, want) and (out[1] == 0).all() and torch.isfinite(out).all()
    if track:  # one addition a token and call
        mass = torch.full_like(c.mass, 0.5).view(-1, page)
        used = chosen.flatten() >= 0
        mass[at[used]] += alone.mass.view(-1, page)[used]
        assert torch.equal(c.mass.view(-1, page), mass)


def test_all_pages_are_attention_over_all(kv):
    """With as many pages as there are, what attend gives, to the rounding of sums in
    another order: 2^-8 of the output in bf16 and 2^-17 of the largest value before."""
    c = make(kv, "bf16", False, 128, 64, 2, 60, 3)
    table, n = tables([3000, 500], 64, 60)
    q = torch.randn(2, 12, 128, device="cuda", generator=gen(9)).bfloat16()
    chosen, held = c.select(q, table, n, 47)
    got, want = c.attend_selected(q, chosen, held).double(), c.attend(q, table, n).double()
    assert ((got - want).abs() <= 2.0 ** -7 * want.abs() + 2.0 ** -16 * 5).all()


def test_offsets_beyond_32_bits(kv):
    """Pages whose keys lie behind 2^32 bytes."""
    c = kv.PagedCache.allocate(20000, 8, 128, 128, torch.bfloat16, bounds=True)  # 5.2 GB of keys
    k = torch.randn(3, 8, 128, 128, device="cuda", generator=gen(1)).bfloat16()
    at = torch.tensor([19999, 0, 17001], dtype=torch.int32, device="cuda")
    c.k[at.long()] = k
    c.bound(at)
    assert torch.equal(c.bounds[at.long()], torch.stack((k.amin(2), k.amax(2)), 2))
    assert c.bounds.count_nonzero() == 3 * 8 * 2 * 128
    q = torch.randn(1, 8, 128, device="cuda", generator=gen(2)).bfloat16()
    compare(c, q, at[None], torch.tensor([300], dtype=torch.int32, device="cuda"), 2, 0, 1)


def test_in_a_graph_and_on_another_stream(kv):
    c = make(kv, "bf16", False, 128, 64, 2, 64)
    table, n = tables([2000, 1500], 64, 64)
    q = torch.randn(2, 12, 128, device="cuda", generator=gen(1)).bfloat16()
    pages = torch.arange(64, dtype=torch.int32, device="cuda")

    def step():
        c.bound(pages)
        chosen, held = c.select(q, table, n, 9)
        return chosen, held, c.attend_selected(q, chosen, held)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        c.k.copy_(torch.randn(c.k.shape, device="cuda", generator=gen(i)))
        q.copy_(torch.randn(q.shape, device="cuda", generator=gen(i + 10)))
        n.copy_(torch.tensor([2000 - 300 * i, 100 + 700 * i], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got_now = [t.clone() for t in got]
        c.bounds.zero_()
        for x, y in zip(got_now, step()):
            assert torch.equal(x, y)
        compare(c, q, table, n, 9, 1, 1)


def test_refusals(kv):
    c, plain = make(kv, "bf16", False, 64, 16, 2, 8), kv.PagedCache.allocate(8, 2, 64, 16)
    table, n = torch.zeros(3, 4, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16, device="cuda")
    for call in (lambda: plain.bound(n), lambda: plain.select(q, table, n, 2), lambda: c.bound(n.long()),
                 lambda: c.bound(n.cpu()), lambda: c.bound(table[:, :2]), lambda: c.select(q[:, :3], table, n, 2),
                 lambda: c.select(q[:2], table, n, 2), lambda: c.select(q.float(), table, n, 2),
                 lambda: c.select(q, table.long(), n, 2), lambda: c.select(q, table, n[:2], 2),
                 lambda: c.select(q, table, n, 1), lambda: c.select(q, table, n, 3, first=-1),
                 lambda: c.select(q, table, n, 3, last=0), lambda: c.select(q, table, n, 2 ** 31),
                 lambda: c.select(q.requires_grad_(), table, n, 2)):
        with pytest.raises(ValueError):
            call()
    q = q.detach()
    chosen, held = c.select(q, table, n, 2)
    for call in (lambda: c.attend_selected(q, chosen, held, -1.0), lambda: c.attend_selected(q, chosen, held, 0.0),
                 lambda: c.attend_selected(q[:2], chosen, held), lambda: c.attend_selected(q[:, :3], chosen, held),
                 lambda: c.attend_selected(q, chosen.long(), held), lambda: c.attend_selected(q, chosen, held, track=True)):
        with pytest.raises(ValueError):
            call()
    one = make(kv, "bf16", False, 64, 16, 1, 8)
    assert one.heads.kv_heads == 1 and one.heads.pages == 8 and one.heads.k.data_ptr() == one.k.data_ptr()
    for bad in (torch.zeros(8, 2, 2, 64), torch.zeros(8, 2, 2, 64, device="cuda"),
                torch.zeros(8, 2, 64, dtype=torch.bfloat16, device="cuda")):
        with pytest.raises(ValueError):
            kv.PagedCache(plain.k, plain.v, bounds=bad)
