"""The key-value cache's operators on the GPU against plain implementations in
64 bits: lengths from none to many pages, odd groups, strides, absent pages,
masked places that hold anything, ties, values that are not finite, other
streams, graphs and offsets beyond 32 bits."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
UNIT = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}  # half a step of one value


@pytest.fixture(scope="module")
def kv(rans):
    import kv_cache
    return kv_cache


def make(kv, dtype, mx, dim, page, heads, pages, seed=0, track=True):
    """A tracked cache of random contents."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = kv.PagedCache.allocate(pages, heads, dim, page, DTYPES[dtype], mx=mx, track=track)
    for t, s in ((c.k, c.k_scale), (c.v, c.v_scale)):
        if mx:
            t.copy_(torch.randint(0, 256, t.shape, device="cuda", generator=g))
            s.copy_(torch.randint(122, 130, s.shape, device="cuda", generator=g))
        else:
            t.copy_(torch.randn(t.shape, device="cuda", generator=g))
    if track:
        c.mass.copy_(torch.rand(c.mass.shape, device="cuda", generator=g))
    return c


def tables(lengths, page, pages, seed=0, more=0):
    """Pages of each sequence in no order, `more` columns of -1 behind the
    longest."""
    order = np.random.default_rng(seed).permutation(pages)
    width = max(-(-n // page) for n in lengths) + more
    t = np.full((len(lengths), width), -1, np.int32)
    at = 0
    for row, n in zip(t, lengths):
        need = -(-n // page)
        row[:need] = order[at:at + need]
        at += need
    assert at <= pages
    return torch.from_numpy(t).cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda")


GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)


def opened(c, which):
    """Keys or values of a whole cache in f64 on the host."""
    x = getattr(c, which).cpu()
    if not c.mx:
        return x.double().numpy()
    x = x.numpy()
    s = getattr(c, which + "_scale").cpu().numpy().astype(np.int64)
    code = np.stack((x & 15, x >> 4), -1).reshape(*x.shape[:-1], -1)
    power = np.where(s == 255, np.nan, np.ldexp(1.0, (s - 127).astype(np.int32)))
    return np.where(code & 8, -1, 1) * GRID[code & 7] * power.repeat(32, -1)


# ------------------------------------------------------------ append and read
def rounded(x):
    """What 4-bit storage makes of f64 values: the nearest of the grid by
    distance, ties to the even code."""
    y = np.asarray(x, np.float64).reshape(-1, 32)
    out = np.empty_like(y)
    for i, row in enumerate(y):
        if not np.isfinite(row).all():
            out[i] = np.nan
            continue
        most = np.abs(row).max()
        e = -127 if most == 0 else max(math.frexp(most)[1] - 3, -127)
        a = np.abs(row) / 2.0 ** e
        far = np.abs(a[:, None] - GRID)
        near = far == far.min(1, keepdims=True)
        even = near & (np.arange(8) % 2 == 0)
        pick = np.where(even.any(1), even.argmax(1), near.argmax(1))
        out[i] = np.sign(row) * GRID[pick] * 2.0 ** e
    return out.reshape(np.shape(x))


@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("dtype,mx", [("bf16", False), ("f16", False), ("f32", False),
                                      ("bf16", True), ("f16", True)])
def test_append_and_read(kv, dtype, mx, dim):
    heads, page, tokens = 3, 16, 53
    c = make(kv, dtype, mx, dim, page, heads, 9)
    before = [opened(c, w) for w in "kv"]
    mass, position = c.mass.clone(), c.position.clone()
    g = torch.Generator(device="cuda").manual_seed(1)
    # q, k and v as columns of one projection; magnitudes over the type's range
    qkv = torch.randn(tokens, 5 * heads, dim, device="cuda", generator=g)
    qkv *= torch.exp2(torch.randint(-12, 9, (tokens, 1, 1), device="cuda", generator=g).float())
    qkv = qkv.to(DTYPES[dtype])
    qkv[3] = 0
    k, v = qkv[:, heads:2 * heads], qkv[:, 3 * heads:4 * heads]
    slots = torch.randperm(9 * page, device="cuda", generator=g)[:tokens]
    slots[5], slots[7], slots[9] = -1, 9 * page, 2 ** 40  # outside the cache: skipped
    positions = torch.arange(100, 100 + tokens, dtype=torch.int32, device="cuda")
    c.append(k, v, slots, positions)
    got = c.read(slots)
    s = slots.cpu().numpy()
    there = (s >= 0) & (s < 9 * page)
    for w, new, old, back in (("k", k, before[0], got[0]), ("v", v, before[1], got[1])):
        x = new.double().cpu().numpy()
        x = rounded(x) if mx else x
        want = old.copy()
        want[s[there] // page, :, s[there] % page] = x[there]
        assert np.array_equal(opened(c, w), want)
        x[~there] = 0
        # the 4-bit values' own rounding to f16 below its smallest step
        assert np.array_equal(back.double().cpu().numpy(),
                              torch.from_numpy(x).to(DTYPES[dtype]).double().numpy())
    at = torch.from_numpy(s[there]).cuda()
    mass[at // page, :, at % page] = 0
    position[at // page, :, at % page] = positions[torch.from_numpy(there).cuda()][:, None]
    assert torch.equal(c.mass, mass) and torch.equal(c.position, position)


def test_append_at_any_alignment(kv):
    """Rows that start and step by odd numbers of values."""
    heads, dim, page, tokens = 2, 64, 32, 40
    for dtype, mx in (("bf16", True), ("bf16", False), ("f32", False)):
        c = make(kv, dtype, mx, dim, page, heads, 2)
        flat = torch.randn(3 + tokens * 2 * (heads * (dim + 1) + 1), device="cuda").to(DTYPES[dtype])
        size = (tokens, heads, dim)
        k = flat.as_strided(size, (heads * (dim + 1) + 1, dim + 1, 1), 3)
        v = flat.as_strided(size, (heads * (dim + 1) + 1, dim + 1, 1), 5)
        slots = torch.arange(tokens, device="cuda")
        pos = slots.int()
        c.append(k, v, slots, pos)
        got = c.read(slots)
        # a last dimension that is not dense, and heads in another order
        c.append(k.transpose(1, 2).contiguous().transpose(1, 2), v, slots, pos)
        for a, b in zip(got, c.read(slots)):
            assert torch.equal(a, b)
        for a, x in zip(got, (k, v)):
            x = x.double().cpu().numpy()
            assert np.array_equal(a.double().cpu().numpy(), rounded(x) if mx else x)


def test_4_bit_rounding_at_its_edges(kv):
    """Ties, powers of two, saturation, subnormals, zeros of both signs and
    blocks that are not finite, for every exponent of bf16."""
    page, rows = 16, []
    base = np.array([0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6, 7, 7.5, 7.96875, 0.5, 1, 1.5, 2, 3,
                     4, 0.249, 0.251, 0.749, 0.751, 2.49, 2.51, 4.99, 5.01, 0.1, 0.01, 1e-3, 1e-5,
                     0, 0], np.float64)
    for e in range(-133, 126):
        rows.append(np.stack([base, -base]).reshape(-1) * 2.0 ** e)
        rows.append(np.concatenate([base[::-1] / 2, np.full(32, 2.0 ** min(e + 2, 127) / 2 ** e)])
                    * 2.0 ** e)
    x = torch.tensor(np.array(rows)).clamp(-3e38, 3e38).bfloat16()
    x[4, 3], x[6, 40], x[8, 0] = math.inf, math.nan, -math.inf
    tokens = len(rows)
    c = make(kv, "bf16", True, 64, page, 1, -(-tokens // page), track=False)
    x = x.cuda()[:, None]
    slots = torch.arange(tokens, device="cuda")
    c.append(x, x.flip(2), slots)
    k, v = c.read(slots)
    want = rounded(x.double().cpu().numpy())
    # what lies below bf16's smallest step rounds once more on the way out
    want = torch.from_numpy(want).bfloat16().double().numpy()
    got = k.double().cpu().numpy()
    assert np.array_equal(got, want, equal_nan=True)
    assert np.array_equal(v.flip(2).double().cpu().numpy(), want, equal_nan=True)
    assert np.array_equal(opened(c, "k").transpose(0, 2, 1, 3).reshape(-1, 64)[:tokens],
                          rounded(x.double().cpu().numpy())[:, 0], equal_nan=True)


# --------------------------------------------------------------------- attend
def attend64(c, q, table, lengths, scale):
    """(out, weights summed over a kv head's queries, what a row's error grows
    with, the largest sum |q||k| scale) in f64; weights as (sequences, kv heads,
    places)."""
    k, v = opened(c, "k"), opened(c, "v")
    q, table, lengths = q.double().cpu().numpy(), table.cpu().numpy(), lengths.cpu().numpy()
    page, heads = c.page_size, c.kv_heads
    group = q.shape[1] // heads
    out, size = np.zeros(q.shape), np.zeros(q.shape)
    weight = np.zeros((len(q), heads, table.shape[1] * page))
    spread = 0.0
    for b in range(len(q)):
        n = min(max(lengths[b], 0), table.shape[1] * page)
        j = np.arange(n)
        p = table[b, j // page]
        j = j[(p >= 0) & (p < c.pages)]
        if not len(j):
            continue
        at = table[b, j // page], j % page
        for h in range(heads):
            kk, vv = k[at[0], h, at[1]], v[at[0], h, at[1]]
            qq = q[b, h * group:(h + 1) * group]
            with np.errstate(invalid="ignore"):
                s = qq @ kk.T * scale
            top = s.max(1, keepdims=True)
            top[np.isneginf(top)] = 0
            with np.errstate(invalid="ignore"):
                e = np.exp(s - top)
                tot = e.sum(1, keepdims=True)
                w = np.where(tot == 0, 0, e / np.where(tot == 0, 1, tot))
                out[b, h * group:(h + 1) * group] = w @ vv
                size[b, h * group:(h + 1) * group] = w @ np.abs(vv)
            weight[b, h, j] = w.sum(0)
            if np.isfinite(kk).all():
                spread = max(spread, float((np.abs(qq) @ np.abs(kk).T).max() * abs(scale)))
    return out, weight, size, spread


def off_by(dim, tokens, spread, dtype):
    """How far a weight may be off, relative: a score is a sum of dim products
    in f32 (dim + 8 roundings of at most its sum of magnitudes, the scaling
    among them), two scores make a weight, whose exponential, sums and division
    add some roundings and the sum over tokens one for each 64 of them; the
    weights that multiply values keep 16 bits of a 16-bit type."""
    f32 = 2.0 ** -24
    kept = 0.0 if dtype == "f32" else 2.0 ** -16
    return 2 * (dim + 8) * f32 * max(spread, 1.0) + (16 + tokens / 64) * f32 + kept


def check_attend(kv, c, dtype, q, table, lengths, scale=None):
    want, weight, size, spread = attend64(c, q, table, lengths,
                                          c.head_dim ** -0.5 if scale is None else scale)
    mass = c.mass.clone() if c.mass is not None else None
    got = c.attend(q, table, lengths, scale)
    n = table.shape[1] * c.page_size
    rel = off_by(c.head_dim, n, spread, dtype)
    bound = UNIT[dtype] * np.abs(want) + rel * size + 1e-30
    if dtype == "f16":
        bound += 2.0 ** -25  # half of f16's smallest step
    far = np.abs(got.double().cpu().numpy() - want)
    assert (far <= bound).all(), (far.max(), (far / bound).max())
    if mass is not None:
        old = mass.double().cpu().numpy()
        expect = old.copy()
        add = np.zeros_like(old)
        t, group = table.cpu().numpy(), q.shape[1] // c.kv_heads
        for b in range(len(t)):
            for w, p in enumerate(t[b]):
                if 0 <= p < c.pages:
                    add[p] += weight[b, :, w * c.page_size:(w + 1) * c.page_size]
        expect += add
        far = np.abs(c.mass.double().cpu().numpy() - expect)
        ok = (rel + group * 2.0 ** -24) * add + len(t) * 2.0 ** -24 * expect + 1e-30
        assert (far <= ok).all(), (far.max(), (far / ok).max())
    return got


STORES = [("bf16", False), ("f16", False), ("f32", False), ("bf16", True), ("f16", True)]


@pytest.mark.parametrize("dtype,mx", STORES)
@pytest.mark.parametrize("dim,page,heads,group", [(64, 16, 2, 7), (96, 32, 3, 1), (128, 64, 2, 6),
                                                  (192, 128, 1, 5), (256, 16, 1, 16),
                                                  (128, 256, 1, 40), (64, 64, 5, 17),
                                                  (192, 32, 1, 24), (256, 16, 2, 20), (96, 128, 1, 33)])
def test_attend(kv, dtype, mx, dim, page, heads, group):
    """Every storage, width and page size: lengths of none, one, just around
    tiles and pages, and some hundreds."""
    lengths = [0, 1, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 257, 700]
    pages = sum(-(-n // page) for n in lengths)
    c = make(kv, dtype, mx, dim, page, heads, pages, seed=dim + group)
    table, n = tables(lengths, page, pages, seed=group, more=2)
    q = torch.randn(len(lengths), heads * group, dim, device="cuda").to(DTYPES[dtype])
    check_attend(kv, c, dtype, q, table, n)


@pytest.mark.parametrize("dtype,mx", STORES)
@pytest.mark.parametrize("length", [5000, 33333])
def test_attend_one_long_sequence(kv, dtype, mx, length):
    c = make(kv, dtype, mx, 128, 64, 1, -(-length // 64), seed=length)
    table, n = tables([length], 64, c.pages)
    q = 2 * torch.randn(1, 6, 128, device="cuda").to(DTYPES[dtype])
    check_attend(kv, c, dtype, q, table, n)


@pytest.mark.parametrize("dtype,mx", STORES)
@pytest.mark.parametrize("heads,group,top", [(8, 2, 60), (4, 3, 420), (2, 1, 900), (3, 18, 300)])
def test_attend_many_sequences(kv, dtype, mx, heads, group, top):
    """More groups than workgroups and fewer, so that a workgroup's share is
    several groups, ends inside of one or where one starts; every fifth sequence
    is empty.  The same call gives the same bits."""
    rng = np.random.default_rng(top)
    lengths = [0 if i % 5 == 3 else int(rng.integers(1, top)) for i in range(230)]
    pages = sum(-(-n // 32) for n in lengths)
    c = make(kv, dtype, mx, 64, 32, heads, pages, seed=top)
    table, n = tables(lengths, 32, pages, seed=top)
    q = torch.randn(len(lengths), heads * group, 64, device="cuda").to(DTYPES[dtype])
    got = check_attend(kv, c, dtype, q, table, n)
    assert torch.equal(c.attend(q, table, n), got)


@pytest.mark.parametrize("dtype,mx", STORES)
def test_attend_what_is_masked_can_be_anything(kv, dtype, mx):
    """Behind a sequence's last token lie NaN and infinities; table entries
    that are no page of the cache leave their tokens out; lengths beyond the
    table are cut."""
    page, dim = 16, 64
    c = make(kv, dtype, mx, dim, page, 2, 40, seed=3)
    table, n = tables([37, 1, 100, 48, 200], page, 40, seed=4)
    order = table.cpu().numpy()
    spare = sorted(set(range(40)) - set(order.ravel().tolist()))
    for b, m in enumerate([37, 1, 100, 48, 200]):
        p = order[b, (m - 1) // page]
        places = slice((m - 1) % page + 1, page)
        for t, s in ((c.k, c.k_scale), (c.v, c.v_scale)):
            if mx:
                s[p, :, places] = 255
            else:
                t[p, :, places] = math.nan if b % 2 else math.inf
    table[0, 1] = -1       # a hole: tokens 16 to 31
    table[2, 0] = 40       # no page of the cache
    table[3, :] = -7       # nothing left
    table[1, 3:] = spare[0]
    n[4] = 10 ** 6         # cut to the table
    table[4] = torch.tensor(np.resize(order[4, :13], table.shape[1]), device="cuda")
    q = torch.randn(5, 6, dim, device="cuda").to(DTYPES[dtype])
    # the last page of sequence 4 holds masked values only if its length ends there
    c2 = c
    for t, s in ((c2.k, c2.k_scale), (c2.v, c2.v_scale)):
        p = order[4, 199 // page]
        if mx:
            s[p] = 127
        else:
            t[p] = 1.0
    got = check_attend(kv, c, dtype, q, table, n)
    assert not got[3].any()
    assert torch.isfinite(got).all()
    n.zero_()
    assert not c.attend(q, table, n).any()
    n.fill_(-5)
    assert not c.attend(q, table, n).any()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_attend_scores_that_are_not_finite(kv, dtype):
    """A key of -infinity weighs nothing, a row of them gives zeros; NaN and
    +infinity make the row NaN, and no other row."""
    c = make(kv, dtype, False, 64, 16, 1, 8, seed=5, track=False)
    table, n = tables([20, 20, 20, 20, 16], 16, 10, seed=5)
    table = table % 8  # pages shared between sequences
    table = torch.tensor([[0, 1], [2, 3], [4, 5], [6, 7], [2, 0]], dtype=torch.int32, device="cuda")
    q = torch.ones(5, 2, 64, device="cuda").to(DTYPES[dtype])
    c.k[0, 0, 3, 0] = -math.inf
    c.k[2] = 0
    c.k[3] = 0
    c.k[2, 0, :, 7] = -math.inf
    c.k[3, 0, :, 9] = -math.inf
    c.k[4, 0, 5, 1] = math.nan
    c.k[7, 0, 2, 0] = math.inf
    got = c.attend(q, table, n).double().cpu().numpy()
    want, _, size, spread = attend64(c, q, table, n, 0.125)
    bound = UNIT[dtype] * np.abs(want) + off_by(64, 32, 64.0, dtype) * size + 1e-30 + 2.0 ** -25
    assert (np.abs(got - want)[0] <= bound[0]).all()
    assert not got[1].any() and not got[4].any()
    assert np.isnan(got[2]).all() and np.isnan(got[3]).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_attend_values_that_are_not_finite(kv, dtype):
    """They spoil their own column, for the heads and the sequence that read
    them, and nothing else."""
    c = make(kv, dtype, False, 64, 16, 2, 12, seed=6)
    table, n = tables([70, 100], 16, 12, seed=6)
    q = torch.randn(2, 6, 64, device="cuda").to(DTYPES[dtype])
    want = c.attend(q, table, n)
    c.v[table[0, 2], 0, 5, 17] = math.inf
    c.v[table[1, 6], 1, 3, 40] = math.nan
    got = c.attend(q, table, n)
    spoiled = torch.zeros_like(got, dtype=torch.bool)
    spoiled[0, :3, 17] = spoiled[1, 3:, 40] = True
    assert not torch.isfinite(got[spoiled]).any()
    assert torch.equal(got[~spoiled], want[~spoiled])


@pytest.mark.parametrize("dtype,mx", STORES)
def test_attend_scores_far_apart(kv, dtype, mx):
    """Scores in the thousands: the running maximum carries, the largest token
    first, last or in the middle."""
    c = make(kv, dtype, mx, 128, 64, 1, 24, seed=6)
    table, n = tables([500, 500, 500], 64, 24, seed=6)
    q = torch.randn(3, 4, 128, device="cuda").to(DTYPES[dtype])
    check_attend(kv, c, dtype, q, table, n, scale=20.0)
    check_attend(kv, c, dtype, q, table, n, scale=-3.0)
    check_attend(kv, c, dtype, q, table, n, scale=0.0)


def test_attend_strides_and_tracking(kv):
    """Queries as columns of a projection or of odd alignment, a table that is
    a slice of a wider one, weights kept only where asked for."""
    c = make(kv, "bf16", False, 128, 32, 2, 20, seed=7)
    table, n = tables([100, 250, 33], 32, 20, seed=7)
    wide = torch.full((3, 40), 10 ** 6, dtype=torch.int32, device="cuda")
    wide[:, 5:5 + table.shape[1]] = table
    qkv = torch.randn(3, 16, 128, device="cuda").bfloat16()
    q = qkv[:, :8]
    want = check_attend(kv, c, "bf16", q, table, n)
    assert torch.equal(c.attend(q, wide[:, 5:5 + table.shape[1]], n), want)
    odd = torch.zeros(3 * 8 * 129 + 1, device="cuda", dtype=torch.bfloat16)
    odd = odd[1:].as_strided((3, 8, 128), (8 * 129, 129, 1)).copy_(q)
    assert torch.equal(c.attend(odd, table, n), want)
    assert torch.equal(c.attend(q.transpose(1, 2).contiguous().transpose(1, 2), table, n), want)
    before = c.mass.clone()
    assert torch.equal(c.attend(q, table, n, track=False), want)
    assert torch.equal(c.mass, before)
    c.attend(q, table, n)
    assert not torch.equal(c.mass, before)
    # as often as called: the same bits
    for _ in range(3):
        assert torch.equal(c.attend(q, table, n), want)


def test_attend_counts_shared_pages_for_every_sequence(kv):
    """Sequences that share a prompt's pages both add to its tokens' mass."""
    c = make(kv, "bf16", False, 64, 16, 1, 6, seed=8)
    table = torch.tensor([[0, 1, 2], [0, 1, 3], [0, 1, 4]], dtype=torch.int32, device="cuda")
    n = torch.tensor([48, 40, 33], dtype=torch.int32, device="cuda")
    check_attend(kv, c, "bf16", torch.randn(3, 3, 64, device="cuda").bfloat16(), table, n)


# ---------------------------------------------------------------------- evict
def evict64(c, table, lengths, seen, budget, recent, into=None):
    """New lengths, and for every sequence and kv head the tokens' moves as
    (page, place) pairs from and to."""
    mass, position = c.mass.cpu().numpy().astype(np.float64), c.position.cpu().numpy()
    table, lengths, seen = table.cpu().numpy(), lengths.cpu().numpy(), seen.cpu().numpy()
    page, moves = c.page_size, []
    new = np.minimum(lengths, budget)
    for b, n in enumerate(lengths):
        n = min(max(n, 0), table.shape[1] * page)
        new[b] = min(n, budget)
        j = np.arange(n)
        p, at = table[b, j // page], j % page
        there = (p >= 0) & (p < c.pages)
        for h in range(c.kv_heads):
            m = np.where(there, mass[np.where(there, p, 0), h, at], 0)
            m[np.isnan(m)] = -np.inf
            pos = position[np.where(there, p, 0), h, at]
            kind = np.where(~there, 2, np.where(pos >= int(seen[b]) - recent, 0, 1))
            m = np.where(kind == 1, m, 0)
            kept = np.sort(np.lexsort((j, -m, kind))[:budget])
            if into is not None:
                src, dst = kept, np.arange(len(kept))
                to = into.cpu().numpy()[b, dst // page]
            elif n > budget:
                src, dst = kept[kept >= budget], np.setdiff1d(np.arange(budget), kept)
                to = table[b, dst // page]
            else:
                continue
            for s, d, t in zip(src, dst, to):
                if 0 <= p[s] < c.pages and 0 <= t < c.pages:
                    moves.append((h, p[s], s % page, t, d % page))
    return new, moves


def check_evict(kv, c, table, lengths, seen, budget, recent, into=None):
    names = [w for w in ("k", "v", "k_scale", "v_scale", "mass", "position") if getattr(c, w) is not None]
    new, moves = evict64(c, table, lengths, seen, budget, recent, into)
    want = {w: getattr(c, w).clone() for w in names}
    if moves:
        h, p, s, t, d = (torch.from_numpy(x).cuda().long() for x in np.array(moves).T)
        for w in names:
            want[w][t, h, d] = getattr(c, w)[p, h, s]
    got = c.evict(table, lengths, seen, budget, recent, into)
    assert np.array_equal(got.cpu().numpy(), new)
    for w in names:
        a, b = getattr(c, w), want[w]
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), w
    return got


def spread_positions(c, table, lengths, seed=0):
    """Tokens in no order: position 2r + 1 for the r-th of a sequence."""
    rng = np.random.default_rng(seed)
    c.position.fill_(-1)
    for b, n in enumerate(lengths.tolist()):
        j = np.arange(n)
        p = torch.from_numpy(table[b].cpu().numpy()[j // c.page_size].astype(np.int64)).cuda()
        ok = p >= 0
        for h in range(c.kv_heads):
            pos = torch.from_numpy(2 * rng.permutation(n).astype(np.int32) + 1).cuda()
            c.position[p[ok], h, torch.from_numpy(j % c.page_size).cuda()[ok]] = pos[ok]
    return (2 * lengths).int()


@pytest.mark.parametrize("dtype,mx,dim,page", [("bf16", False, 128, 64), ("f16", False, 64, 16),
                                               ("f32", False, 96, 32), ("bf16", True, 96, 16),
                                               ("f16", True, 256, 128), ("bf16", False, 192, 256)])
@pytest.mark.parametrize("other", [False, True], ids=["in place", "into"])
def test_evict(kv, dtype, mx, dim, page, other):
    """Lengths of none, one, below, at, just above and far above the budget;
    ties and zeros among the masses."""
    lengths, budget = [0, 1, 99, 100, 101, 116, 150, 199, 200, 201, 700, 1500], 100
    heads, wide = 3, -(-budget // page)
    need = sum(-(-n // page) for n in lengths)
    for recent in (0, 1, 37, 100):
        c = make(kv, dtype, mx, dim, page, heads, need + len(lengths) * wide, seed=recent)
        c.mass.copy_((c.mass * 20).floor() / 4)  # many ties, zeros among them
        table, n = tables(lengths, page, need, seed=recent, more=1)
        seen = spread_positions(c, table, n, recent)
        into = None
        if other:
            into = torch.arange(need, c.pages, device="cuda").int().reshape(len(lengths), wide)
        check_evict(kv, c, table, n, seen, budget, recent, into)


@pytest.mark.parametrize("length,budget", [(9000, 8999), (9000, 4096), (40000, 39990), (40000, 512),
                                           (70001, 30000), (2049, 2048), (1025, 1), (1024, 1023)])
@pytest.mark.parametrize("other", [False, True], ids=["in place", "into"])
def test_evict_long(kv, length, budget, other):
    page, heads = 64, 2
    wide, need = -(-budget // page), -(-length // page)
    c = make(kv, "bf16", True, 64, page, heads, need + wide, seed=length)
    c.mass[:, :, ::3] = 0
    table, n = tables([length], page, need, seed=budget)
    seen = spread_positions(c, table, n, budget)
    into = torch.arange(need, need + wide, device="cuda").int()[None] if other else None
    check_evict(kv, c, table, n, seen, budget, budget // 3, into)


def test_evict_masses_that_are_not_numbers(kv):
    """NaN counts as -infinity; both zeros are alike; negative masses sort as
    numbers; all alike keeps the lowest indices."""
    page, n = 16, 400
    c = make(kv, "bf16", False, 64, page, 2, 25, seed=9)
    flat = c.mass.view(-1)
    flat.copy_(torch.randn(flat.shape, device="cuda"))
    flat[::7], flat[1::7], flat[2::7], flat[3::7] = math.nan, math.inf, -math.inf, 0.0
    flat[4::7] = -0.0
    table, lengths = tables([n], page, 25)
    seen = spread_positions(c, table, lengths)
    for budget in (390, 300, 200, 100, 50, 3):
        check_evict(kv, c, table, lengths, seen, budget, 2)
    c.mass.fill_(1.0)
    check_evict(kv, c, table, lengths, seen, 77, 0)
    c.position.fill_(2 ** 31 - 1)
    seen.fill_(2 ** 31 - 1)
    check_evict(kv, c, table, lengths, seen, 55, 0)
    c.position.fill_(-2 ** 31)
    seen.fill_(-2 ** 31)
    check_evict(kv, c, table, lengths, seen, 44, 44)


def test_evict_leaves_absent_pages_out(kv):
    """Tokens whose table entry is no page go first and are neither read nor
    written; lengths beyond the table are cut."""
    page = 16
    c = make(kv, "f16", True, 64, page, 2, 30, seed=10)
    table, lengths = tables([200, 150, 64], page, 30, seed=10)
    seen = spread_positions(c, table, lengths)
    table[0, 1], table[0, 9], table[1, 2], table[2, :] = -1, 30, -9, -1
    lengths[1] = 10 ** 6
    check_evict(kv, c, table, lengths, seen, 60, 10)
    check_evict(kv, c, table, lengths, seen, 500, 10)


# ------------------------------------------------------- streams, graphs, size
def test_on_another_stream(kv):
    """Calls on a side stream see what was queued there before them."""
    c = make(kv, "bf16", True, 128, 64, 2, 40, seed=11)
    table, n = tables([1000, 700], 64, 40, seed=11)
    q = torch.randn(2, 12, 128, device="cuda").bfloat16()
    want = c.attend(q, table, n, track=False)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    big = torch.randn(4096, 4096, device="cuda")
    with torch.cuda.stream(side):
        late = torch.zeros_like(q)
        for _ in range(8):
            big = (big @ big).clamp_(-1, 1)
        late.copy_(q)
        got = [c.attend(late, table, n, track=False) for _ in range(3)]
    side.synchronize()
    for x in got:
        assert torch.equal(x, want)


def test_two_streams_at_once(kv):
    """Calls on one cache that overlap do not share anything but the cache."""
    c = make(kv, "bf16", False, 128, 64, 2, 400, seed=12)
    table, n = tables([20000, 5000], 64, 400, seed=12)
    qs = [torch.randn(2, 12, 128, device="cuda").bfloat16() for _ in range(2)]
    want = [c.attend(q, table, n, track=False) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(c.attend(qs[i], table, n, track=False))
    torch.cuda.synchronize()
    for i in range(2):
        for x in got[i]:
            assert torch.equal(x, want[i])


def test_under_graph_capture(kv):
    """A step of append, attend and evict, captured and replayed with other
    inputs and eager work between, gives what eager calls give."""
    page, heads = 16, 2
    table, _ = tables([130, 90], page, 16, seed=13)
    inputs = []
    g = torch.Generator(device="cuda").manual_seed(13)
    for step in range(4):
        inputs.append((torch.randn(2, 16, 64, device="cuda", generator=g).bfloat16(),
                       torch.tensor([120 + step, 80 + step], dtype=torch.int32, device="cuda")))

    def step(c, qkv, n):
        c.append(qkv[:, 12:14], qkv[:, 14:], c.slots(table, torch.arange(2, device="cuda"), n), n)
        out = c.attend(qkv[:, :12], table, n + 1)
        return out, c.evict(table, n + 1, n + 1, 100, 20)

    eager = make(kv, "bf16", True, 64, page, heads, 16, seed=14)
    want = [tuple(t.clone() for t in step(eager, *x)) + (eager.mass.clone(),) for x in inputs]
    c = make(kv, "bf16", True, 64, page, heads, 16, seed=14)
    state = {w: getattr(c, w).clone() for w in ("k", "v", "k_scale", "v_scale", "mass", "position")}
    qkv, n = (t.clone() for t in inputs[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(c, qkv, n)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, left = step(c, qkv, n)
    for w, t in state.items():
        getattr(c, w).copy_(t)
    for x, (a, b, mass) in zip(inputs, want):
        qkv.copy_(x[0])
        n.copy_(x[1])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, a) and torch.equal(left, b) and torch.equal(c.mass, mass)
        (torch.randn(1000, 1000, device="cuda") @ torch.randn(1000, 1000, device="cuda")).sum().item()
        other = make(kv, "f16", False, 64, page, heads, 16, seed=15)
        other.attend(torch.randn(2, 4, 64, device="cuda").half(), table, n)


def test_offsets_beyond_32_bits(kv):
    """The last pages of a cache of more than 2^32 values, their bytes beyond
    2^33."""
    pages, heads, page, dim = 66000, 8, 64, 128
    assert pages * heads * page * dim > 2 ** 32
    k, v = (torch.empty(pages, heads, page, dim, dtype=torch.bfloat16, device="cuda")
            for _ in range(2))
    mass = torch.zeros(pages, heads, page, device="cuda")
    position = torch.zeros(pages, heads, page, dtype=torch.int32, device="cuda")
    c = kv.PagedCache(k, v, torch.bfloat16, mass=mass, position=position)
    small = make(kv, "bf16", False, dim, page, heads, 8, seed=16)
    last = [pages - 1, 3, pages - 2, pages // 2 + 1, pages - 3, pages - 7, 0, 40000]
    for w in ("k", "v", "mass", "position"):
        getattr(c, w)[last] = getattr(small, w)
    t_small = torch.arange(4, device="cuda").int()[None]
    t_big = torch.tensor(last[:4], dtype=torch.int32, device="cuda")[None]
    n = torch.tensor([250], dtype=torch.int32, device="cuda")
    q = torch.randn(1, 16, dim, device="cuda").bfloat16()
    new = torch.randn(2, 1, heads, dim, device="cuda").bfloat16()
    for cache, table in ((c, t_big), (small, t_small)):
        slot = cache.slots(table, torch.zeros(1, device="cuda"), n.long())
        cache.append(new[0], new[1], slot, n)
        assert torch.equal(cache.read(slot)[1], new[1])
    seen, n = n + 1, n + 1
    assert torch.equal(c.attend(q, t_big, n), small.attend(q, t_small, n))
    into = [torch.tensor([x], dtype=torch.int32, device="cuda") for x in (last[4:6], [4, 5])]
    for cache, table, other in ((c, t_big, into[0]), (small, t_small, into[1])):
        cache.evict(table, n, seen, 100, 7, other)
        cache.evict(table, n, seen, 200, 7)
    for w in ("k", "v", "mass", "position"):
        assert torch.equal(getattr(c, w)[last], getattr(small, w)), w


# -------------------------------------------------------------------- refusals
def test_refusals(kv):
    c = make(kv, "bf16", False, 64, 16, 2, 8)
    table, n = tables([20, 30], 16, 8)
    q = torch.zeros(2, 4, 64, device="cuda", dtype=torch.bfloat16)
    k = torch.zeros(2, 2, 64, device="cuda", dtype=torch.bfloat16)
    slots, pos = torch.tensor([1, 2], device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    bad = [
        lambda: c.attend(q.float(), table, n), lambda: c.attend(q.cpu(), table, n),
        lambda: c.attend(q[:, :3], table, n), lambda: c.attend(q[:, :0], table, n),
        lambda: c.attend(q[0], table, n), lambda: c.attend(q[..., :32], table, n),
        lambda: c.attend(q[:1], table, n), lambda: c.attend(q, table.long(), n),
        lambda: c.attend(q, table, n.long()), lambda: c.attend(q, table, n[:1]),
        lambda: c.attend(q, table.cpu(), n), lambda: c.attend(q, table[0], n),
        lambda: c.attend(q, table.t().contiguous().t(), n),
        lambda: c.attend(q.float().requires_grad_().bfloat16(), table, n),
        lambda: c.append(k, k, slots), lambda: c.append(k, k, slots.int(), pos),
        lambda: c.append(k, k[:1], slots, pos), lambda: c.append(k, k, slots[:1], pos),
        lambda: c.append(k, k, slots, pos[:1]), lambda: c.append(k, k, slots, pos.long()),
        lambda: c.append(q, q, slots, pos), lambda: c.append(k.half(), k, slots, pos),
        lambda: c.read(slots.int()), lambda: c.read(slots.cpu()),
        lambda: c.evict(table, n, n, 0), lambda: c.evict(table, n, n, -1),
        lambda: c.evict(table, n, n, 10, 11), lambda: c.evict(table, n, n, 10, -1),
        lambda: c.evict(table, n, n[:1], 10), lambda: c.evict(table, n.long(), n, 10),
        lambda: c.evict(table, n, n, 17, 0, table[:, :1]),
        lambda: c.evict(table, n, n, 10, 0, table[:1]),
        lambda: kv.PagedCache.allocate(4, 2, 80), lambda: kv.PagedCache.allocate(4, 2, 64, 48),
        lambda: kv.PagedCache.allocate(4, 2, 64, dtype=torch.float32, mx=True),
        lambda: kv.PagedCache.allocate(4, 2, 64, dtype=torch.float64),
        lambda: kv.PagedCache.allocate(0, 2, 64),
        lambda: kv.PagedCache(c.k, c.v.half(), torch.bfloat16),
        lambda: kv.PagedCache(c.k, c.v[:4], torch.bfloat16),
        lambda: kv.PagedCache(c.k[:, :, ::2], c.v[:, :, ::2], torch.bfloat16),
        lambda: kv.PagedCache(c.k, c.v, torch.bfloat16, mass=c.mass),
        lambda: kv.PagedCache(c.k, c.v, torch.bfloat16, k_scale=c.mass),
        lambda: kv.PagedCache(c.k, c.v.cpu(), torch.bfloat16),
    ]
    before = [getattr(c, w).clone() for w in ("k", "v", "mass", "position")]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print("accepted:", i)
    plain = make(kv, "bf16", False, 64, 16, 2, 8, track=False)
    with pytest.raises(ValueError):
        plain.evict(table, n, n, 10)
    with pytest.raises(ValueError):
        plain.attend(q, table, n, track=True)
    plain.append(k, k, slots)
    for a, w in zip(before, ("k", "v", "mass", "position")):
        assert torch.equal(a, getattr(c, w))
    # nothing to do is no error
    c.append(k[:0], k[:0], slots[:0], pos[:0])
    assert c.read(slots[:0])[0].shape == (0, 2, 64)
    assert c.attend(q[:0], table[:0], n[:0]).shape == (0, 4, 64)
    assert not c.attend(q, table[:, :0], n).any()
    assert c.evict(table[:0], n[:0], n[:0], 10).shape == (0,)
    with torch.no_grad():
        c.attend(q.clone().requires_grad_(), table, n)
