"""The page pool against a plain implementation: whole numbers, all equal."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv_pages(rans):
    import kv_pages
    return kv_pages


class Plain:
    """The pool in Python, one sequence, token and entry after the other."""

    def __init__(self, pages, page, free, count):
        self.pages, self.page, self.free, self.count = pages, page, list(free), min(max(count, 0), pages)

    def extend(self, table, lengths, new, tokens, seen=None):
        batch, width, page = len(table), len(table[0]) if len(table) else 0, self.page
        slots, positions, filled = [-1] * tokens, [0] * tokens, [-1] * tokens
        starts, grown, at, wanted, have = [0], [], 0, 0, self.count
        for b in range(batch):
            n, m = min(max(lengths[b], 0), width * page), max(new[b], 0)
            first, at = at, at + m
            fits = n + m <= width * page and at <= tokens
            old = -(-n // page)
            need = -(-(n + m) // page) - old if fits else 0
            wanted += need
            served = fits and (need == 0 or wanted <= have)
            if served:
                for k in range(old, old + need):
                    self.count -= 1
                    x = self.free[self.count]
                    table[b][k] = x if 0 <= x < self.pages else -1
            for t in range(min(first, tokens), min(at, tokens)):
                index = n + t - first
                positions[t] = np.int64((seen[b] if seen is not None else n) + t - first).astype(np.int32)
                p = table[b][index // page] if served else -1
                if 0 <= p < self.pages:
                    slots[t] = p * page + index % page
                    if index % page == page - 1:
                        filled[t] = p
            starts.append(min(at, tokens))
            grown.append(n + m if served else n)
        return slots, positions, filled, starts, grown

    def release(self, table, lengths):
        for row, n in zip(table, lengths):
            n = min(max(n, 0), len(row) * self.page)
            for k in range(-(-n // self.page), len(row)):
                if 0 <= row[k] < self.pages and self.count < self.pages:
                    self.free[self.count] = row[k]
                    self.count += 1
                row[k] = -1


def ints(x, **kw):
    return torch.tensor(x, dtype=torch.int32, device="cuda", **kw)


def make(rng, batch, width, page, most, spare, holes=0.0):
    """Sequences of up to `most` tokens in pages of a shuffled pool with `spare` more."""
    lengths = [int(rng.integers(0, most + 1)) for _ in range(batch)]
    if batch > 2:
        lengths[1], lengths[2] = 0, most
    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + spare
    order = [int(x) for x in rng.permutation(max(pages, 1))]
    table, at = np.full((batch, width), -1, np.int64), 0
    for b, c in enumerate(counts):
        table[b, :c] = order[at:at + c]
        at += c
        for k in range(c):
            if rng.random() < holes:
                table[b, k] = rng.choice([-1, -7, pages, 2 ** 31 - 1])
    free = order[at:] + [-1] * at
    return max(pages, 1), lengths, table, free[:max(pages, 1)], max(pages, 1) - at


def compare(pool, plain, table, want_table, step=None, want=None):
    assert pool.count.item() == plain.count
    assert pool.free.tolist() == plain.free
    assert table.tolist() == [list(map(int, r)) for r in want_table]
    assert pool._ticket.item() == 0
    if step is not None:
        for got, x, name in zip(step, want, step._fields):
            assert got.tolist() == [int(v) for v in x], name


CASES = [  # batch, width, page, most held, most new, spare pages, rows behind, holes
    (1, 1, 16, 0, 1, 1, 0, 0.0), (1, 4, 16, 17, 1, 3, 0, 0.0), (3, 7, 16, 60, 50, 9, 5, 0.0),
    (5, 9, 32, 200, 90, 4, 0, 0.0), (64, 40, 64, 2049, 1, 80, 0, 0.0), (7, 33, 128, 3000, 1500, 60, 13, 0.3),
    (200, 12, 256, 2000, 1, 30, 1, 0.0), (16, 512, 16, 0, 800, 900, 77, 0.0), (2, 600, 16, 5000, 4000, 700, 0, 0.1),
    (300, 3, 16, 40, 9, 10, 0, 0.0), (2, 130, 256, 20000, 12000, 1000, 3, 0.0),
]


@pytest.mark.parametrize("batch,width,page,most,new,spare,pad,holes", CASES)
@pytest.mark.parametrize("seen", [False, True])
def test_extend_and_release(kv_pages, batch, width, page, most, new, spare, pad, holes, seen):
    rng = np.random.default_rng(batch * 1000 + width)
    pages, lengths, table, free, count = make(rng, batch, width, page, most, spare, holes)
    fresh = [int(rng.integers(0, new + 1)) for _ in range(batch)]
    fresh[-1] = new
    ahead = [int(x) for x in rng.integers(0, 2 ** 31 - 20000, batch)] if seen else None
    tokens = sum(fresh) + pad
    pool = kv_pages.PagePool(pages, page, ints(free), ints([count]))
    plain = Plain(pages, page, free, count)
    want_table, got_table = table.copy(), ints(table)
    for _ in range(2):  # the second time from what the first one left
        step = pool.extend(got_table, ints(lengths), ints(fresh), tokens, None if ahead is None else ints(ahead))
        want = plain.extend(want_table, lengths, fresh, tokens, ahead)
        compare(pool, plain, got_table, want_table, step, want)
        assert step.slots.dtype is torch.int64
        lengths = [max(0, x - int(rng.integers(0, 3 * page))) for x in want[4]]
        pool.release(got_table, ints(lengths))
        plain.release(want_table, lengths)
        compare(pool, plain, got_table, want_table)


def test_numbers_out_of_range(kv_pages):
    """Negative lengths and new tokens are none, lengths beyond the row its end; what
    does not fit the row or the batch gets nothing, and later sequences still do."""
    free = list(range(12))
    lengths, new = [-5, 7, 1000, 3, 20, 2 ** 31 - 1, -2 ** 31], [3, -4, 0, 70, 30, 0, 2]
    for tokens in (0, 2, 3, 34, 72, 200):
        table = np.full((7, 4), -1)
        table[1:5, :2] = np.arange(20, 28).reshape(4, 2)
        pool, plain = kv_pages.PagePool(40, 16, ints(free + [0] * 28), ints([12])), Plain(40, 16, free + [0] * 28, 12)
        got = ints(table)
        step = pool.extend(got, ints(lengths), ints(new), tokens)
        compare(pool, plain, got, table, step, plain.extend(table, lengths, new, tokens))
    many = [2 ** 31 - 1] * 9  # sums beyond 32 bits
    table = np.full((9, 4), -1)
    pool, plain, got = kv_pages.PagePool(12, 16, ints(free), ints([12])), Plain(12, 16, free, 12), ints(table)
    step = pool.extend(got, ints([0] * 9), ints(many), 50)
    compare(pool, plain, got, table, step, plain.extend(table, [0] * 9, many, 50))


def test_a_short_pool_serves_in_order(kv_pages):
    """Sequences get all of their pages or none; after the first that does not, those
    that need no page are still served."""
    table = np.full((5, 4), -1)
    table[3, 0] = 9
    lengths, new = [0, 0, 0, 3, 0], [40, 40, 16, 5, 0]
    pool, plain, got = kv_pages.PagePool(10, 16, ints(list(range(10))), ints([5])), Plain(10, 16, range(10), 5), ints(table)
    step = pool.extend(got, ints(lengths), ints(new), 101)
    want = plain.extend(table, lengths, new, 101)
    assert want[4] == [40, 0, 0, 8, 0]
    compare(pool, plain, got, table, step, want)


def test_counts_and_pages_that_are_wrong(kv_pages):
    """A count beyond the pool counts as its end, and a stack of what are no pages gives
    none away; nothing is written outside."""
    for count in (-3, 0, 4, 99):
        free = [2, 17, -5, 1]
        table = np.full((3, 5), -1)
        pool, plain, got = kv_pages.PagePool(4, 16, ints(free), ints([count])), Plain(4, 16, free, count), ints(table)
        step = pool.extend(got, ints([0, 0, 0]), ints([16, 17, 40]), 80)
        compare(pool, plain, got, table, step, plain.extend(table, [0, 0, 0], [16, 17, 40], 80))
        pool.release(got, ints([0, 16, 0]))
        plain.release(table, [0, 16, 0])
        compare(pool, plain, got, table)


@pytest.mark.parametrize("width", [5, 700])
def test_a_page_given_back_twice_stays_inside(kv_pages, width):
    table = np.full((80, width), -1)
    table[:, 0] = 3
    table[:, -1] = 1
    pool, plain, got = kv_pages.PagePool(50, 16), Plain(50, 16, range(49, -1, -1), 50), ints(table)
    plain.count = 7
    pool.count.fill_(7)
    pool.release(got, ints([0] * 80))
    plain.release(table, [0] * 80)
    compare(pool, plain, got, table)


@pytest.mark.parametrize("batch,width", [(3, 64), (512, 64), (513, 64), (4, 8192), (4096, 1), (4096, 70), (1, 32768),
                                         (1, 40000), (64, 256), (64, 260), (65, 4), (64, 4), (16, 1024), (1, 16384),
                                         (1, 16388), (5, 1000), (1, 4), (17, 516), (63, 252)])
def test_release_of_tables(kv_pages, batch, width):
    rng = np.random.default_rng(width)
    table = np.full((batch, width), -1)
    table[rng.random((batch, width)) < 0.4] = 0
    at = np.flatnonzero(table == 0)
    table.flat[at] = rng.permutation(len(at))
    table[rng.random((batch, width)) < 0.01] = -9
    lengths = [int(x) for x in rng.integers(0, width * 4, batch)]
    pages = len(at) + 1
    pool, plain, got = kv_pages.PagePool(pages, 16), Plain(pages, 16, range(pages - 1, -1, -1), 0), ints(table)
    pool.count.zero_()
    pool.release(got, ints(lengths))
    want = table.copy()
    plain.release(want, lengths)
    compare(pool, plain, got, want)


@pytest.mark.parametrize("batch", [1000, 4096])
def test_extend_of_many_sequences(kv_pages, batch):
    rng = np.random.default_rng(batch)
    pages, lengths, table, free, count = make(rng, batch, 6, 16, 70, 5000)
    new = [int(x) for x in rng.integers(0, 9, batch)]
    tokens = sum(new) + 5
    pool, plain, got = kv_pages.PagePool(pages, 16, ints(free), ints([count])), Plain(pages, 16, free, count), ints(table)
    step = pool.extend(got, ints(lengths), ints(new), tokens)
    compare(pool, plain, got, table, step, plain.extend(table, lengths, new, tokens))


@pytest.mark.parametrize("first,columns", [(3, 20), (4, 20), (8, 14), (4, 17)])
def test_rows_of_a_wider_table(kv_pages, first, columns):
    """A table cut to the pages in use, at any alignment, and what lies beside it, which
    stays."""
    width = 6 if first % 2 else 8
    wide = torch.full((4, columns + 3), 77, dtype=torch.int32, device="cuda")[:, :columns]
    table = wide[:, first:first + width]
    table.fill_(-1)
    pool, plain, want = kv_pages.PagePool(30, 16), Plain(30, 16, range(29, -1, -1), 30), np.full((4, table.shape[1]), -1)
    lengths, new = [0] * 4, [90, 17, 96, 0]
    step = pool.extend(table, ints(lengths), ints(new), 203)
    compare(pool, plain, table, want, step, plain.extend(want, lengths, new, 203))
    pool.release(table, ints([16, 17, 50, 0]))
    plain.release(want, [16, 17, 50, 0])
    compare(pool, plain, table, want)
    assert (wide[:, :first] == 77).all() and (wide[:, first + table.shape[1]:] == 77).all()


def test_empty_calls(kv_pages):
    pool = kv_pages.PagePool(5, 16)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    step = pool.extend(none.view(0, 3), none, none, 4)
    assert step.slots.tolist() == [-1] * 4 and step.positions.tolist() == [0] * 4 and step.starts.tolist() == [0]
    step = pool.extend(torch.empty(2, 0, dtype=torch.int32, device="cuda"), ints([0, 3]), ints([0, 1]), 1)
    assert step.slots.tolist() == [-1] and step.lengths.tolist() == [0, 0]
    pool.release(none.view(0, 3), none)
    pool.release(torch.empty(2, 0, dtype=torch.int32, device="cuda"), ints([0, 3]))
    assert pool.count.item() == 5 and pool.free.tolist() == [4, 3, 2, 1, 0]


def test_in_a_graph_and_on_another_stream(kv_pages):
    """A captured step and its release, replayed with other lengths between eager work."""
    table, want = torch.full((40, 30), -1, dtype=torch.int32, device="cuda"), np.full((40, 30), -1)
    pool, plain = kv_pages.PagePool(900, 16), Plain(900, 16, range(899, -1, -1), 900)
    lengths, new, keep = (torch.zeros(40, dtype=torch.int32, device="cuda") for _ in range(3))
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        pool.extend(table, lengths, new, 3000)
        pool.release(table, keep)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step = pool.extend(table, lengths, new, 3000)
        pool.release(table, keep)
    held, rng = [0] * 40, np.random.default_rng(3)
    for i in range(4):
        fresh = [int(x) for x in rng.integers(0, 75, 40)]
        lengths.copy_(ints(held))
        new.copy_(ints(fresh))
        result = plain.extend(want, held, fresh, 3000)
        held = [max(0, x - int(rng.integers(0, 60))) for x in result[4]]
        keep.copy_(ints(held))
        plain.release(want, held)
        graph.replay()
        torch.cuda.synchronize()
        compare(pool, plain, table, want, step, result)


def test_refusals(kv_pages):
    pool = kv_pages.PagePool(8, 16)
    table, n = torch.full((3, 4), -1, dtype=torch.int32, device="cuda"), ints([0, 0, 0])
    for bad in (dict(table=table.long()), dict(table=table.cpu()), dict(table=table.t()),
                dict(table=table[:1].expand(3, 4)), dict(lengths=n[:2]), dict(lengths=n.long()), dict(new=n.cpu()),
                dict(new=n[None]), dict(tokens=-1), dict(tokens=2 ** 31), dict(seen=n[:1])):
        args = {**dict(table=table, lengths=n, new=n, tokens=4, seen=None), **bad}
        with pytest.raises(ValueError):
            pool.extend(**args)
        if "new" not in bad and "tokens" not in bad and "seen" not in bad:
            with pytest.raises(ValueError):
                pool.release(args["table"], args["lengths"])
    many = torch.empty(5000, 1, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        pool.extend(many, many[:, 0], many[:, 0], 1)
    for bad in (dict(pages=0), dict(page_size=48), dict(free=ints([1] * 8)), dict(count=ints([1])),
                dict(free=ints([1] * 7), count=ints([1])), dict(free=ints([1] * 8), count=ints([1, 1])),
                dict(free=ints([1] * 8).long(), count=ints([1])), dict(free=torch.zeros(8, dtype=torch.int32),
                                                                      count=torch.zeros(1, dtype=torch.int32))):
        with pytest.raises(ValueError):
            kv_pages.PagePool(**{**dict(pages=8, page_size=16), **bad})
