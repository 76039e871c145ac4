"""Prompts of an AttentionStack that do not fit: refused before anything is written, or,
where the pool has no pages for them, named and not counted."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def bench(rans):
    import rans_bench
    return rans_bench


def make(bench, **kw):
    return bench.AttentionStack(layers=1, batch=3, budget=96, slack=16, recent=24, page=16, mx=False,
                                pooled=True, **kw)


def state(stack):
    c = stack.layers[0].cache
    return [t.clone() for t in (c.k, c.v, stack.table, stack.lengths, stack.seen, stack.pool.free, stack.pool.count)]


@pytest.mark.parametrize("rows,new", [(60, [40, 0, 40]), (100, [40, 0, 40]), (0, [40, 0, 40]), (80, [40, 40]),
                                      (80, [40, 0, 40, 0]), (80, [60, -20, 40]), (112, [0, 112, 0]),
                                      (92, [92, 0, 0]), (300, [100, 100, 100])])
def test_prompts_that_are_refused(bench, rows, new):
    """Too few or too many rows or sequences; a row with no place for a next token."""
    stack = make(bench, track=False)
    h = torch.randn(300, 1536, device="cuda").bfloat16()
    stack.write(h[:55], [20, 35, 0])
    before = state(stack)
    with pytest.raises(ValueError):
        stack.write(h[:rows], new)
    assert stack.each == [20, 35, 0] and stack.held == 35
    assert all(torch.equal(x, y) for x, y in zip(state(stack), before))
    assert stack.write(h[:91], [91, 0, 0]) == []  # the longest
    assert stack.each == stack.lengths.tolist() == [111, 35, 0]


def test_prompts_without_pages_are_not_counted(bench):
    """Rows that got nothing are named, and the budget is that of what the rows hold: the
    steps after them reach it when they do, with every token in its place."""
    stack = make(bench, track=True)
    h = torch.randn(200, 1536, device="cuda").bfloat16()
    taken = int(stack.pool.count) - 9
    stack.pool.count.fill_(9)  # as if another table held the others
    refused = stack.write(h[:150], [40, 20, 90])
    assert stack.each == stack.lengths.tolist() == stack.seen.tolist() == [40, 20, 0] and stack.held == 40
    assert refused == [2]
    assert stack.write(h[:60], [0, 60, 0]) == []
    assert stack.write(h[:40], [0, 0, 40]) == [2]
    assert stack.each == stack.lengths.tolist() == [40, 80, 0] and stack.held == 80
    stack.pool.count.add_(taken)
    want = [40, 80, 0]
    for step in range(50):
        stack.step(h[:3])
        want = [n + 1 for n in want]
        if max(want) == 112:
            want = [min(n, 96) for n in want]
        assert stack.each == stack.lengths.tolist() == want, step
