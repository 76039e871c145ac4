"""What an AttentionStack refuses before it needs a GPU."""
import pytest


@pytest.fixture
def bench(rans):
    import rans_bench
    return rans_bench


@pytest.mark.parametrize("kw", [dict(slack=0), dict(slack=-64), dict(budget=0), dict(slack=0, pooled=True)])
def test_a_row_at_its_budget_takes_a_token(bench, kw):
    """Without slack it would not, and the token would be lost."""
    with pytest.raises(ValueError, match="slack"):
        bench.AttentionStack(**{**dict(layers=1, batch=1, budget=64, recent=8, page=16), **kw})


def test_prompts_and_endings_take_a_pool(bench):
    """Refused before the host's counts change."""
    stack = object.__new__(bench.AttentionStack)
    stack.pool, stack.batch, stack.each, stack.held, stack.budget, stack.slack = None, 2, [5, 9], 9, 64, 16
    for call in (lambda: stack.write([None] * 3, [1, 2]), lambda: stack.finish([1])):
        with pytest.raises(ValueError, match="pool"):
            call()
    assert stack.each == [5, 9] and stack.held == 9
