"""The serve command times attention over all pages without what only the choice of
pages needs."""
import pytest

pytestmark = pytest.mark.gpu


def test_all_pages_are_timed_without_bounds(rans, monkeypatch):
    import kv_cache
    import rans_bench
    calls = []

    def spied(name):
        plain = getattr(kv_cache.PagedCache, name)

        def call(self, x, *args, **kwargs):
            if self.bounds is not None:  # not the heads' view of a cache
                calls.append((name, x.dim()))
            return plain(self, x, *args, **kwargs)
        monkeypatch.setattr(kv_cache.PagedCache, name, call)
    for name in ("bound", "attend", "select"):
        spied(name)
    r = rans_bench.serve(layers=2, batch=2, longest=700, count=4, steps=8)
    assert r["finite"]
    names = [name for name, _ in calls]
    first, last = names.index("attend"), len(names) - 1 - names[::-1].index("attend")
    assert set(names[first:last + 1]) == {"attend"}  # the steps over all pages
    # then, before pages are chosen, the bounds of whole tables: those pages grew without
    assert calls[last + 1:last + 3] == [("bound", 2)] * 2
    assert set(names[last + 3:]) == {"bound", "select"} and names.count("select") == 2 * 2
