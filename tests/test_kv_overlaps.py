"""Calls whose outputs lie over what they read, without a GPU: refused by the library
before any HIP call, with a message that says so."""
import pytest
import torch

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="a GPU is present, and the memory is none of its own")


@pytest.fixture
def host(rans, monkeypatch):
    """A pool and a rotation over CPU tensors and the library as it is."""
    import kv_cache
    import kv_pages
    import rotary
    monkeypatch.setattr(rans, "_device", lambda: -1)
    monkeypatch.setattr(rans, "_stream", lambda: 0)
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "is_available", lambda: True)
        m.setattr(torch.Tensor, "is_cuda", True)
        cache = kv_cache.PagedCache.allocate(8, 2, 64, 16, torch.float32, track=True, device="cpu", lib=rans._LIB,
                                             bounds=True)
        return cache, kv_pages.PagePool(8, 16, device="cpu", lib=rans._LIB), rotary.Rotary(64, device="cpu", lib=rans._LIB)


def test_what_is_refused_is_named(host):
    """A table whose rows are the lengths too: neither too large nor misaligned."""
    pool = host[1]
    table, n = torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    for call in (lambda: pool.extend(table, table[1, :3], n, 5), lambda: pool.release(table, table[1, :3])):
        with pytest.raises(ValueError, match="memory"):
            call()
