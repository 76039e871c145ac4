"""Calls whose outputs lie over what they read, without a GPU: refused by the library
before any HIP call, with a message that says so."""
import ctypes

import pytest
import torch

EARG = -4

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


# Addresses 1 MiB apart, in the order of their names; never dereferenced.
def places(*names):
    return {name: 0x10000000 + (i << 20) for i, name in enumerate(names)}


def each_pair(call, written, read):
    """Every output over every input, at its first and its last bytes, is refused; next
    to it, it gets as far as a HIP call.  written, read: bytes by name."""
    assert call() > 0
    for out, size in written.items():
        for name, n in read.items():
            if name == out:
                continue
            first = at[name]
            for address in (first, first + max(n - 16, 0), first - max(size - 16, 0)):
                assert call(**{out: address & -16}) == EARG, (out, name, hex(address - first))
            for address in (first + n + 16, first - size):
                assert call(**{out: address & -16}) > 0, (out, name, "beside")


TOKENS, Q_HEADS, K_HEADS, DIM = 10, 4, 2, 64
at = places("q", "k", "v", "q_weight", "k_weight", "positions", "turns", "slots", "q_out", "k_out", "pages_k",
            "pages_v", "scales_k", "scales_v", "mass", "place", "bounds", "list", "table", "lengths", "chosen", "held",
            "work", "free", "count", "ticket", "fresh", "seen", "filled", "starts", "grown")
# q and k are columns of one projection, as far as its last row's
ROWS = {"q": ((TOKENS - 1) * 400 + Q_HEADS * DIM) * 2, "k": ((TOKENS - 1) * 400 + K_HEADS * DIM) * 2, "q_weight": DIM * 4,
        "k_weight": DIM * 4, "positions": TOKENS * 4, "turns": 16 * 8}
PAGES, PAGE = 8, 16
CACHE = {"pages_k": PAGES * K_HEADS * PAGE * DIM * 2, "pages_v": PAGES * K_HEADS * PAGE * DIM * 2,
         "mass": PAGES * K_HEADS * PAGE * 4, "place": PAGES * K_HEADS * PAGE * 4}
CACHE_MX = {**CACHE, "pages_k": PAGES * K_HEADS * PAGE * DIM // 2, "pages_v": PAGES * K_HEADS * PAGE * DIM // 2,
            "scales_k": PAGES * K_HEADS * PAGE * DIM // 32, "scales_v": PAGES * K_HEADS * PAGE * DIM // 32}


def rotation(rotary, kw):
    a = {**at, **kw}
    r = rotary.RotaryDesc(DIM, 16, 0, 1.0, a["turns"])
    x = rotary.RowsDesc(a["q"], a["k"], 400, DIM, 400, DIM, Q_HEADS, K_HEADS, a["q_weight"], a["k_weight"], 1, 0, 1e-6,
                        a["positions"], TOKENS)  # bf16, weights of f32
    return a, ctypes.byref(r), ctypes.byref(x)


def cache_of(kv_cache, a, mx):
    return ctypes.byref(kv_cache.KvCacheDesc(
        pages=PAGES, kv_heads=K_HEADS, page_size=PAGE, head_dim=DIM, dtype=1, mx=int(mx), k=a["pages_k"], v=a["pages_v"],
        k_scale=a["scales_k"] if mx else None, v_scale=a["scales_v"] if mx else None, mass=a["mass"],
        position=a["place"]))


def test_rotate_writes_nothing_that_it_reads(host, lib):
    import rotary

    def call(**kw):
        a, r, x = rotation(rotary, kw)
        return lib.vramc_rotary_apply(r, x, a["q_out"], a["k_out"], None)
    out = {"q_out": TOKENS * Q_HEADS * DIM * 2, "k_out": TOKENS * K_HEADS * DIM * 2}
    each_pair(call, out, {**ROWS, **out})


@pytest.mark.parametrize("mx", [False, True])
def test_append_writes_nothing_that_it_reads(host, lib, mx):
    """The queries, and every tensor of the cache."""
    import kv_cache
    import rotary

    def call(**kw):
        a, r, x = rotation(rotary, kw)
        return lib.vramc_rotary_append(r, x, cache_of(kv_cache, a, mx), a["v"], 400, DIM, a["slots"], a["q_out"], None)
    read = {**ROWS, "v": ((TOKENS - 1) * 400 + K_HEADS * DIM) * 2, "slots": TOKENS * 8}
    pages = CACHE_MX if mx else CACHE
    each_pair(call, {"q_out": TOKENS * Q_HEADS * DIM * 2}, {**read, **pages})
    each_pair(call, pages, read)


def test_append_of_the_cache_s_own_rows(host):
    cache, _, turn = host
    x, n = torch.zeros(8, 2, 64), torch.zeros(8, dtype=torch.int32)
    slots, own = torch.arange(8), cache.v[:, :, 3]
    for q, k, v in ((x, x, own), (x, own, x), (own, x, x)):
        with pytest.raises(ValueError, match="memory"):
            turn.append(cache, q, k, v, slots, n)
    with pytest.raises(ValueError, match="memory"):
        turn.append(cache, x, x, x, slots, cache.position.view(-1)[:8])


@pytest.mark.parametrize("mx", [False, True])
def test_bound_writes_nothing_that_it_reads(host, lib, mx):
    import kv_cache

    def call(**kw):
        a = {**at, **kw}
        return lib.vramc_kv_bound(cache_of(kv_cache, a, mx), a["list"], 12, a["bounds"], None)
    each_pair(call, {"bounds": PAGES * K_HEADS * 2 * DIM * 2}, {"list": 48, **(CACHE_MX if mx else CACHE)})


@pytest.mark.parametrize("turned", [False, True])
def test_select_writes_nothing_that_it_reads(host, lib, turned):
    """Three sequences, 900 entries in rows 1000 apart, scored in a launch of their own;
    the queries' sequences may come in either order."""
    import kv_cache
    need = lib.vramc_kv_select_workspace(cache_of(kv_cache, at, False), Q_HEADS, 900, 3, 8)
    assert need == 3 * K_HEADS * 900 * 8
    last = 2 * 400 if turned else 0

    def call(**kw):
        a = {**at, **kw}
        return lib.vramc_kv_select(cache_of(kv_cache, a, False), a["bounds"], a["q"] + 2 * last, -400 if turned else 400,
                                   DIM, Q_HEADS, a["table"], 1000, 900, a["lengths"], 3, 8, 1, 1, a["chosen"], a["held"],
                                   a["work"], need, None)
    out = {"chosen": 3 * K_HEADS * 8 * 4, "held": 3 * K_HEADS * 4, "work": need}
    each_pair(call, out, {"bounds": PAGES * K_HEADS * 2 * DIM * 2, "q": (2 * 400 + Q_HEADS * DIM) * 2,
                          "table": (2 * 1000 + 900) * 4, "lengths": 12, **out})


# Three sequences in rows of 8 entries, 12 apart, 40 rows of tokens, 64 pages.
POOL = {"free": 64 * 4, "count": 4, "ticket": 4}
TABLE = {"table": (2 * 12 + 8) * 4}


def pool_of(kv_pages, a):
    return ctypes.byref(kv_pages.PagesDesc(64, 16, a["free"], a["count"], a["ticket"]))


def test_extend_writes_nothing_twice(host, lib):
    """Outputs, the table and the pool's tensors over what is read and over each other."""
    import kv_pages

    def call(**kw):
        a = {**at, **kw}
        return lib.vramc_pages_extend(pool_of(kv_pages, a), a["table"], 12, 8, a["lengths"], a["fresh"], a["seen"], 3, 40,
                                      a["slots"], a["positions"], a["filled"], a["starts"], a["grown"], None)
    out = {"slots": 320, "positions": 160, "filled": 160, "starts": 16, "grown": 12, **TABLE, **POOL}
    each_pair(call, out, {"lengths": 12, "fresh": 12, "seen": 12, **out})


def test_release_writes_nothing_twice(host, lib):
    import kv_pages

    def call(**kw):
        a = {**at, **kw}
        return lib.vramc_pages_release(pool_of(kv_pages, a), a["table"], 12, 8, a["lengths"], 3, a["work"], 16, None)
    out = {"work": 16, **TABLE, **POOL}
    each_pair(call, out, {"lengths": 12, **out})


def test_a_pool_of_one_tensor(host):
    """Free pages and their count in the same memory."""
    import kv_pages
    pool = host[1]
    free = torch.arange(8, dtype=torch.int32)
    table, n = torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    pool._desc = kv_pages.PagesDesc(8, 16, free.data_ptr(), free[7:].data_ptr(), pool._ticket.data_ptr())
    pool._ref = ctypes.byref(pool._desc)
    for call in (lambda: pool.extend(table, n, n, 5), lambda: pool.release(table, n)):
        with pytest.raises(ValueError, match="memory"):
            call()
