"""Paths of the key-value cache's kernels that only certain sizes reach, each
against a plain implementation in 64 bits."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv(rans):
    import kv_cache
    return kv_cache


@pytest.mark.parametrize("length", [32768, 32769, 65537, 140000])
@pytest.mark.parametrize("budget_of", [lambda n: n - 3, lambda n: n // 2, lambda n: 700])
def test_evict_in_pieces(kv, length, budget_of):
    """Keys that are held at once and keys that go through in pieces, every
    digit of them: masses differ in their last bits only, or are one of few."""
    budget, page = budget_of(length), 128
    pages = -(-length // page)
    for seed, few in ((0, False), (1, True)):
        g = torch.Generator(device="cuda").manual_seed(length + seed)
        c = kv.PagedCache.allocate(pages, 2, 64, page, torch.float16, mx=True, track=True)
        c.k.copy_(torch.randint(0, 256, c.k.shape, device="cuda", generator=g))
        bits = torch.randint(0, 4 if few else 5000, c.mass.shape, device="cuda", generator=g)
        c.mass.copy_((bits + 0x3f800000).int().view(torch.float32))
        c.position.copy_(torch.arange(pages * page, device="cuda").view(pages, 1, page).expand_as(c.mass))
        table = torch.randperm(pages, device="cuda", generator=g).int()[None]
        n = torch.tensor([length], dtype=torch.int32, device="cuda")
        mass, position, k = (getattr(c, w)[table[0].long()].transpose(0, 1).flatten(1, 2).cpu().numpy()
                             for w in ("mass", "position", "k"))
        assert c.evict(table, n, n, budget, 100).tolist() == [budget]
        got = [getattr(c, w)[table[0].long()].transpose(0, 1).flatten(1, 2).cpu().numpy()
               for w in ("mass", "position", "k")]
        for h in range(2):
            recent = position[h, :length] >= length - 100
            order = np.lexsort((np.arange(length), -mass[h, :length].astype(np.float64), ~recent))
            kept = np.sort(order[:budget])
            at = np.arange(budget)
            at[np.setdiff1d(at, kept)] = kept[kept >= budget]
            for x, y in zip((mass, position, k), got):
                assert np.array_equal(y[h, :budget], x[h][at])


def test_attend_in_a_compiled_program(kv):
    """A compiled program breaks at the call and makes it; a traced one is
    refused, as it would go on without the kernel."""
    c = kv.PagedCache.allocate(8, 2, 64, 16, torch.bfloat16)
    c.k.normal_()
    c.v.normal_()
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    n = torch.tensor([50, 20], dtype=torch.int32, device="cuda")
    q = torch.randn(2, 6, 64, device="cuda").bfloat16()
    want = c.attend(q * 2, table, n) + 1
    run = torch.compile(lambda q: c.attend(q * 2, table, n) + 1, backend="eager")
    for _ in range(3):
        assert torch.equal(run(q), want)
    with pytest.raises(ValueError):
        torch.jit.trace(lambda q: c.attend(q, table, n) + 1, (q,), check_trace=False)


@pytest.mark.parametrize("dtype,mx,dim", [(torch.float32, False, 64), (torch.float32, False, 96),
                                          (torch.bfloat16, False, 192), (torch.float16, True, 96),
                                          (torch.bfloat16, True, 256)])
def test_caches_aligned_to_16_bytes_only(kv, dtype, mx, dim):
    """What a cache's tensors have to be aligned to, and no more: every operation
    gives what it gives on tensors of their own."""
    heads, page, pages = 2, 16, 9

    def off(shape, dt):  # 16 bytes behind an address of 512
        n = int(np.prod(shape)) * dt.itemsize
        t = torch.zeros(n + 16, dtype=torch.uint8, device="cuda")[16:]
        assert t.data_ptr() % 32 == 16
        return t.view(dt).view(shape)

    a = kv.PagedCache.allocate(pages, heads, dim, page, dtype, mx=mx, track=True)
    names = [w for w in ("k", "v", "k_scale", "v_scale", "mass", "position") if getattr(a, w) is not None]
    b = kv.PagedCache(**{w: off(tuple(getattr(a, w).shape), getattr(a, w).dtype) for w in names}, dtype=dtype)
    g = torch.Generator(device="cuda").manual_seed(dim)
    k, v = (torch.randn(100, heads, dim, device="cuda", generator=g).to(dtype) for _ in range(2))
    q = torch.randn(2, 6, dim, device="cuda", generator=g).to(dtype)
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:100]
    at = torch.arange(100, dtype=torch.int32, device="cuda")
    order = torch.randperm(pages, device="cuda", generator=g).int()
    table, into = order[:8].view(2, 4), order[8:].view(1, 1)
    n = torch.tensor([60, 33], dtype=torch.int32, device="cuda")
    got = []
    for c in (a, b):
        c.append(k, v, slots, at)
        got.append([*c.read(slots), c.attend(q, table, n), c.evict(table[:1], n[:1], n[:1], 9, 3, into),
                    c.evict(table, n, n, 30, 7)] + [getattr(c, w) for w in names])
    for x, y in zip(*got):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dim,heads", [(96, 8), (192, 4), (256, 4)])
def test_attend_in_f32_is_as_exact_as_f32(kv, dim, heads):
    """The error against 64 bits, in the 2-norm, is at most half again that of
    elementary f32 operations on the same numbers."""
    for seed in range(4):
        g = torch.Generator(device="cuda").manual_seed(seed)
        c = kv.PagedCache.allocate(3 * 56, heads, dim, 32, torch.float32)
        c.k.normal_(generator=g)
        c.v.normal_(generator=g)
        table = torch.randperm(3 * 56, device="cuda", generator=g).int().view(3, 56)
        n = torch.tensor([1777, 1500, 900], dtype=torch.int32, device="cuda")
        q = 2 * torch.randn(3, heads, dim, device="cuda", generator=g)
        got = c.attend(q, table, n).double()
        far = torch.zeros(2, dtype=torch.float64, device="cuda")
        for b in range(3):
            k, v = (x[table[b].long()].transpose(0, 1).flatten(1, 2)[:, :int(n[b])] for x in (c.k, c.v))

            def plain(t):
                w = torch.softmax((q[b].to(t)[:, None] @ k.to(t).transpose(1, 2).contiguous()) * dim ** -0.5, -1)
                return (w @ v.to(t))[:, 0].double()

            want = plain(torch.float64)
            far += torch.stack([(got[b] - want).square().sum(), (plain(torch.float32) - want).square().sum()])
        own, elementary = far.sqrt().tolist()
        assert own <= 1.5 * elementary, (seed, own / elementary)
