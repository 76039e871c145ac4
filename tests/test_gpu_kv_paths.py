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


@pytest.mark.parametrize("dtype,mx,group,track", [("bf16", False, 3, True), ("bf16", True, 5, False),
                                                  ("f16", True, 1, True), ("f32", False, 2, False),
                                                  ("f16", False, 18, True)])
def test_attend_more_sequences_than_threads(kv, dtype, mx, group, track):
    """600 and 1100 sequences, empty ones among them and at both ends: a thread
    of a workgroup counts several, and a share begins in any of them."""
    import test_gpu_kv_cache as T
    for batch in (600, 1100):
        rng = np.random.default_rng(batch)
        lengths = [0 if i < 3 or i > batch - 5 or rng.random() < 0.3 else int(rng.integers(1, 150)) for i in range(batch)]
        lengths[batch // 2] = 2500
        pages = sum(-(-n // 16) for n in lengths)
        c = T.make(kv, dtype, mx, 64, 16, 2, pages, seed=batch, track=track)
        table, n = T.tables(lengths, 16, pages, seed=batch)
        q = torch.randn(batch, 2 * group, 64, device="cuda").to(T.DTYPES[dtype])
        got = T.check_attend(kv, c, dtype, q, table, n)
        assert torch.equal(c.attend(q, table, n), got)


@pytest.mark.parametrize("dtype,mx", [("bf16", False), ("f16", False), ("f32", False), ("bf16", True), ("f16", True)])
@pytest.mark.parametrize("dim,group", [(64, 2), (96, 2), (192, 2), (256, 2), (64, 24), (96, 24), (128, 24),
                                       (192, 32), (256, 40)])
def test_attend_joins_many_parts(kv, dtype, mx, dim, group):
    """One sequence for many workgroups: every width's join, of 16 heads and of 32."""
    import test_gpu_kv_cache as T
    c = T.make(kv, dtype, mx, dim, 32, 1, 110, seed=dim + group)
    table, n = T.tables([3500], 32, 110, seed=group)
    q = torch.randn(1, group, dim, device="cuda").to(T.DTYPES[dtype])
    T.check_attend(kv, c, dtype, q, table, n)


def test_4_bit_rounding_of_f16_at_its_edges(kv):
    """Ties, powers of two, saturation, subnormals, zeros and blocks that are not
    finite, for every exponent of f16."""
    import test_gpu_kv_cache as T
    base = np.array([0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6, 7, 7.5, 7.9921875, 0.5, 1, 1.5, 2, 3, 4, 0.2490234375,
                     0.251, 0.749, 0.751, 2.49, 2.51, 4.99, 5.01, 0.1, 0.01, 1e-3, 1e-5, 0, 0], np.float64)
    rows = [np.concatenate([base, -base[::-1]]) * 2.0 ** e for e in range(-26, 14)]
    rows += [np.concatenate([base / 2, np.full(32, 65504.0)]), np.full(64, 2.0 ** -24), np.full(64, -0.0)]
    x = torch.tensor(np.array(rows)).clamp(-65504, 65504).half()
    x[4, 3], x[6, 40], x[8, 0] = np.inf, np.nan, -np.inf
    tokens = len(rows)
    c = kv.PagedCache.allocate(-(-tokens // 16), 1, 64, 16, torch.float16, mx=True)
    x = x.cuda()[:, None]
    slots = torch.arange(tokens, device="cuda")
    c.append(x, x.flip(2), slots)
    k, v = c.read(slots)
    want = T.rounded(x.double().cpu().numpy())
    assert np.array_equal(T.opened(c, "k").transpose(0, 2, 1, 3).reshape(-1, 64)[:tokens], want[:, 0], equal_nan=True)
    want = torch.from_numpy(want).half().double().numpy()  # below f16's smallest step
    assert np.array_equal(k.double().cpu().numpy(), want, equal_nan=True)
    assert np.array_equal(v.flip(2).double().cpu().numpy(), want, equal_nan=True)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
def test_4_bit_blocks_that_are_nan_in_live_tokens(kv, dtype, dim):
    """A NaN block of keys spoils the outputs of its kv head and sequence, one of
    values its 32 columns there, and neither anything else."""
    import test_gpu_kv_cache as T
    c = T.make(kv, dtype, True, dim, 16, 2, 24, seed=dim)
    table, n = T.tables([150, 200], 16, 24, seed=dim)
    q = torch.randn(2, 6, dim, device="cuda").to(T.DTYPES[dtype])
    mass = c.mass.clone()
    want = c.attend(q, table, n)
    after = c.mass.clone()
    last = dim // 32 - 1
    c.v_scale[table[0, 3], 0, 5, last] = 255
    c.v_scale[table[1, 7], 1, 2, 0] = 255
    c.mass.copy_(mass)
    got = c.attend(q, table, n)
    spoiled = torch.zeros_like(got, dtype=torch.bool)
    spoiled[0, :3, 32 * last:] = spoiled[1, 3:, :32] = True
    assert torch.isnan(got[spoiled]).all() and torch.equal(got[~spoiled], want[~spoiled])
    assert torch.equal(c.mass, after)
    c.v_scale.clamp_(max=129)
    c.k_scale[table[0, 0], 1, 0, last] = 255
    c.mass.copy_(mass)
    got = c.attend(q, table, n)
    spoiled.zero_()
    spoiled[0, 3:] = True
    # what the new block's scale of 129 in place of the old one changes is in no other row
    same = torch.ones_like(spoiled)
    same[0] = same[1, 3:] = False
    assert torch.isnan(got[spoiled]).all() and torch.isfinite(got[~spoiled]).all()
    assert torch.equal(got[same], want[same])
    theirs = torch.zeros_like(c.mass, dtype=torch.bool)
    theirs[table[0, :10].long(), 1] = True
    assert torch.equal(c.mass[~theirs], after[~theirs])
    place = torch.arange(160, device="cuda").view(10, 16) < 150
    assert torch.isnan(c.mass[table[0, :10].long(), 1][place]).all()
    assert torch.equal(c.mass[table[0, :10].long(), 1][~place], mass[table[0, :10].long(), 1][~place])


@pytest.mark.parametrize("dtype,mx", [("bf16", False), ("f16", False), ("f32", False), ("bf16", True), ("f16", True)])
@pytest.mark.parametrize("dim,group", [(64, 4), (128, 20)])
@pytest.mark.parametrize("octaves", [14, 22, 27, 31])
def test_attend_light_tokens_alone_in_a_column(kv, dtype, mx, dim, group, octaves):
    """The heavy tokens' values are zero, so that outputs are what tokens of
    2^-octaves of their weight add up to: those keep their bits too."""
    import test_gpu_kv_cache as T
    page, pages, length = 32, 8, 230
    c = T.make(kv, dtype, mx, dim, page, 1, pages, seed=octaves, track=False)
    table, n = T.tables([length], page, pages, seed=octaves)
    g = torch.Generator(device="cuda").manual_seed(octaves)
    score = -octaves * np.log(2.0) - torch.rand(length, device="cuda", generator=g)
    heavy = torch.randperm(length, device="cuda", generator=g)[:5]
    score[heavy] = 0
    k = torch.zeros(length, 1, dim, device="cuda")
    k[:, 0, 0] = score
    v = 2 + 4 * torch.rand(length, 1, dim, device="cuda", generator=g)
    if dtype != "bf16":
        v = v * 2.0 ** 13 * torch.where(torch.rand(v.shape, device="cuda", generator=g) < 0.5, -1, 1)
    v[heavy] = 0
    slots = c.slots(table, torch.zeros(length, device="cuda"), torch.arange(length, device="cuda"))
    c.append(k.to(T.DTYPES[dtype]), v.to(T.DTYPES[dtype]), slots)
    q = torch.zeros(1, group, dim, device="cuda").to(T.DTYPES[dtype])
    q[..., 0] = 1
    T.check_attend(kv, c, dtype, q, table, n, scale=1.0)
