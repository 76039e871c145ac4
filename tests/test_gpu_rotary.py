"""Norms and rotation against the formula in 64 bits.

Tolerances.  A result is z = (x w c -+ x' w' s) r, rounded once to its type.  In f32
cosine and sine are off by 2^-22 (2^-24 of rounding the angle's rest, up to 2^-2 turns
and so 2 pi 2^-26 radians, and the functions' own last bits), r by 2^-21 (a sum of up
to 256 squares over eight lanes' values and five steps, the mean, an approximate
root), and the products and their sum by three roundings: together less than 2^-19 of
(|x w| + |x' w'|) r.  Rounding to T adds eps / 2 of the result."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


@pytest.fixture(scope="module")
def rotary(rans):
    import rotary
    return rotary


@pytest.fixture(scope="module")
def kv(rans):
    import kv_cache
    return kv_cache


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def values(seed, *shape, dtype=torch.bfloat16, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=gen(seed)) * scale).to(dtype)


def expected(x, positions, inverse, interleaved, weight, eps, amplitude=1.0):
    """The formula in 64 bits on the CPU, and the magnitude that errors go by."""
    y = x.double().cpu()
    if weight is not None:
        y = y * weight.double().cpu() / torch.sqrt(y.square().mean(-1, keepdim=True) + eps)
    angle = positions.double().cpu()[:, None, None] * inverse.double().cpu()
    c, s = angle.cos() * amplitude, angle.sin() * amplitude
    half = inverse.numel()
    z, size = y.clone(), y.abs()
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    z[..., a], z[..., b] = y[..., a] * c - y[..., b] * s, y[..., b] * c + y[..., a] * s
    both = amplitude * (y[..., a].abs() + y[..., b].abs())
    size[..., a], size[..., b] = both, both
    return z, size


def check(got, want, size):
    eps = torch.finfo(got.dtype).eps
    tiny = torch.finfo(got.dtype).tiny if got.dtype is torch.float16 else 0.0
    off = (got.double().cpu() - want).abs()
    allowed = eps / 2 * want.abs() + 2.0 ** -19 * size + tiny * eps
    assert torch.isfinite(got).all() and (off <= allowed).all(), float((off - allowed).max())


SIZES = [  # tokens, q heads, kv heads, dim, rotary columns, interleaved, dtype, norms, weights' dtype
    (1, 12, 2, 128, 128, False, "bf16", "qk", None), (1, 1, 1, 64, 64, False, "f16", "", None),
    (7, 40, 8, 128, 128, False, "bf16", "qk", "f32"), (33, 5, 3, 96, 96, False, "bf16", "q", None),
    (64, 7, 1, 64, 32, True, "f16", "k", "f32"), (17, 3, 2, 192, 64, False, "f32", "qk", None),
    (5, 9, 4, 256, 256, True, "f32", "", None), (1023, 3, 2, 96, 48, True, "bf16", "qk", None),
    (1024, 3, 2, 64, 16, False, "bf16", "qk", None), (1025, 2, 5, 256, 128, False, "f16", "qk", None),
    (2051, 6, 1, 192, 192, False, "bf16", "qk", None), (8193, 2, 1, 64, 64, False, "f16", "qk", "f32"),
    (8199, 1, 2, 128, 80, True, "f32", "q", None), (3, 100, 33, 128, 128, False, "bf16", "qk", None),
    (9000, 5, 3, 96, 96, False, "bf16", "", None),
]


@pytest.mark.parametrize("tokens,heads,kv_heads,dim,columns,interleaved,dtype,norms,weight", SIZES)
def test_rotate(rotary, tokens, heads, kv_heads, dim, columns, interleaved, dtype, norms, weight):
    t = DTYPES[dtype]
    q, k = values(tokens, tokens, heads, dim, dtype=t, scale=3.0), values(tokens + 1, tokens, kv_heads, dim, dtype=t)
    w = [(1 + 0.5 * values(i, dim, dtype=torch.float32)).to(DTYPES[weight or dtype]) if n in norms else None
         for i, n in enumerate("qk")]
    positions = torch.randint(-1000, 2 ** 20, (tokens,), device="cuda", generator=gen(5)).int()
    turn = rotary.Rotary(dim, 1e4, columns, interleaved)
    inverse = torch.tensor([1e4 ** (-2 * i / columns) for i in range(columns // 2)], dtype=torch.float64)
    before = q.clone(), k.clone()
    got = turn.rotate(q, k, positions, *w, eps=1e-5)
    assert torch.equal(q, before[0]) and torch.equal(k, before[1])
    for x, y, weight in zip((q, k), got, w):
        assert y.shape == x.shape and y.dtype is t and y.is_contiguous()
        check(y, *expected(x, positions, inverse, interleaved, weight, 1e-5))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("tokens", [3, 1500])
def test_strides(rotary, dtype, tokens):
    """Columns of one projection, rows that are not aligned, a dimension that is not
    dense, one row for all tokens."""
    t, turn = DTYPES[dtype], rotary.Rotary(64)
    inverse = torch.tensor([1e4 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64)
    w = values(9, 64, dtype=t)
    positions = torch.arange(tokens, dtype=torch.int32, device="cuda") * 7
    fused = values(1, tokens, 6, 64, dtype=t)
    odd = values(2, tokens, 6 * 64 + 3, dtype=t)[:, 1:385].unflatten(1, (6, 64))
    turned = values(3, 64, 6, tokens, dtype=t).permute(2, 1, 0)
    same = values(4, 1, 6, 64, dtype=t).expand(tokens, 6, 64)
    heads_first = values(5, 6, tokens, 64, dtype=t).transpose(0, 1)
    for x in (fused, odd, turned, same, heads_first):
        q, k = turn.rotate(x[:, :4], x[:, 4:], positions, w, w)
        check(q, *expected(x[:, :4], positions, inverse, False, w, 1e-6))
        check(k, *expected(x[:, 4:], positions, inverse, False, w, 1e-6))


def test_positions(rotary):
    """The smallest and largest positions, and what is the same at every one: angles are
    exact up to their last whole turn.  At 2^31 an angle in 64 bits is off by 2^31 *
    2^-53 radians, far below the tolerance; frequencies of 0 turn nothing."""
    at = torch.tensor([0, 1, -1, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda")
    q = values(1, 6, 2, 64, dtype=torch.float32)
    inverse = torch.tensor([1.0, 0.5, 1e-3, 0.0, 3.0, 2 * math.pi, 0.25, 1e-9], dtype=torch.float64)
    turn = rotary.Rotary(64, inverse=inverse, amplitude=1.25)
    got, k = turn.rotate(q, q, at)
    assert torch.equal(got, k)
    check(got, *expected(q, at, inverse, False, None, 0, 1.25))
    assert torch.equal(got[..., 16:], q[..., 16:])
    assert torch.equal(got[:, :, 3], q[:, :, 3] * 1.25)


@pytest.mark.parametrize("interleaved", [False, True])
def test_values_that_are_not_finite(rotary, interleaved):
    """Columns that do not rotate keep infinities and NaN; those that do pass them on
    within their pair; a norm passes them to its head alone."""
    x = values(1, 3, 4, 64, dtype=torch.float32)
    x[0, 0, 40], x[0, 1, 50], x[1, 2, 3] = math.inf, math.nan, -math.inf
    at = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")
    turn = rotary.Rotary(64, rotary_dim=32, interleaved=interleaved)
    got, _ = turn.rotate(x, x, at)
    bad = ~torch.isfinite(got)
    pair = [3, 2] if interleaved else [3, 19]
    want = torch.zeros_like(bad)
    want[0, 0, 40] = want[0, 1, 50] = True
    want[1, 2, pair] = True
    assert torch.equal(bad, want) and got[0, 0, 40] == math.inf
    ones = torch.ones(64, device="cuda")
    got, _ = turn.rotate(x, x, at, ones, ones)
    heads = torch.isfinite(got).all(-1)
    assert heads.sum() == 12 - 3 and not heads[0, 0] and not heads[0, 1] and not heads[1, 2]


def test_zeros_and_large_values(rotary):
    """A head of zeros stays zeros for a positive eps; bf16's and f16's largest values
    have a finite norm as long as f32 holds the sum of their squares."""
    turn, at = rotary.Rotary(128), torch.zeros(2, dtype=torch.int32, device="cuda")
    one = torch.ones(128, device="cuda")
    x = torch.zeros(2, 3, 128, device="cuda", dtype=torch.float16)
    x[1] = 65504.0
    q, k = turn.rotate(x, x, at, one, one)
    assert (q[0] == 0).all() and torch.equal(q[1], torch.ones_like(q[1])) and torch.equal(q, k)


def held(cache, slots):
    return cache.read(slots)


@pytest.mark.parametrize("tokens,heads,kv_heads,dim,columns,interleaved,dtype,mx,page", [
    (1, 12, 2, 128, 128, False, "bf16", True, 64), (16, 12, 2, 128, 128, False, "bf16", False, 64),
    (5, 7, 1, 64, 32, True, "f16", True, 16), (300, 4, 4, 96, 96, False, "f32", False, 32),
    (1030, 6, 3, 96, 48, True, "bf16", True, 16), (2047, 5, 1, 256, 256, False, "f16", True, 128),
    (1500, 2, 2, 192, 192, False, "bf16", False, 256), (4100, 3, 5, 64, 64, False, "f16", False, 64),
])
@pytest.mark.parametrize("track", [False, True])
def test_append_is_rotate_and_append(rotary, kv, tokens, heads, kv_heads, dim, columns, interleaved, dtype, mx, page, track):
    """Bit for bit what the two calls leave, with padding among the tokens and the
    rest of the cache as it was."""
    t = DTYPES[dtype]
    fused = values(tokens, tokens, heads + 2 * kv_heads, dim, dtype=t)
    q, k, v = fused.split((heads, kv_heads, kv_heads), 1)
    w = values(1, dim, dtype=t), values(2, dim, dtype=t)
    pages = -(-tokens // page) + 2
    caches = []
    for _ in range(2):
        c = kv.PagedCache.allocate(pages, kv_heads, dim, page, t, mx, track)
        for x in (c.k, c.v) + ((c.k_scale, c.v_scale) if mx else ()):
            x.fill_(3)
        if track:
            c.mass.fill_(5.0)
        caches.append(c)
    order = torch.randperm(pages * page, device="cuda", generator=gen(3))[:tokens]
    slots = torch.where(torch.rand(tokens, device="cuda", generator=gen(4)) < 0.1, -1, order)
    slots[0] = order[0]
    if tokens > 4:
        slots[3] = pages * page + 5  # no slot of the cache
    positions = torch.randint(0, 100000, (tokens,), device="cuda", generator=gen(5)).int()
    turn = rotary.Rotary(dim, 1e6, columns, interleaved)
    got = turn.append(caches[0], q, k, v, slots, positions, *w)
    want, turned = turn.rotate(q, k, positions, *w)
    caches[1].append(turned, v, slots, positions if track else None)
    assert torch.equal(got, want)
    for name in ("k", "v", "k_scale", "v_scale", "mass", "position"):
        x, y = (getattr(c, name) for c in caches)
        assert (x is None) == (y is None)
        assert x is None or torch.equal(x, y), name


def test_in_a_graph(rotary, kv):
    turn, c = rotary.Rotary(64), kv.PagedCache.allocate(9, 2, 64, 16)
    x = torch.zeros(40, 8, 64, dtype=torch.bfloat16, device="cuda")
    at = torch.zeros(40, dtype=torch.int32, device="cuda")
    slots = torch.arange(40, device="cuda")
    turn.append(c, x[:, :4], x[:, 4:6], x[:, 6:], slots, at)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = turn.append(c, x[:, :4], x[:, 4:6], x[:, 6:], slots, at)
    for i in range(3):
        x.copy_(values(i, 40, 8, 64))
        at.copy_(torch.arange(40, device="cuda") * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        want, k = turn.rotate(x[:, :4], x[:, 4:6], at)
        keys, v = c.read(slots)
        assert torch.equal(q, want) and torch.equal(keys, k) and torch.equal(v, x[:, 6:])


def test_empty_calls(rotary, kv):
    turn, c = rotary.Rotary(64), kv.PagedCache.allocate(2, 2, 64, 16)
    none = torch.empty(0, 2, 64, dtype=torch.bfloat16, device="cuda")
    at = torch.empty(0, dtype=torch.int32, device="cuda")
    q, k = turn.rotate(none, none, at)
    assert q.shape == none.shape and k.shape == none.shape
    assert turn.append(c, none, none, none, at.long(), at).shape == none.shape
    some = values(1, 3, 2, 64)
    q, k = turn.rotate(some[:, :0], some, torch.arange(3, dtype=torch.int32, device="cuda"))
    assert q.shape == (3, 0, 64) and k.shape == (3, 2, 64)


def test_refusals(rotary, kv):
    for bad in (dict(head_dim=80), dict(rotary_dim=24), dict(rotary_dim=256), dict(rotary_dim=0), dict(base=-1.0),
                dict(inverse=torch.ones(2, 8)), dict(inverse=torch.ones(5)), dict(inverse=torch.ones(8), rotary_dim=32),
                dict(device="cpu")):
        with pytest.raises(ValueError):
            rotary.Rotary(**{**dict(head_dim=128), **bad})
    turn, c = rotary.Rotary(64), kv.PagedCache.allocate(2, 2, 64, 16)
    x, at, w = values(1, 3, 2, 64), torch.arange(3, dtype=torch.int32, device="cuda"), values(2, 64)
    good = dict(q=x, k=x, positions=at, q_weight=w, k_weight=w)
    for bad in (dict(q=x[0]), dict(q=x.cpu()), dict(q=x.double()), dict(k=x.float()), dict(k=x[:2]), dict(k=x[..., :32]),
                dict(positions=at.long()), dict(positions=at[:2]), dict(q_weight=w[:32]), dict(k_weight=w.half()),
                dict(q_weight=w.float()), dict(q_weight=values(3, 72)[4:68]), dict(eps=-1.0), dict(eps=math.nan),
                dict(q=x.clone().requires_grad_()), dict(k_weight=w.clone().requires_grad_())):
        with pytest.raises(ValueError):
            turn.rotate(**{**good, **bad})
        if "q" not in bad or bad["q"].dtype is not torch.float64:
            with pytest.raises(ValueError):
                turn.append(**{**good, **bad}, cache=c, v=x, slots=at.long())
    for bad in (dict(v=x[:2]), dict(v=x.float()), dict(v=x.cpu()), dict(slots=at), dict(slots=at.long()[:2]),
                dict(k=x[:, :1]), dict(cache=kv.PagedCache.allocate(2, 2, 128, 16)),
                dict(cache=kv.PagedCache.allocate(2, 2, 64, 16, torch.float16))):
        with pytest.raises(ValueError):
            turn.append(**{**dict(good, cache=c, v=x, slots=at.long()), **bad})
