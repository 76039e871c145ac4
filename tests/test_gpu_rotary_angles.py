"""f32 rows keep the angle's bits beyond 32: cosines next to a quarter turn, sines next to
a half, whose value is what the rounding of an angle would change.

Tolerance, relative.  At d turns (2^-20 to 2^-6) from the quarter the value is 2 pi d (1 +
d^2 ..), the rest's rounding at most 2^-26 turns, 2^-6 of it, which is put back to its
first order (the second is below 2^-40 / d, 2^-20 of that).  The functions are off by a few
units of 2^-23 (4 are taken), what is put back by 3 roundings of 2^-24 of at most 2^-6,
the sum and two products by one each: under 6 * 2^-23, and 2^-20 is allowed.  Without
what is put back it is off by up to 2^-6."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 96, 256])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("position", [1, -1, 3, 40001])
def test_angles_next_to_quarter_turns(rans, dim, interleaved, position):
    import kv_cache
    import rotary
    half = dim // 2
    g = torch.Generator().manual_seed(dim)
    d = torch.exp2(-6 - 14 * torch.rand(half, generator=g, dtype=torch.float64))
    quarter = torch.randint(-1, 3, (half,), generator=g).double() / 4
    sign = torch.randint(0, 2, (half,), generator=g) * 2 - 1
    inverse = 2 * math.pi * (quarter + d * sign + torch.randint(0, 1 if abs(position) < 9 else 2, (half,), generator=g)) / position
    turn = rotary.Rotary(dim, inverse=inverse, interleaved=interleaved)
    a, b = (slice(0, dim, 2), slice(1, dim, 2)) if interleaved else (slice(0, half), slice(half, dim))
    x = torch.zeros(5, 3, dim, device="cuda")
    x[..., a] = 1.0  # cosines into these, sines into the others
    at = torch.full((5,), position, dtype=torch.int32, device="cuda")
    angle = position * inverse
    want = torch.zeros(dim, dtype=torch.float64)
    want[a], want[b] = angle.cos(), angle.sin()
    cache = kv_cache.PagedCache.allocate(1, 3, dim, 16, torch.float32)
    slots = torch.arange(5, device="cuda")
    q, k = turn.rotate(x, x, at)
    again = turn.append(cache, x, x, x, slots, at)
    for got in (q, k, again, cache.read(slots)[0]):
        off = (got.double().cpu() - want).abs() / want.abs()
        assert (off <= 2.0 ** -20).all(), float(off.max())
