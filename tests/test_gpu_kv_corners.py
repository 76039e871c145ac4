"""Scores of pages are sums over the corner of the bounds that a query points to, and
nothing of the other corner: pages alike in the first have the same score to the bit, so
that the lower index is taken, and a far other corner loses nothing."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
PAGE, HEADS = 16, 2
# query heads of a kv head and entries of the table: scored where they are chosen from, by
# vectors, and by the matrix cores
SHAPES = [(64, 1, 190), (64, 8, 400), (64, 9, 190), (96, 5, 90), (128, 5, 90), (128, 1, 300), (128, 6, 1000),
          (128, 17, 300), (192, 3, 47), (256, 8, 200), (256, 40, 200)]


@pytest.fixture(scope="module")
def kv(rans):
    import kv_cache
    return kv_cache


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make(kv, dim, pages, dtype):
    """A cache whose bounds are given, a table of all its pages, and full lengths."""
    c = kv.PagedCache.allocate(pages, HEADS, dim, PAGE, dtype, bounds=True)
    order = torch.randperm(pages, device="cuda", generator=gen(pages)).int()
    return c, order[None], torch.full((1,), pages * PAGE, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dim,group,pages", SHAPES)
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_pages_alike_where_the_query_points(kv, dtype, dim, group, pages):
    """The same corner for all pages, the other one anywhere: every score is a tie."""
    t = DTYPES[dtype]
    c, table, n = make(kv, dim, pages, t)
    sign = torch.randint(0, 2, (HEADS, 1, dim), device="cuda", generator=gen(1)) * 2 - 1
    q = (torch.rand(HEADS, group, dim, device="cuda", generator=gen(2)) + 0.01) * sign
    corner = torch.randn(HEADS, dim, device="cuda", generator=gen(3))
    away = torch.exp(3 * torch.randn(pages, HEADS, dim, device="cuda", generator=gen(4))).clamp(max=1000.0)
    up = (sign[:, 0] > 0).expand(pages, -1, -1)
    c.bounds[:, :, 0] = torch.where(up, corner - away, corner).to(t)
    c.bounds[:, :, 1] = torch.where(up, corner, corner + away).to(t)
    for count in (2, 3, 17, pages // 2, pages - 1):
        chosen, held = c.select(q.view(1, -1, dim).to(t), table, n, count, 0, 1)
        at = torch.cat((table[0, :count - 1], table[0, -1:]))
        want = at[None] * HEADS + torch.arange(HEADS, dtype=torch.int32, device="cuda")[:, None]
        assert torch.equal(chosen, want), count
        assert held.tolist() == [count * PAGE] * HEADS


@pytest.mark.parametrize("dim,group,pages", SHAPES)
@pytest.mark.parametrize("dtype,far", [("bf16", 2.0 ** 60), ("f32", 2.0 ** 100), ("f16", 2.0 ** 15)])
@pytest.mark.parametrize("side", [1, -1])
def test_a_far_other_corner(kv, dtype, far, dim, group, pages, side):
    """Scores are dim times a small whole number of each page's, whatever lies on the
    other side of zero; the largest are taken."""
    t = DTYPES[dtype]
    c, table, n = make(kv, dim, pages, t)
    height = torch.randint(1, 60, (pages, HEADS), device="cuda", generator=gen(5))
    c.bounds[:, :, 0 if side > 0 else 1] = -side * far
    c.bounds[:, :, 1 if side > 0 else 0] = (side * height)[..., None].to(t)
    q = torch.full((1, HEADS * group, dim), float(side), device="cuda").to(t)
    score = height[table[0].long()].T.cpu()  # of a kv head's pages in the table's order
    for count in (2, 9, pages // 3 + 2):
        chosen, _ = c.select(q, table, n, count, 0, 1)
        for h in range(HEADS):
            best = torch.sort(score[h, :-1], descending=True, stable=True).indices[:count - 1].sort().values.tolist()
            assert chosen[h].tolist() == [int(table[0, i]) * HEADS + h for i in best + [pages - 1]], (h, count)
