"""Steps of attention layers over pages that their queries choose, fewer than there are:
the choice is the formula's over the keys that the cache holds, and the output dense
attention over its tokens.  And a captured step of the pool, ordered behind what its
tensors were filled by."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def bench(rans):
    import rans_bench
    return rans_bench


def turned(x, positions):
    """RMS norms of each head (weights of one, eps 1e-6) and the rotation, in 64 bits on
    the CPU, rounded as the layer does."""
    y = x.double().cpu()
    y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + 1e-6)
    angle = positions.double()[:, None, None] * 1e6 ** (-torch.arange(0, 128, 2, dtype=torch.float64) / 128)
    a, b = y.chunk(2, -1)
    return torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()), -1).to(x.dtype)


def projected(layer, h, positions):
    x = torch.nn.functional.rms_norm(h, h.shape[-1:])
    q, k, v = (p(x).view(h.shape[0], -1, 128) for p in (layer.q_proj, layer.k_proj, layer.v_proj))
    return turned(q, positions), turned(k, positions), v.cpu()


def choice(c, q, row, n, count):
    """For each kv head the numbers of the sequence's pages: the first, the last, and
    those of the largest scores by the keys that lie in them, in f64."""
    pages = -(-n // c.page_size)
    k = c.k[row[:pages].long()].double().cpu()  # pages, kv heads, places, dim
    low, high = k.amin(2), k.amax(2)
    picks = []
    for h, group in enumerate(q.double().cpu().unflatten(0, (c.kv_heads, -1))):
        score = torch.stack([torch.maximum(x * low[:, h], x * high[:, h]).sum(1) for x in group]).amax(0)
        forced = (torch.arange(pages) == 0) | (torch.arange(pages) == pages - 1)
        order = np.lexsort((np.arange(pages), -score.numpy(), ~forced.numpy()))
        picks.append(sorted(order[:count].tolist()))
    return picks


@pytest.mark.parametrize("count,new", [(3, [100, 7, 161]), (5, [1, 250, 95]), (2, [64, 80, 48])])
def test_steps_over_chosen_pages(bench, count, new, monkeypatch):
    """bf16 pages; the output as near dense attention as a layer over all pages is held
    to, 2^-6 for the roundings of projections, keys, queries and outputs."""
    import kv_cache
    page = 16
    stack = bench.AttentionStack(layers=2, batch=3, budget=288, slack=32, page=page, mx=False, track=False, pooled=True,
                                 turned=True, count=count)
    chosen, ins, outs = [], [], []
    plain = kv_cache.PagedCache.select

    def select(self, q, table, lengths, *args):
        result = plain(self, q, table, lengths, *args)
        chosen.append((self, q.clone(), table.clone(), lengths.tolist(), result[0].clone(), result[1].tolist()))
        return result
    monkeypatch.setattr(kv_cache.PagedCache, "select", select)
    for layer in stack.layers:
        layer.register_forward_hook(lambda m, args, out: (ins.append(args[0].clone()), outs.append(out.clone()), None)[2])
    torch.manual_seed(7)
    h = torch.randn(sum(new), 1536, device="cuda").bfloat16()
    stack.write(h, new)
    past = [[[] for _ in new] for _ in stack.layers]
    with torch.no_grad():
        at = torch.cat([torch.arange(n) for n in new])
        for layer, p in zip(stack.layers, past):
            _, k, v = projected(layer, h, at)
            for rows, keys, values in zip(p, k.split(new), v.split(new)):
                rows += list(zip(keys, values))
    fewer = 0
    for step in range(20):
        held = [n + step for n in new]
        chosen.clear(), ins.clear(), outs.clear()
        stack.step(torch.randn(3, 1536, device="cuda").bfloat16())
        assert len(chosen) == len(ins) == 2
        for layer, p, x, got, (c, q, table, lengths, pages, tokens) in zip(stack.layers, past, ins, outs, chosen):
            assert c is layer.cache and lengths == [n + 1 for n in held]
            with torch.no_grad():
                q_want, k, v = projected(layer, x, torch.tensor(held))
            attended = []
            for b, rows in enumerate(p):
                rows.append((k[b], v[b]))
                n = len(rows)
                picks = choice(c, q[b], table[b], n, count)
                fewer += len(picks[0]) < -(-n // page)
                keys, values = (torch.stack([t[i] for t in rows], 1).double() for i in range(2))  # kv, tokens, dim
                for head, pick in enumerate(picks):
                    row = pages[2 * b + head].tolist()
                    numbers = table[b].tolist()
                    assert row == [numbers[i] * 2 + head for i in pick] + [-1] * (len(row) - len(pick)), (step, b, head)
                    in_them = [t for i in pick for t in range(i * page, min(n, (i + 1) * page))]
                    assert tokens[2 * b + head] == len(in_them)
                    w = torch.softmax(q_want[b].double().unflatten(0, (2, -1))[head] @ keys[head, in_them].T / 128 ** 0.5, -1)
                    attended.append((w @ values[head, in_them]).flatten())
            with torch.no_grad():
                want = x + layer.o_proj(torch.stack(attended).view(3, -1).to(x.dtype).cuda())
            off = float((got - want).double().norm() / (want - x).double().norm())
            assert off <= 2.0 ** -6, (step, off)
    assert fewer > 20  # most steps had pages to leave out


def test_a_pool_s_step_in_a_graph(rans):
    """Its first calls, on a stream that waits for the one that filled the tensors, and
    replays against eager calls on a pool of their own."""
    import kv_pages

    def make():
        return kv_pages.PagePool(900, 16), torch.full((40, 30), -1, dtype=torch.int32, device="cuda")
    (pool, table), (eager, own) = make(), make()
    lengths, new, keep = (torch.zeros(40, dtype=torch.int32, device="cuda") for _ in range(3))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        pool.extend(table, lengths, new, 3000)
        pool.release(table, keep)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step = pool.extend(table, lengths, new, 3000)
        pool.release(table, keep)
    rng, held = np.random.default_rng(4), [0] * 40
    for _ in range(4):
        lengths.copy_(torch.tensor(held, dtype=torch.int32))
        new.copy_(torch.from_numpy(rng.integers(0, 75, 40).astype(np.int32)))
        want = eager.extend(own, lengths, new, 3000)
        held = [max(0, n - int(rng.integers(0, 60))) for n in want.lengths.tolist()]
        keep.copy_(torch.tensor(held, dtype=torch.int32))
        eager.release(own, keep)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(step, want):
            assert torch.equal(x, y)
        assert torch.equal(table, own) and torch.equal(pool.count, eager.count)
        n = int(pool.count)
        assert torch.equal(pool.free[:n], eager.free[:n])
