"""Everything around the cache where it is used: steps of attention layers with
rANS-coded projections, norms and rotary positions, pages from a pool and chosen by
queries, against dense attention over all past tokens."""
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
    inverse = 1e6 ** (-torch.arange(0, 128, 2, dtype=torch.float64) / 128)
    angle = positions.double().cpu()[:, None, None] * inverse
    a, b = y.chunk(2, -1)
    return torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()), -1).to(x.dtype)


def projected(layer, h, positions):
    x = torch.nn.functional.rms_norm(h, h.shape[-1:])
    q, k, v = (p(x).view(h.shape[0], -1, 128) for p in (layer.q_proj, layer.k_proj, layer.v_proj))
    return turned(q, positions), turned(k, positions), v.cpu()


def dense(layer, h, past):
    """The layer's step with each sequence's past as plain tensors, attention in f64."""
    q, k, v = projected(layer, h, torch.tensor([len(p) for p in past], device="cuda"))
    out = []
    for b, p in enumerate(past):
        p.append((k[b], v[b]))
        keys, values = (torch.stack([t[i] for t in p], 1).double() for i in range(2))  # kv, tokens, dim
        w = torch.softmax(q[b].double().unflatten(0, (2, -1)) @ keys.transpose(-1, -2) / 128 ** 0.5, -1)
        out.append((w @ values).flatten())
    return h + layer.o_proj(torch.stack(out).to(h.dtype).cuda())


def pages_are_whole(stack):
    """Every page is in the pool or in one place of the table, none twice."""
    free = stack.pool.free[:int(stack.pool.count)].tolist()
    held = stack.table[stack.table >= 0].tolist()
    assert sorted(free + held) == list(range(stack.pool.pages))
    page = stack.layers[0].cache.page_size
    for row, n in zip(stack.table.tolist(), stack.lengths.tolist()):
        assert [x >= 0 for x in row] == [i < -(-n // page) for i in range(len(row))]


def bounds_are_of_keys(stack):
    """Of all pages but each sequence's last."""
    for layer in stack.layers:
        c = layer.cache
        for row, n in zip(stack.table.tolist(), stack.lengths.tolist()):
            at = row[:max(0, -(-n // c.page_size) - 1)]
            k = c.k[at]
            assert torch.equal(c.bounds[at], torch.stack((k.amin(2), k.amax(2)), 2))


@pytest.mark.parametrize("count", [0, 9])
def test_steps_match_dense_attention(bench, count):
    """Prompts of different lengths, then tokens; with as many pages chosen as there are.
    bf16 pages give what dense attention gives to a few roundings of 2^-8 (the
    projections' inputs, queries, keys, outputs) through two layers, as the plain steps
    are held to."""
    stack = bench.AttentionStack(layers=2, batch=3, budget=128, slack=64, page=16, mx=False, track=False, pooled=True,
                                 turned=True, count=count)
    torch.manual_seed(1)
    new = [37, 1, 90]
    h = torch.randn(sum(new), 1536, device="cuda").bfloat16()
    stack.write(h, new)
    past = [[[] for _ in new] for _ in stack.layers]
    with torch.no_grad():
        at = torch.cat([torch.arange(n) for n in new]).cuda()
        for layer, p in zip(stack.layers, past):
            _, k, v = projected(layer, h, at)
            for rows, keys, values in zip(p, k.split(new), v.split(new)):
                rows += list(zip(keys, values))
    for step in range(20):
        h = torch.randn(3, 1536, device="cuda").bfloat16()
        got, want = stack.step(h), h
        with torch.no_grad():
            for layer, p in zip(stack.layers, past):
                want = dense(layer, want, p)
        off = float((got - want).double().norm() / (want - h).double().norm())
        assert off <= 2 * 2.0 ** -6, (step, off)
    assert stack.lengths.tolist() == stack.seen.tolist() == [n + 20 for n in new]
    pages_are_whole(stack)
    if count:
        bounds_are_of_keys(stack)


@pytest.mark.parametrize("pooled", [False, True])
def test_eviction_and_chosen_pages(bench, pooled):
    """Steps past the budget, attention over a few pages: evicted layers keep their
    newest tokens, and the bounds follow what has moved."""
    stack = bench.AttentionStack(layers=2, batch=2, budget=64, slack=32, recent=24, page=16, mx=False, pooled=pooled,
                                 turned=True, count=4)
    torch.manual_seed(2)
    for step in range(150):
        out = stack.step(torch.randn(2, 1536, device="cuda").bfloat16())
        assert stack.lengths.tolist() == [stack.held] * 2 and stack.held < 96
        if step % 10 == 7 or stack.held == 64:
            bounds_are_of_keys(stack)
            if pooled:
                pages_are_whole(stack)
    assert torch.isfinite(out).all() and stack.seen.tolist() == [150, 150]
    c = stack.layers[0].cache
    for b in range(2):
        at = c.position[stack.table[b].clamp(min=0).long()].transpose(0, 1).flatten(1)[:, :stack.held]
        for held in at.tolist():
            assert len(set(held)) == stack.held and set(range(127, 150)) <= set(held)


def test_sequences_come_and_go(bench):
    """A row that ends gives its pages to the next prompts; what a full pool refuses
    leaves the others as they are, and a step after it is that of a fresh stack."""
    make = lambda: bench.AttentionStack(layers=1, batch=3, budget=96, slack=16, page=16, mx=False, track=False,  # noqa: E731
                                        pooled=True, turned=True, count=3)
    stack, fresh = make(), make()
    for a, b in zip(stack.layers, fresh.layers):
        b.load_state_dict(a.state_dict())
        for name in ("q_proj", "k_proj", "v_proj", "o_proj"):
            setattr(b, name, getattr(a, name))
    torch.manual_seed(3)
    first = torch.randn(200, 1536, device="cuda").bfloat16()
    stack.write(first, [96, 90, 14])
    pages_are_whole(stack)
    stack.finish([0, 2])
    assert stack.lengths.tolist() == [0, 90, 0]
    pages_are_whole(stack)
    stack.held = 90
    stack.pool.count.fill_(int(stack.pool.count) - 8)  # as if another table held them
    again = torch.randn(80, 1536, device="cuda").bfloat16()
    stack.write(again, [40, 0, 40])
    stack.write(again[:64], [0, 0, 64])  # more than is left
    assert stack.lengths.tolist() == stack.seen.tolist() == [40, 90, 40]
    fresh.write(torch.cat((again[:40], first[96:186], again[40:])), [40, 90, 40])
    h = torch.randn(3, 1536, device="cuda").bfloat16()
    assert torch.equal(stack.step(h), fresh.step(h))


def test_rows_used_again_are_evicted_in_time(bench):
    """Prompts in rows that others have left: the budget holds for what a row holds now,
    not for all that it ever has, and no token is refused."""
    stack = bench.AttentionStack(layers=1, batch=2, budget=64, slack=16, recent=8, page=16, mx=False, pooled=True)
    torch.manual_seed(5)
    prompt = torch.randn(120, 1536, device="cuda").bfloat16()
    for _ in range(3):
        stack.write(prompt[:90], [60, 30])
        stack.finish([0])
        stack.write(prompt[:60], [60, 0])
        stack.finish([0, 1])
    assert stack.held == 0 and int(stack.pool.count) == stack.pool.pages
    stack.write(prompt, [60, 60])
    want = 60
    for step in range(60):
        stack.step(prompt[:2])
        want = 64 if want == 79 else want + 1
        assert stack.lengths.tolist() == [want] * 2 and stack.held == want
    assert stack.seen.tolist() == [120] * 2
    pages_are_whole(stack)


def test_chosen_pages_need_filled(bench):
    """A layer that chooses pages by bounds is told which pages became full."""
    stack = bench.AttentionStack(layers=1, batch=1, budget=64, slack=16, page=16, mx=False, pooled=True, count=2)
    layer, h = stack.layers[0], torch.zeros(1, 1536, device="cuda", dtype=torch.bfloat16)
    room = stack.pool.extend(stack.table, stack.lengths, stack.one, 1)
    with pytest.raises(ValueError, match="filled"):
        layer(h, stack.table, room.lengths, room.slots, room.positions)
    assert not layer.cache.k.any() and not layer.cache.v.any()


def test_a_step_in_a_graph(bench):
    """A whole step of two layers, captured once and replayed with other tokens, lengths
    and pages, between eager work, against the same calls made eagerly."""
    stack = bench.AttentionStack(layers=2, batch=4, budget=200, slack=56, page=16, mx=False, track=False, pooled=True,
                                 turned=True, count=5)
    eager = bench.AttentionStack(layers=2, batch=4, budget=200, slack=56, page=16, mx=False, track=False, pooled=True,
                                 turned=True, count=5)
    for a, b in zip(stack.layers, eager.layers):
        for name in ("q_proj", "k_proj", "v_proj", "o_proj"):
            setattr(b, name, getattr(a, name))
    torch.manual_seed(4)
    new = [150, 3, 77, 16]
    prompt = torch.randn(sum(new), 1536, device="cuda").bfloat16()
    h = torch.zeros(4, 1536, device="cuda", dtype=torch.bfloat16)
    lengths, seen = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")

    @torch.no_grad()
    def step():
        room = stack.pool.extend(stack.table, lengths, stack.one, 4, seen)
        x = h
        for layer in stack.layers:
            x = layer(x, stack.table, room.lengths, room.slots, room.positions, room.filled)
        seen.add_(room.lengths - lengths)
        lengths.copy_(room.lengths)
        return x

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.synchronize()
    lengths.zero_()
    seen.zero_()
    stack.pool.release(stack.table, lengths)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for s in (stack, eager):
        s.write(prompt, new)
    lengths.copy_(stack.lengths)
    seen.copy_(stack.seen)
    for _ in range(6):
        h.copy_(torch.randn(4, 1536, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager.step(h))
        assert lengths.tolist() == eager.lengths.tolist() and seen.tolist() == eager.seen.tolist()


def test_serve_command(bench):
    r = bench.serve(layers=1, batch=2, longest=700, count=4, steps=16)
    assert r["finite"] and r["free_pages"] < r["free_pages_at_the_end"]
