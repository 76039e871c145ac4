"""The cache where it is used: attention layers with rANS-coded projections,
token by token, against dense attention over all past tokens; and held at a
budget by eviction."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def bench(rans):
    import rans_bench
    return rans_bench


def dense(layer, h, past):
    """The layer's step with its past as plain tensors, attention in f64."""
    n = h.shape[0]
    x = torch.nn.functional.rms_norm(h, h.shape[-1:])
    q, k, v = (p(x).view(n, -1, 128) for p in (layer.q_proj, layer.k_proj, layer.v_proj))
    past.append((k, v))
    k, v = (torch.stack([t[i] for t in past], 2).double().cpu() for i in range(2))  # n, kv, tokens, dim
    q = q.double().cpu().unflatten(1, (2, -1))
    w = torch.softmax(q @ k.transpose(-1, -2) / 128 ** 0.5, -1)
    out = (w @ v).flatten(1, 2).to(h.dtype).cuda()
    return h + layer.o_proj(out.view(n, -1)), w.sum(2)


@pytest.mark.parametrize("mx", [False, True])
def test_steps_match_dense_attention(bench, mx):
    """Below the budget: bf16 pages give what dense attention gives, to a few
    roundings of 2^-8 through two layers; 4-bit pages to the error of values
    that are off by up to an eighth (a quarter where the largest saturate)."""
    stack = bench.AttentionStack(layers=2, batch=3, budget=128, slack=64, recent=16, page=16, mx=mx)
    past = [[], []]
    torch.manual_seed(1)
    for step in range(40):
        h = torch.randn(3, 1536, device="cuda").bfloat16()
        got, want = stack.step(h), h
        with torch.no_grad():
            for layer, p in zip(stack.layers, past):
                want, weight = dense(layer, want, p)
        off = float((got - want).double().norm() / (want - h).double().norm())
        assert off <= (0.25 if mx else 2 * 2.0 ** -6), (step, off)
    assert stack.lengths.tolist() == [40] * 3
    if not mx:  # the mass of a layer's tokens adds up to a share for every query head and step
        for layer in stack.layers:
            c = layer.cache
            for b in range(3):
                mass = c.mass[stack.table[b].long()].transpose(0, 1).flatten(1)[:, :40]
                assert torch.allclose(mass.sum(1), torch.full((2,), 6 * 40.0, device="cuda"), rtol=1e-4)


def test_steps_hold_the_budget(bench):
    """Beyond budget + slack tokens every layer is cut to the budget again: the
    newest tokens are all there, no token twice, and steps go on."""
    stack = bench.AttentionStack(layers=1, batch=2, budget=64, slack=16, recent=24, page=16)
    torch.manual_seed(2)
    for step in range(200):
        out = stack.step(torch.randn(2, 1536, device="cuda").bfloat16())
        assert stack.lengths.tolist() == [stack.held] * 2 and stack.held < 80
        if stack.held == 64 and step > 64:
            c = stack.layers[0].cache
            for b in range(2):
                at = c.position[stack.table[b].long()].transpose(0, 1).flatten(1)[:, :64]
                for h in range(2):
                    held = at[h].tolist()
                    assert len(set(held)) == 64 and max(held) == step
                    assert set(range(step - 23, step + 1)) <= set(held)
    assert torch.isfinite(out).all() and stack.seen.tolist() == [200, 200]


def test_tokens_command(bench):
    r = bench.tokens(layers=1, batch=2, budget=128, steps=70)
    assert r["finite"] and r["cache_bits_per_value"] == 4.25
