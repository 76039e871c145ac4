"""The key-value cache's operators: what a served model calls between its
projections, at the sizes where their speed counts.

- "attend": attention of one new token of each sequence over a paged cache,
  with the tokens' accumulated weight kept where the cache is tracked;
- "append": the keys and values of new tokens written into their pages, as
  they are or in microscaled 4-bit floating point, and read back from there;
- "evict": the tokens of the least accumulated weight dropped, in place or
  into other pages.

A cache is held in tensors: keys and values (pages, kv heads, page, dim), in
the model's type or ("mx") as 4-bit codes, two to a byte, with a scale byte
for every 32 of them; mass (f32) and position (int32), (pages, kv heads,
page), where it is tracked; table (int32, sequences x pages, -1 for none) and
lengths (int32).  Slot s of the cache is place s % page of page s // page.

A case is a dict: "op", "dtype", "mx", "track", "heads" (kv heads), "dim",
"page", "batch" (sequences), and
- attend: "group" (query heads of a kv head), "length" (of the longest
  sequence), "ragged" (a seed for the other lengths; 0: all alike), "capacity"
  (tokens that a row of the table has room for);
- append: "tokens" of each sequence, "fused" (q, k and v are columns of one
  projection's output), "group" (its query heads), "holes" (share of tokens
  that are padding, with slot -1);
- evict: "length", "ragged", "budget", "recent", "into" (other pages).
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # magnitudes of a 4-bit code
BLOCK = 32                                        # values to a scale
MAX_VALUES = 16 * 32768 * 8 * 128                 # keys of the largest cache


def _case(op, heads, dim, page, batch, dtype="bf16", mx=False, track=False, **more):
    return dict(op=op, heads=heads, dim=dim, page=page, batch=batch, dtype=dtype, mx=mx,
                track=track, **more)


def _attend(heads, group, dim, page, batch, length, ragged=0, capacity=0, **more):
    return _case("attend", heads, dim, page, batch, group=group, length=length, ragged=ragged,
                 capacity=max(capacity, length), **more)


def listed():
    named = [
        # the first tokens of a conversation with a 1.5B model (12 query heads
        # over 2): the shortest call of a token step, where latency counts; its
        # table has room for the conversation
        ("attend 5 tokens b1", _attend(2, 6, 128, 64, 1, 5, capacity=4096)),
        # one long document before the same model: the length has to be split
        # to fill the card
        ("attend 32768 tokens b1", _attend(2, 6, 128, 64, 1, 32768)),
        # sixteen conversations of a model 5120 wide, of different lengths: the
        # largest cache here, bound by reading it
        ("attend 32768 tokens b16", _attend(8, 5, 128, 64, 16, 32768, ragged=1)),
        # the same conversations in a cache of 4-bit values
        ("attend 32768 tokens b16 mx", _attend(8, 5, 128, 64, 16, 32768, ragged=1, mx=True)),
        # a decode step under eviction: many sequences held near a budget of
        # 2048 tokens, the weights accumulated
        ("attend 2049 tokens b64 tracked", _attend(2, 6, 128, 64, 64, 2049, ragged=2, track=True)),
        # a small f16 model with 7 query heads to a kv head: small pages, 4-bit
        # values, odd lengths, an empty sequence among them
        ("attend 2999 tokens b7 f16 mx", _attend(2, 7, 64, 16, 7, 2999, ragged=3, dtype="f16",
                                                 mx=True, track=True)),
        # a head of its own for every query head, unusual width, in f32
        ("attend 1777 tokens b3 f32", _attend(8, 1, 96, 32, 3, 1777, ragged=4, dtype="f32")),
        # a decode step's new tokens of sixteen sequences into 4-bit pages
        ("append 1 token b16 mx", _case("append", 2, 128, 64, 16, mx=True, track=True, tokens=1,
                                        group=6, fused=True, holes=0.0)),
        # a prompt's keys and values into 4-bit pages, straight from the fused
        # projection's output
        ("append 32768 tokens mx", _case("append", 8, 128, 64, 1, mx=True, track=True,
                                         tokens=32768, group=5, fused=True, holes=0.0)),
        # a decode step of 64 sequences at their budget: one token each goes
        ("evict 2049 to 2048 b64", _case("evict", 2, 128, 64, 64, track=True, length=2049,
                                         ragged=0, budget=2048, recent=256, into=False)),
        # long prompts cut to an eighth into pages of their own, so that pages
        # shared with other sequences stay as they are
        ("evict 32768 to 4096 b4", _case("evict", 8, 128, 64, 4, track=True, length=32768,
                                         ragged=0, budget=4096, recent=512, into=True)),
        # a few odd sequences of an f16 model, some of them under the budget
        ("evict 1999 to 500 b5 f16", _case("evict", 3, 64, 16, 5, dtype="f16", track=True,
                                           length=1999, ragged=5, budget=500, recent=33,
                                           into=True)),
    ]
    return [dict(c, name=n) for n, c in named]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "append", "evict"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    mx = dtype != "f32" and rng.random() < 0.5
    heads, dim = rng.choice([1, 2, 3, 4, 8, 16]), rng.choice([64, 96, 128, 128, 192, 256])
    page, batch = rng.choice([16, 32, 64, 128]), _log_uniform(rng, 1, 64)
    most = MAX_VALUES // (heads * dim * batch)  # tokens of a sequence
    if dtype == "f32":
        most //= 2
    ragged = rng.choice([0, rng.randrange(1, 1000)])
    if op == "attend":
        length = _log_uniform(rng, 1, min(most, 40000))
        capacity = min(most, length * rng.choice([1, 1, 2, 8]))
        return _attend(heads, rng.choice([1, 2, 4, 5, 7, 8, 12, 16, 24]), dim, page, batch, length,
                       ragged, capacity, dtype=dtype, mx=mx, track=rng.random() < 0.4)
    if op == "append":
        tokens = _log_uniform(rng, 1, max(1, min(most // 16, 40000)))
        return _case(op, heads, dim, page, batch, dtype, mx, rng.random() < 0.5, tokens=tokens,
                     group=rng.choice([1, 4, 6]), fused=rng.random() < 0.5,
                     holes=rng.choice([0.0, 0.0, 0.2]))
    length = _log_uniform(rng, 2, max(2, min(most // 4, 40000)))
    budget = max(1, rng.choice([length - 1, length - page, length // 2, length // 5]))
    return _case(op, heads, dim, page, batch, dtype, mx, True, length=length, ragged=ragged,
                 budget=budget, recent=rng.randrange(0, budget + 1), into=rng.random() < 0.5)


# --------------------------------------------------------------------- inputs
def _lengths(case):
    """Tokens of every sequence, by the case alone: the first is the longest,
    others are anything down to none."""
    n, rng = case["length"], random.Random(case["ragged"])
    if not case["ragged"]:
        return [n] * case["batch"]
    rest = [rng.choice([rng.randint(0, n), rng.randint(n // 2, n), n - rng.randint(0, n // 16)])
            for _ in range(case["batch"] - 1)]
    if len(rest) > 4:
        rest[2] = 0
    return [n] + rest


def _values(shape, dtype, gen, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=gen) * scale).to(dtype)


def _stored(case, pages, gen):
    """Keys or values of a whole cache, as the case stores them: values or
    codes (and scales) of some distribution of magnitudes."""
    shape = (pages, case["heads"], case["page"], case["dim"])
    if not case["mx"]:
        return _values(shape, DTYPES[case["dtype"]], gen), None
    codes = torch.randint(0, 256, shape[:3] + (shape[3] // 2,), dtype=torch.uint8, device="cuda",
                          generator=gen)
    scales = torch.randint(124, 128, shape[:3] + (shape[3] // BLOCK,), dtype=torch.uint8,
                           device="cuda", generator=gen)
    return codes, scales


def _table(counts, width, first, gen, pages):
    """Each sequence's pages, in no order, -1 behind them."""
    order = torch.randperm(pages, device="cuda", generator=gen).int()
    table = torch.full((len(counts), width), -1, dtype=torch.int32, device="cuda")
    at = first
    for row, n in zip(table, counts):
        row[:n] = order[at:at + n]
        at += n
    return table, order[at:]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(1000003 * seed + 29)
    dtype, heads, dim, page = DTYPES[case["dtype"]], case["heads"], case["dim"], case["page"]
    batch, op = case["batch"], case["op"]
    lengths = _lengths(case) if op != "append" else [case["tokens"]] * batch
    counts = [-(-n // page) for n in lengths]
    budget = case.get("budget", 0)
    wide = -(-budget // page) if case.get("into") else 0
    pages = sum(counts) + batch * wide + 3
    state = dict(op=op, dtype=dtype, mx=case["mx"], page=page)
    state["k"], state["k_scale"] = _stored(case, pages, gen)
    state["v"], state["v_scale"] = _stored(case, pages, gen)
    capacity = -(-case.get("capacity", max(lengths)) // page)
    state["table"], spare = _table(counts, capacity, 0, gen, pages)
    state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    state["mass"] = state["position"] = None
    if case["track"]:
        # weights as attention leaves them: most tokens hold little, some
        # nothing at all, a few a lot
        shape = (pages, heads, page)
        mass = torch.randn(shape, device="cuda", generator=gen).mul_(2).exp_()
        mass[torch.rand(shape, device="cuda", generator=gen) < 0.1] = 0.0
        state["mass"] = mass
        state["position"] = torch.zeros(shape, dtype=torch.int32, device="cuda")
    # each place of a sequence's pages: its slot, and whether a token is there
    place = torch.arange(capacity * page, device="cuda")
    slot = state["table"].long().repeat_interleave(page, 1) * page + place % page
    there = place < state["lengths"][:, None]
    if op == "attend":
        # what lies behind a sequence's last token is anything
        behind = slot[~there & (slot >= 0)]
        at = behind // page, slice(None), behind % page
        (state["k_scale"] if case["mx"] else state["k"])[at] = 255 if case["mx"] else math.nan
        (state["v_scale"] if case["mx"] else state["v"])[at] = 255 if case["mx"] else math.nan
        state["q"] = _values((batch, heads * case["group"], dim), dtype, gen, 2.0)
        state["scale"] = dim ** -0.5
    elif op == "append":
        rows = batch * case["tokens"]
        if case["fused"]:
            qkv = _values((rows, (case["group"] + 2) * heads, dim), dtype, gen)
            k, v = qkv[:, -2 * heads:-heads], qkv[:, -heads:]
        else:
            k, v = (_values((rows, heads, dim), dtype, gen) for _ in range(2))
        # outlier channels, as keys have them, and tokens that are nearly zero
        k *= torch.where(torch.rand(dim, device="cuda", generator=gen) < 0.03, 8.0, 1.0).to(dtype)
        v *= torch.where(torch.rand(rows, 1, 1, device="cuda", generator=gen) < 0.01, 2.0 ** -12,
                         1.0).to(dtype)
        slots = slot[:, :case["tokens"]].reshape(-1)
        if case["holes"]:
            slots = torch.where(torch.rand(rows, device="cuda", generator=gen) < case["holes"], -1,
                                slots)
        state.update(k_new=k, v_new=v, slots=slots.contiguous(),
                     positions=torch.arange(case["tokens"], dtype=torch.int32,
                                            device="cuda").repeat(batch))
    else:
        # tokens lie in no order after earlier evictions; each has seen twice
        # as many as it holds
        state["seen"] = 2 * state["lengths"]
        order = torch.argsort(torch.rand(batch, heads, capacity * page, device="cuda",
                                         generator=gen).masked_fill_(~there[:, None], 2.0), -1)
        back = torch.argsort(order, -1)
        where = torch.where(there[:, None], 2 * back + 1, 0).int()
        b, j = torch.nonzero(there, as_tuple=True)
        state["position"][slot[b, j] // page, :, slot[b, j] % page] = where[b, :, j]
        state.update(budget=budget, recent=case["recent"], into=None)
        if case["into"]:
            state["into"] = spare[:batch * wide].reshape(batch, wide).contiguous()
            base = state["into"].long()[:, :, None] * page + torch.arange(page, device="cuda")
            state["slots"] = base.reshape(batch, -1)[:, :budget].reshape(-1).contiguous()
        else:
            state["slots"] = torch.where(there, slot, -1)[:, :budget].reshape(-1).contiguous()
    if own:
        package = os.path.join(ROOT, "vram-compression_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
        import kv_cache
        state["cache"] = kv_cache.PagedCache(state["k"], state["v"], dtype, state["k_scale"],
                                             state["v_scale"], state["mass"], state["position"])
    return state


# ---------------------------------------------------------------- plain forms
def _power(scales):
    """2^(byte - 127) of scale bytes, NaN for 255."""
    bits = scales.to(torch.int32) << 23
    power = torch.where(scales == 0, 0x400000, bits).view(torch.float32)
    return torch.where(scales == 255, math.nan, power)


def _opened(stored, scales):
    """Cache rows as f32 values."""
    if scales is None:
        return stored.float()
    grid = torch.tensor(GRID + tuple(-g for g in GRID), device=stored.device)
    pair = torch.stack((stored & 15, stored >> 4), -1).flatten(-2).long()
    return (grid[pair].unflatten(-1, (-1, BLOCK)) * _power(scales)[..., None]).flatten(-2)


def _closed(x):
    """f32 values as 4-bit codes and scale bytes."""
    x = x.unflatten(-1, (-1, BLOCK))
    most = x.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    exponent = torch.frexp(torch.where(bad, 1.0, most))[1] - 3  # floor(log2) - 2
    byte = torch.where(most == 0, 0, (exponent + 127).clamp(0, 252))
    y = x * _power((254 - byte).to(torch.uint8))
    a = y.abs()
    code = ((a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5)
            + (a > 5))
    code = torch.where(bad, 0, code + 8 * torch.signbit(x)).flatten(-2)
    return ((code[..., 0::2] | code[..., 1::2] << 4).to(torch.uint8),
            torch.where(bad, 255, byte).squeeze(-1).to(torch.uint8))


def _plain_attend(s):
    table, page, q = s["table"], s["page"], s["q"].float()
    rows = table.long().clamp(min=0)
    batch, heads = table.shape[0], s["k"].shape[1]

    def laid(stored, scales):  # (batch, heads, tokens, dim) in f32
        x = _opened(stored[rows], None if scales is None else scales[rows])
        return x.transpose(1, 2).flatten(2, 3)

    there = torch.arange(table.shape[1] * page, device=q.device) < s["lengths"][:, None]
    there = (there & (table >= 0).repeat_interleave(page, 1))[:, None, None]
    q = q.unflatten(1, (heads, -1))
    scores = torch.matmul(q, laid(s["k"], s["k_scale"]).transpose(-1, -2)) * s["scale"]
    scores = scores.masked_fill_(~there, -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(torch.isinf(top) & (top < 0), 0.0, top))
    del scores
    total = weights.sum(-1, keepdim=True)
    weights = torch.where(total == 0, 0.0, weights / total)
    values = laid(s["v"], s["v_scale"])
    out = torch.matmul(weights, torch.where(there[:, 0, 0, :, None][:, None], values, 0.0))
    out = out.flatten(1, 2).to(s["dtype"])
    if s["mass"] is None:
        return [out]
    share = weights.sum(2).unflatten(-1, (-1, page)).transpose(1, 2).flatten(0, 1)
    s["mass"].index_add_(0, rows.flatten(), share)
    return [out, s["mass"]]


def _plain_read(s, slots):
    at = slots.clamp(min=0) // s["page"], slice(None), slots.clamp(min=0) % s["page"]
    outs = []
    for stored, scales in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])):
        x = _opened(stored[at], None if scales is None else scales[at])
        outs.append(torch.where((slots >= 0)[:, None, None], x, 0.0).to(s["dtype"]))
    return outs


def _plain_append(s):
    written = s["slots"] >= 0
    slots = s["slots"][written]
    at = slots // s["page"], slice(None), slots % s["page"]
    for new, stored, scales in ((s["k_new"], s["k"], s["k_scale"]),
                                (s["v_new"], s["v"], s["v_scale"])):
        if scales is None:
            stored[at] = new[written]
        else:
            stored[at], scales[at] = _closed(new[written].float())
    if s["mass"] is not None:
        s["mass"][at] = 0.0
        s["position"][at] = s["positions"][written][:, None]
    return _held(s)


def _plain_evict(s):
    table, page, budget, into = s["table"], s["page"], s["budget"], s["into"]
    rows = table.long().clamp(min=0)
    length = s["lengths"][:, None, None]
    slot = (rows[:, :, None] * page + torch.arange(page, device=rows.device)).flatten(1)[:, None]
    index = torch.arange(slot.shape[-1], device=rows.device)
    mass, position = (x[rows].transpose(1, 2).flatten(2) for x in (s["mass"], s["position"]))
    bits = torch.where(torch.isnan(mass), -math.inf, mass + 0.0).view(torch.int32)
    rank = torch.where(bits < 0, -(bits & 0x7fffffff), bits).long()
    rank = torch.where(position >= s["seen"][:, None, None] - s["recent"], 1 << 33, rank)
    rank = torch.where(index < length, rank, -(1 << 40))
    best = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :budget]
    kept = torch.zeros_like(rank, dtype=torch.bool).scatter_(-1, best, True) & (index < length)
    end = slot.shape[-1]

    def ordered(chosen, most):  # the first `most` chosen indices, `end` behind them
        return torch.where(chosen, index, end).sort(-1).values[..., :most]

    if into is None:
        most = max(0, min(budget, end - budget))
        to = ordered(~kept & (index < torch.clamp(length, max=budget)), most)
        source = ordered(kept & (index >= budget), most)
        to_slot = slot.expand_as(rank).gather(-1, to.clamp(max=end - 1))
    else:
        source = ordered(kept, budget)
        most = source.shape[-1]
        to_slot = into.long()[:, :, None] * page + torch.arange(page, device=rows.device)
        to_slot = to_slot.flatten(1)[:, None, :most].expand_as(source)
    moved = source < end
    head = torch.arange(rank.shape[1], device=rows.device)[:, None].expand_as(moved)[moved]
    to_slot = to_slot[moved]
    source = slot.expand_as(rank).gather(-1, source.clamp(max=end - 1))[moved]
    for x in (s["k"], s["v"], s["k_scale"], s["v_scale"], s["mass"], s["position"]):
        if x is not None:
            x[to_slot // page, head, to_slot % page] = x[source // page, head, source % page]
    return _held(s) + [s["lengths"].clamp(max=budget)]


def _held(s):
    """What the cache holds after a call: its buffers, or the values that 4-bit
    codes stand for."""
    if s["mx"]:
        out = s["cache"].read(s["slots"]) if own else _plain_read(s, s["slots"])
    else:
        out = s["k"], s["v"]
    return [*out] + ([] if s["mass"] is None else [s["mass"], s["position"]])


def run(state):
    s, op = state, state["op"]
    if not own:
        return {"attend": _plain_attend, "append": _plain_append, "evict": _plain_evict}[op](s)
    cache = s["cache"]
    if op == "attend":
        out = cache.attend(s["q"], s["table"], s["lengths"], s["scale"])
        return [out] if s["mass"] is None else [out, s["mass"]]
    if op == "append":
        cache.append(s["k_new"], s["v_new"], s["slots"],
                     None if s["mass"] is None else s["positions"])
        return _held(s)
    lengths = cache.evict(s["table"], s["lengths"], s["seen"], s["budget"], s["recent"], s["into"])
    return _held(s) + [lengths]


# -------------------------------------------------- the definitions in 64 bits
def _power64(exponent):
    """2^exponent from its bits (pow is off by a bit for some)."""
    return (exponent.long() + 1023 << 52).view(torch.float64)


def _value64(stored, scales):
    """Cache rows as f64 values."""
    if scales is None:
        return stored.double()
    low, high = stored % 16, stored // 16
    code = torch.stack((low, high), -1).reshape(*stored.shape[:-1], -1).double()
    sign = torch.where(code >= 8, -1.0, 1.0)
    code = code % 8
    octave = torch.clamp(torch.floor(code / 2) - 1, min=0)
    size = torch.where(code < 2, code / 2, (1 + code % 2 / 2) * _power64(octave))
    power = _power64(scales.long() - 127)
    power[scales == 255] = math.nan
    return sign * size * power.repeat_interleave(BLOCK, -1)


def _rounded64(x):
    """What 4-bit storage makes of f64 values."""
    y = x.reshape(-1, BLOCK)
    most = y.abs().amax(1, keepdim=True)
    whole = torch.floor(torch.log2(most.clamp(min=2.0 ** -140)))
    whole += (_power64(whole + 1) <= most).double() - (_power64(whole) > most).double()
    unit = _power64((whole - 2).clamp(-127, 125))
    a = (y / unit).abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = torch.clamp(torch.round(a / step) * step, max=6.0)
    return (torch.sign(y) * a * unit).reshape(x.shape)


def _exact_attend(case, s):
    page, heads, group = case["page"], case["heads"], case["group"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    mass = None if s["mass"] is None else s["mass"].double()
    for b, n in enumerate(_lengths(case)):
        if not n:
            continue
        rows = s["table"][b, :-(-n // page)].long()
        for h in range(heads):
            k, v = (_value64(s[x][rows, h], None if s[x + "_scale"] is None else
                             s[x + "_scale"][rows, h]).reshape(-1, case["dim"])[:n]
                    for x in ("k", "v"))
            mine = slice(h * group, (h + 1) * group)
            w = torch.softmax(s["q"][b, mine].double() @ k.t().contiguous() * s["scale"], -1)
            out[b, mine] = w @ v
            if mass is not None:
                add = torch.zeros(len(rows) * page, dtype=torch.float64, device="cuda")
                add[:n] = w.sum(0)
                mass[rows, h] += add.reshape(-1, page)
    return [out] if mass is None else [out, mass]


def _exact_append(case, s):
    page, keep = case["page"], s["slots"] >= 0
    slots = s["slots"][keep]
    outs = []
    for new, stored in ((s["k_new"], s["k"]), (s["v_new"], s["v"])):
        if case["mx"]:
            x = _rounded64(new.double())
            outs.append(x * keep[:, None, None])
        else:
            x = stored.double()
            x[slots // page, :, slots % page] = new[keep].double()
            outs.append(x)
    if s["mass"] is None:
        return outs
    mass = s["mass"].double()
    mass[slots // page, :, slots % page] = 0
    return outs + [mass, None]


def _exact_evict(case, s):
    page, budget = case["page"], case["budget"]
    names = ("k", "v", "mass") if not case["mx"] else ("mass",)
    held = {x: s[x].double() for x in names}
    if case["mx"]:
        held["k"], held["v"] = (_value64(s[x], s[x + "_scale"]) for x in ("k", "v"))
    mass, position = s["mass"].cpu().numpy(), s["position"].cpu().numpy()
    table = s["table"].cpu().numpy().astype(np.int64)
    into = None if s["into"] is None else s["into"].cpu().numpy().astype(np.int64)
    seen = s["seen"].tolist()
    for b, n in enumerate(_lengths(case)):
        index = np.arange(n)
        pages, places = table[b, index // page], index % page
        for h in range(case["heads"]):
            shielded = position[pages, h, places] >= seen[b] - case["recent"]
            order = np.lexsort((index, -mass[pages, h, places].astype(np.float64), ~shielded))
            kept = np.sort(order[:budget])
            if into is not None:
                source, to = kept, np.arange(len(kept))
                to_page = into[b, to // page]
            else:
                source = kept[kept >= budget]
                to = np.setdiff1d(np.arange(min(n, budget)), kept)
                to_page = table[b, to // page]
            at = tuple(torch.from_numpy(x).cuda() for x in (pages[source], places[source],
                                                            to_page, to % page))
            for x in held.values():
                x[at[2], h, at[3]] = x[at[0], h, at[1]]
    k, v = held["k"], held["v"]
    if case["mx"]:
        slots = s["slots"].clamp(min=0)
        there = (s["slots"] >= 0)[:, None, None]
        k, v = (torch.where(there, x[slots // page, :, slots % page], 0.0) for x in (k, v))
    return [k, v, held["mass"], None, None]


def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "append": _exact_append,
            "evict": _exact_evict}[case["op"]](case, s)


def work(case):
    """Every stored byte of the tokens that a pass is about, read or written
    once, its other inputs and outputs once."""
    op, heads, dim, batch = case["op"], case["heads"], case["dim"], case["batch"]
    size = 4 if case["dtype"] == "f32" else 2
    stored = 2 * (dim // 2 + dim // BLOCK if case["mx"] else dim * size)  # K and V of a token
    if op == "append":
        tokens = batch * case["tokens"] * heads
        values = 2 * dim * size
        moved = tokens * (values + stored + 8 * case["track"])
        return {"bytes": moved + (tokens * (stored + values) if case["mx"] else 0),
                "flops": 2 * dim * tokens}
    lengths = _lengths(case)
    tokens = sum(lengths) * heads
    if op == "attend":
        queries = batch * heads * case["group"]
        return {"bytes": tokens * (stored + 8 * case["track"]) + 2 * queries * dim * size
                + 4 * (tokens // heads // case["page"] + batch),
                "flops": 4 * dim * tokens * case["group"]}
    moved = heads * sum(min(n, case["budget"]) if case["into"] else
                        min(case["budget"], max(0, n - case["budget"])) for n in lengths)
    read = heads * sum(min(n, case["budget"]) for n in lengths) if case["mx"] else 0
    return {"bytes": 8 * tokens + moved * 2 * (stored + 8) + read * (stored + 2 * dim * size),
            "flops": 8 * tokens}
