"""What the page pool, the rotation and the choice of pages refuse, without a GPU:
arguments of the C ABI before any HIP call, and calls that something outside the
kernels watches."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EUNSUPPORTED, EWORKSPACE, EARG = -1, -3, -4
P = ctypes.c_void_p(0x10000)  # never dereferenced: every call below returns before launching


def at(address):
    return ctypes.c_void_p(address)


@pytest.fixture(scope="module")
def kv(rans):
    import kv_cache
    kv_cache.bind(rans._LIB)
    return kv_cache


@pytest.fixture(scope="module")
def kv_pages(rans):
    import kv_pages
    kv_pages.bind(rans._LIB)
    return kv_pages


@pytest.fixture(scope="module")
def rotary(rans):
    import rotary
    rotary.bind(rans._LIB)
    return rotary


HEADERS = {"vramc_pages.h": ("kv_pages", [("vramc_pages", "PagesDesc")]),
           "vramc_rotary.h": ("rotary", [("vramc_rotary", "RotaryDesc"), ("vramc_rotary_rows", "RowsDesc")])}


@pytest.mark.parametrize("header", list(HEADERS))
def test_headers(header, rans, lib, tmp_path):
    """What they declare is exported, they compile as C, and the mirrors have their
    structures' sizes."""
    import importlib
    module, structures = HEADERS[header]
    module = importlib.import_module(module)
    path = os.path.join(ROOT, "include", header)
    text = re.sub(r"/\*.*?\*/", "", open(path).read(), flags=re.S)
    names = re.findall(r"^(?:int|int64_t|void)\s+(\w+)\s*\(", text, flags=re.M)
    assert set(names) == set(module.EXPORTS) and len(names) == len(set(names))
    for name in names:
        assert hasattr(lib, name), name
    gcc = shutil.which("gcc")
    if gcc is None or not os.path.isdir("/opt/rocm/include"):
        pytest.skip("needs gcc and the ROCm headers")
    src = tmp_path / "use.c"
    src.write_text(f'#include "{header}"\n' + "".join(
        f"typedef char same{i}[sizeof({s}) == {ctypes.sizeof(getattr(module, m))} ? 1 : -1];\n"
        for i, (s, m) in enumerate(structures)) + f"int main(void) {{ return {names[0]} ? 0 : 1; }}\n")
    for std, lang in (("c99", "c"), ("c++17", "c++")):
        subprocess.check_call([gcc, f"-std={std}", "-x", lang, "-fsyntax-only", f"-I{os.path.dirname(path)}",
                               "-I/opt/rocm/include", "-D__HIP_PLATFORM_AMD__", str(src)])


# ------------------------------------------------------------------------ pool
def pool(kv_pages, **kw):
    base = dict(pages=64, page_size=16, free=0x100000, count=0x110000, ticket=0x120000)
    return ctypes.byref(kv_pages.PagesDesc(**{**base, **kw}))


# Three sequences: a table of rows 12 entries apart and 8 wide, 40 rows of tokens.
EXTEND = dict(table=0x200000, row=12, width=8, lengths=0x210000, fresh=0x220000, seen=0x230000, batch=3, tokens=40,
              slots=0x240000, positions=0x250000, filled=0x260000, starts=0x270000, grown=0x280000)


def extend(kv_pages, lib, pool_kw={}, **kw):
    a = {**EXTEND, **kw}
    pointer = {k: a[k] and at(a[k]) for k in a if k not in ("row", "width", "batch", "tokens")}
    return lib.vramc_pages_extend(pool(kv_pages, **pool_kw), pointer["table"], a["row"], a["width"], pointer["lengths"],
                                  pointer["fresh"], pointer["seen"], a["batch"], a["tokens"], pointer["slots"],
                                  pointer["positions"], pointer["filled"], pointer["starts"], pointer["grown"], None)


def test_extend_refuses(kv_pages, lib):
    for kw, code in ((dict(pages=0), EARG), (dict(pages=-5), EARG), (dict(page_size=48), EUNSUPPORTED),
                     (dict(free=None), EARG), (dict(count=None), EARG), (dict(ticket=None), EARG)):
        assert extend(kv_pages, lib, kw) == code
        assert lib.vramc_pages_release_workspace(pool(kv_pages, **kw), 8, 3) == code
        assert lib.vramc_pages_release(pool(kv_pages, **kw), P, 8, 8, P, 3, P, 1 << 20, None) == code
    for name in ("table", "lengths", "fresh", "slots", "positions", "filled", "starts", "grown"):
        assert extend(kv_pages, lib, **{name: None}) == EARG, name
    for kw in (dict(width=-1), dict(width=1 << 26, row=1 << 26), dict(batch=-1), dict(batch=4097), dict(row=7),
               dict(row=0), dict(row=-12), dict(tokens=-1), dict(tokens=2 ** 31 - 1)):
        assert extend(kv_pages, lib, **kw) == EARG, kw


@pytest.mark.parametrize("name,size", [("slots", 40 * 8), ("positions", 40 * 4), ("filled", 40 * 4), ("starts", 16),
                                       ("grown", 12)])
def test_extend_writes_nothing_that_it_reads(kv_pages, lib, name, size):
    """Some workgroups write while others read."""
    read = [(EXTEND["lengths"], 12), (EXTEND["fresh"], 12), (EXTEND["seen"], 12), (EXTEND["table"], 4 * (2 * 12 + 8)),
            (0x100000, 64 * 4), (0x110000, 4), (0x120000, 4)]
    for first, n in read:
        for address in (first, first + n - 4, first - size + 4):
            assert extend(kv_pages, lib, **{name: address}) == EARG, (hex(first), hex(address))


@pytest.mark.skipif(torch.cuda.is_available(), reason="a GPU is present, and the addresses are none of its own")
def test_extend_next_to_what_it_reads(kv_pages, lib):
    """Touching is not overlapping: these get as far as a HIP call."""
    for kw in (dict(grown=EXTEND["lengths"] + 12), dict(grown=EXTEND["lengths"] - 12), dict(starts=EXTEND["seen"] - 16),
               dict(slots=0x100000 + 64 * 4), dict(seen=None), dict(positions=EXTEND["table"] + 4 * (2 * 12 + 8))):
        assert extend(kv_pages, lib, **kw) > 0, kw


@pytest.mark.parametrize("name,size", [("lengths", 12), ("fresh", 12), ("seen", 12), ("free", 256), ("count", 4),
                                       ("ticket", 4)])
def test_extend_writes_no_table_that_it_reads_besides(kv_pages, lib, name, size):
    table, end = EXTEND["table"], EXTEND["table"] + 4 * (2 * 12 + 8)
    for address in (table, end - 4, table - size + 4):
        kw = {name: address}
        assert (extend(kv_pages, lib, **kw) if name in EXTEND else extend(kv_pages, lib, kw)) == EARG, hex(address)


def test_release_reads_no_lengths_where_it_writes(kv_pages, lib):
    for first, n in ((0x100000, 256), (0x110000, 4)):
        for address in (first, first + n - 4, first - 12 + 4):
            assert lib.vramc_pages_release(pool(kv_pages), P, 12, 8, at(address), 3, at(0x300000), 16, None) == EARG


def test_release_refuses(kv_pages, lib):
    p = pool(kv_pages)
    need = lib.vramc_pages_release_workspace(p, 8, 3)
    assert need == 16
    ok = [p, P, 12, 8, at(0x30000), 3, P, need, None]
    for i, value, code in ((0, None, EARG), (1, None, EARG), (2, 7, EARG), (3, -1, EARG), (3, 1 << 26, EARG),
                           (4, None, EARG), (5, -1, EARG), (5, 4097, EARG), (6, None, EWORKSPACE),
                           (6, at(0x10004), EARG), (7, need - 1, EWORKSPACE)):
        bad = list(ok)
        bad[i] = value
        assert lib.vramc_pages_release(*bad) == code, (i, value)
    table, size = 0x200000, 4 * (2 * 12 + 8)
    for name, first, n in (("lengths", None, 12), ("free", 0x100000, 256), ("count", 0x110000, 4)):
        for near in (0, n - 4, -size + 4):
            args = list(ok)
            args[1] = at((first or table) + near)
            if first is None:
                args[4] = at(table)
            assert lib.vramc_pages_release(*args) == EARG, name
    for i in (3, 5):  # nothing to give back
        none = list(ok)
        none[i] = 0
        assert lib.vramc_pages_release(*none) == 0
    for width, batch in ((-1, 3), (8, -1), (8, 4097), (1 << 26, 3)):
        assert lib.vramc_pages_release_workspace(p, width, batch) == EARG


# -------------------------------------------------------------------- rotation
def rotation(rotary, **kw):
    return ctypes.byref(rotary.RotaryDesc(**{**dict(head_dim=128, pairs=64, interleaved=0, amplitude=1.0, turns=0x10000), **kw}))


ROWS = dict(q=0x1000000, k=0x2000000, q_token=1536, q_head=128, k_token=256, k_head=128, q_heads=12, k_heads=2,
            q_weight=0x20000, k_weight=0x30000, dtype=1, weight_dtype=1, eps=1e-6, positions=0x40000, tokens=100)


def rows(rotary, **kw):
    return ctypes.byref(rotary.RowsDesc(**{**ROWS, **kw}))


def cache(kv, **kw):
    base = dict(pages=8, kv_heads=2, page_size=64, head_dim=128, dtype=1, mx=0, k=0x5000000, v=0x6000000)
    return ctypes.byref(kv.KvCacheDesc(**{**base, **kw}))


BAD_ROTATIONS = [(dict(head_dim=80), EUNSUPPORTED), (dict(head_dim=512), EUNSUPPORTED), (dict(pairs=0), EUNSUPPORTED),
                 (dict(pairs=12), EUNSUPPORTED), (dict(pairs=72), EUNSUPPORTED), (dict(pairs=-8), EUNSUPPORTED),
                 (dict(turns=None), EARG)]
BAD_ROWS = [(dict(dtype=3), EUNSUPPORTED), (dict(weight_dtype=2), EUNSUPPORTED), (dict(q_heads=-1), EARG),
            (dict(k_heads=-2), EARG), (dict(eps=-1.0), EARG), (dict(eps=float("nan")), EARG), (dict(tokens=-1), EARG),
            (dict(tokens=1 << 27), EARG), (dict(tokens=1 << 26), EARG), (dict(q_heads=1 << 17), EARG),
            (dict(q=None), EARG), (dict(k=None), EARG), (dict(positions=None), EARG), (dict(q_weight=0x20008), EARG),
            (dict(k_weight=0x20002), EARG), (dict(q_token=-1), EARG), (dict(k_head=-128), EARG)]


def test_rotation_refuses(kv, rotary, lib):
    r, x, c = rotation(rotary), rows(rotary), cache(kv)
    out = at(0x3000000), at(0x4000000)
    calls = lambda r, x: (lib.vramc_rotary_apply(r, x, *out, None),  # noqa: E731
                          lib.vramc_rotary_append(r, x, c, P, 256, 128, P, out[0], None))
    for kw, code in BAD_ROTATIONS:
        assert calls(rotation(rotary, **kw), x) == (code, code), kw
    for kw, code in BAD_ROWS:
        assert calls(r, rows(rotary, **kw)) == (code, code), kw
    assert calls(None, x) == calls(r, None) == (EARG, EARG)
    none = rows(rotary, tokens=0, q=None, k=None, positions=None)
    assert lib.vramc_rotary_apply(r, none, None, None, None) == 0
    assert lib.vramc_rotary_append(r, none, c, None, 0, 0, None, None, None) == 0
    for q_out, k_out in ((None, out[1]), (out[0], None), (at(0x3000008), out[1]), (out[0], at(0x4000004))):
        assert lib.vramc_rotary_apply(r, x, q_out, k_out, None) == EARG
    ok = [r, x, c, P, 256, 128, P, out[0], None]
    for i, value in ((2, None), (2, cache(kv, head_dim=64)), (2, cache(kv, dtype=2)), (2, cache(kv, kv_heads=4)),
                     (2, cache(kv, k=None)), (3, None), (4, -1), (5, -128), (6, None), (7, None), (7, at(0x3000008))):
        bad = list(ok)
        bad[i] = value
        assert lib.vramc_rotary_append(*bad) == EARG, i


def test_rotation_writes_nothing_that_it_reads(kv, rotary, lib):
    """A thread reads columns that another one's output would lie over."""
    r, x, c = rotation(rotary), rows(rotary), cache(kv)
    q, k, n = ROWS["q"], ROWS["k"], 100 * 1536 * 2
    far = at(0x7000000)
    for first, size in ((q, n), (k, 100 * 256 * 2)):
        for out in (first, first + size - 16, first - n + 16):
            assert lib.vramc_rotary_apply(r, x, at(out), far, None) == EARG
            assert lib.vramc_rotary_append(r, x, c, far, 256, 128, P, at(out), None) == EARG
        assert lib.vramc_rotary_apply(r, x, far, at(first), None) == EARG
    assert lib.vramc_rotary_apply(r, x, far, far, None) == EARG
    assert lib.vramc_rotary_apply(r, x, at(0x7000000 + 100 * 256 * 2 - 16), far, None) == EARG
    assert lib.vramc_rotary_append(r, x, c, far, 256, 128, P, far, None) == EARG


# ------------------------------------------------------------- choice of pages
def test_bound_and_select_refuse(kv, lib):
    c = cache(kv)
    for bad in ((None, P, 3, P), (c, None, 3, P), (c, P, -1, P), (c, P, 1 << 60, P), (c, P, 3, None),
                (c, P, 3, at(0x10008)), (cache(kv, page_size=8), P, 3, P)):
        assert lib.vramc_kv_bound(*bad, None) in (EARG, EUNSUPPORTED)
    assert lib.vramc_kv_bound(c, None, 0, None, None) == 0
    assert lib.vramc_kv_select_workspace(c, 4, 8, 3, 8) == 0  # all pages
    need = lib.vramc_kv_select_workspace(c, 4, 900, 3, 8)
    assert need == 3 * 2 * 900 * 8
    for heads, width, batch, count in ((4, -1, 3, 8), (4, 9, -1, 8), (4, 9, 3, 0), (4, 9, 3, -1), (4, 1 << 27, 3, 8),
                                       (4, 9, 1 << 24, 8), (4, 9, 3, 1 << 28), (3, 9, 3, 8), (0, 9, 3, 8), (-2, 9, 3, 8)):
        assert lib.vramc_kv_select_workspace(c, heads, width, batch, count) == EARG
    assert lib.vramc_kv_select_workspace(cache(kv, pages=1 << 30), 4, 9, 3, 8) == EARG  # page * heads beyond 32 bits
    ok = [c, P, P, 512, 128, 4, P, 900, 900, P, 3, 8, 1, 1, P, P, P, need, None]
    for i, value, code in ((1, None, EARG), (1, at(0x10008), EARG), (2, None, EARG), (5, 3, EARG), (5, 0, EARG),
                           (6, None, EARG), (9, None, EARG), (11, 1, EARG), (12, -1, EARG), (13, 0, EARG),
                           (12, 2 ** 31 - 1, EARG), (14, None, EARG), (15, None, EARG), (16, None, EWORKSPACE),
                           (16, at(0x10008), EARG), (17, need - 1, EWORKSPACE)):
        bad = list(ok)
        bad[i] = value
        assert lib.vramc_kv_select(*bad) == code, (i, value)
    ok[10] = 0  # no sequences
    assert lib.vramc_kv_select(*ok) == 0


def test_select_writes_nothing_that_it_reads(kv, lib):
    """Three sequences of two heads, 900 entries in rows 1000 apart, 8 pages each: some
    workgroups write while others read."""
    table, lengths, chosen, held, work = 0x100000, 0x200000, 0x300000, 0x400000, 0x500000
    c, need = cache(kv), 3 * 2 * 900 * 8

    def call(chosen=chosen, held=held):
        return lib.vramc_kv_select(c, P, P, 512, 128, 4, at(table), 1000, 900, at(lengths), 3, 8, 1, 1, at(chosen),
                                   at(held), at(work), need, None)
    for first, n in ((table, 4 * 2900), (lengths, 12)):
        for at_chosen in (first, first + n - 4, first - 6 * 8 * 4 + 4):
            assert call(chosen=at_chosen) == EARG
        for at_held in (first, first + n - 4, first - 6 * 4 + 4):
            assert call(held=at_held) == EARG
    assert call(held=chosen + 6 * 8 * 4 - 4) == EARG
    if not torch.cuda.is_available():  # touching is not overlapping
        assert call(chosen=lengths + 12) > 0 and call(held=table + 4 * 2900) > 0 and call(held=chosen + 6 * 8 * 4) > 0


def test_fails_loudly_without_gpu(kv_pages, rotary):
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    with pytest.raises(RuntimeError):
        kv_pages.PagePool(8)
    with pytest.raises(RuntimeError):
        rotary.Rotary(128)


# ------------------------------------------------- calls that something watches
class Counted:
    """Stands for the library: counts the calls that would launch."""
    _kv_bound = _pages_bound = _rotary_bound = True

    def __init__(self, answer=0):
        self.calls, self.answer = 0, answer

    def vramc_kv_attend_workspace(self, *args):
        return 64

    vramc_kv_select_workspace = vramc_kv_attend_workspace

    def launch(self, *args):
        self.calls += 1
        return self.answer

    vramc_kv_append = vramc_kv_attend = vramc_kv_bound = vramc_kv_select = launch
    vramc_pages_extend = vramc_pages_release = vramc_rotary_apply = vramc_rotary_append = launch


@pytest.fixture
def host(kv, kv_pages, rotary, rans, monkeypatch):
    """Everything on CPU tensors over a library that only counts, and each operation as
    a function of one tensor of its arguments."""
    monkeypatch.setattr(rans, "_device", lambda: -1)
    monkeypatch.setattr(rans, "_stream", lambda: 0)

    def make(answer=0):
        lib = Counted(answer)
        with monkeypatch.context() as m:
            m.setattr(torch.cuda, "is_available", lambda: True)
            m.setattr(torch.Tensor, "is_cuda", True)
            c = kv.PagedCache.allocate(8, 2, 64, 16, torch.float32, device="cpu", lib=lib, bounds=True)
            pool = kv_pages.PagePool(8, 16, device="cpu", lib=lib)
            turn = rotary.Rotary(64, device="cpu", lib=lib)
            c.heads
        table, n = torch.zeros(3, 2, dtype=torch.int32), torch.full((3,), 20, dtype=torch.int32)
        q, k, slots = torch.zeros(3, 4, 64), torch.zeros(3, 2, 64), torch.arange(3)
        chosen, held = torch.zeros(6, 2, dtype=torch.int32), torch.full((6,), 20, dtype=torch.int32)
        calls = {
            "extend": (lambda t: pool.extend(t, n, n, 7), table), "release": (lambda t: pool.release(t, n), table),
            "rotate q": (lambda x: turn.rotate(x, k, n), q), "rotate k": (lambda x: turn.rotate(q, x, n), k),
            "rotate weight": (lambda w: turn.rotate(q, k, n, w), torch.ones(64)),
            "append q": (lambda x: turn.append(c, x, k, k, slots, n), q),
            "append v": (lambda x: turn.append(c, q, k, x, slots, n), k.clone()),
            "bound": (lambda p: c.bound(p), n), "select": (lambda x: c.select(x, table, n, 2), q),
            "attend_selected": (lambda x: c.attend_selected(x, chosen, held), q),
        }
        return lib, c, calls
    return make


NAMES = ("extend", "release", "rotate q", "rotate k", "rotate weight", "append q", "append v", "bound", "select",
         "attend_selected")


@pytest.mark.parametrize("name", NAMES)
def test_watched_calls_are_refused(host, name):
    """Forward mode would drop the tangent; vmap, function and dispatch modes and tracers
    would not see the call.  The mode of a default device watches nothing."""
    from torch.autograd import forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.overrides import TorchFunctionMode
    from torch.utils._python_dispatch import TorchDispatchMode

    class Function(TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    class Dispatch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    lib, _, calls = host()
    call, x = calls[name]
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="watch"):
            call(forward_ad.make_dual(x, torch.ones_like(x)) if x.is_floating_point() else x)
    with pytest.raises(ValueError, match="watch"):
        torch.func.vmap(lambda t: (call(x), t)[1])(torch.zeros(2))
    for mode in (Function, Dispatch):
        with mode(), pytest.raises(ValueError, match="watch"):
            call(x)
    for trace in (lambda: torch.jit.trace(lambda t: (call(t), t + 1)[1], (x,), check_trace=False),
                  lambda: make_fx(lambda t: (call(t), t + 1)[1])(x)):
        with pytest.raises(ValueError, match="watch"):
            trace()
    assert lib.calls == 0
    with torch.device("cpu"), torch.no_grad():
        call(x)
    with torch.inference_mode():
        call(x)
    assert lib.calls == 2


@pytest.mark.parametrize("name", NAMES)
def test_under_the_compiler_calls_run_as_they_are(host, name):
    lib, _, calls = host()
    call, x = calls[name]
    run = torch.compile(lambda t: (call(t + 0), t + 1)[1], backend="eager")
    for i in range(1, 4):
        assert torch.equal(run(x), x + 1)
        assert lib.calls == i
    torch._dynamo.reset()


@pytest.mark.parametrize("name", ["rotate q", "rotate k", "rotate weight", "append q", "append v", "select",
                                  "attend_selected"])
def test_what_requires_a_gradient_is_refused(host, name):
    lib, _, calls = host()
    call, x = calls[name]
    x = x.clone().requires_grad_()
    with pytest.raises(ValueError, match="gradient"):
        call(x)
    assert lib.calls == 0
    with torch.no_grad():
        call(x)
    assert lib.calls == 1


@pytest.mark.parametrize("name", ["append q", "bound", "select", "attend_selected"])
def test_a_cache_that_requires_a_gradient_is_refused(host, name):
    lib, c, calls = host()
    call, x = calls[name]
    for t in (c.k, c.bounds):
        t.requires_grad_()
        with pytest.raises(ValueError, match="gradient"):
            call(x)
        t.requires_grad_(False)
    assert lib.calls == 0
    call(x)
    assert lib.calls == 1


@pytest.mark.parametrize("name", NAMES)
def test_what_the_library_answers_is_raised(host, name):
    call, x = host(answer=EARG)[2][name]
    with pytest.raises(ValueError, match=str(EARG)):
        call(x)
    call, x = host(answer=2)[2][name]
    with pytest.raises(RuntimeError, match="HIP error 2"):
        call(x)


def test_the_tensors_stay_their_own(host, kv_pages):
    _, c, _ = host()
    with pytest.raises(AttributeError):
        c.bounds = torch.zeros_like(c.bounds)
    for name in ("free", "count"):
        assert isinstance(getattr(kv_pages.PagePool, name), property) and getattr(kv_pages.PagePool, name).fset is None
