"""What the key-value cache refuses, without a GPU: arguments of the C ABI that
would be read while they are written, and calls that something outside the
kernels watches."""
import ctypes

import pytest
import torch

EARG = -4


def at(address):
    return ctypes.c_void_p(address)


@pytest.fixture(scope="module")
def kv(rans):
    import kv_cache
    kv_cache.bind(rans._LIB)
    return kv_cache


def desc(kv):
    return ctypes.byref(kv.KvCacheDesc(pages=8, kv_heads=2, page_size=64, head_dim=128, dtype=1, mx=0, k=0x10000,
                                       v=0x20000, mass=0x30000, position=0x40000))


# Three sequences: lengths and seen of 12 bytes, a table of rows 12 entries apart
# and 8 wide, other pages of rows 4 apart and 2 wide.
EVICT = dict(table=0x100000, lengths=0x110000, seen=0x120000, into=0x130000, new=0x140000, work=0x150000)


def evict(kv, lib, **kw):
    a = {**EVICT, **kw}
    c = desc(kv)
    need = lib.vramc_kv_evict_workspace(c, 8, 3, 100, a["into"] is not None)
    return lib.vramc_kv_evict(c, at(a["table"]), 12, 8, at(a["lengths"]), at(a["seen"]), 3, 100, 5,
                              a["into"] and at(a["into"]), 4 if a["into"] else 0, 2 if a["into"] else 0,
                              at(a["new"]), at(a["work"]), need, None)


@pytest.mark.parametrize("new", [
    EVICT["lengths"], EVICT["lengths"] - 8, EVICT["lengths"] + 8, EVICT["seen"], EVICT["seen"] + 8,
    EVICT["table"], EVICT["table"] - 8, EVICT["table"] + 4 * 10, EVICT["table"] + 4 * (2 * 12 + 8) - 4,
    EVICT["into"], EVICT["into"] + 4 * (2 * 4 + 2) - 4])
def test_new_lengths_apart_from_what_is_read(kv, lib, new):
    """Workgroups of a sequence's other kv heads may read its length, what it has
    seen and its rows after the first has written the new length."""
    assert evict(kv, lib, new=new) == EARG
    if new < EVICT["into"] - 12:
        assert evict(kv, lib, new=new, into=None) == EARG


@pytest.mark.skipif(torch.cuda.is_available(), reason="a GPU is present, and the addresses are none of its own")
def test_new_lengths_next_to_what_is_read(kv, lib):
    """Touching is not overlapping: these get as far as a HIP call."""
    for new in (EVICT["lengths"] - 12, EVICT["lengths"] + 12, EVICT["table"] + 4 * (2 * 12 + 8),
                EVICT["table"] + 4 * 8, EVICT["table"] + 4 * (12 + 9), EVICT["into"] + 4 * (2 * 4 + 2)):
        assert evict(kv, lib, new=new) > 0


def test_evict_workspace_is_aligned(kv, lib):
    assert evict(kv, lib, work=0x150004) == EARG
    assert evict(kv, lib, work=0x150008) == EARG


# ------------------------------------------------- calls that something watches
class Counted:
    """Stands for the library: counts the calls that would launch."""
    _kv_bound = True

    def __init__(self, answer=0):
        self.calls, self.answer = 0, answer

    def vramc_kv_attend_workspace(self, *args):
        return 64

    vramc_kv_evict_workspace = vramc_kv_attend_workspace

    def launch(self, *args):
        self.calls += 1
        return self.answer

    vramc_kv_append = vramc_kv_read = vramc_kv_attend = vramc_kv_evict = launch


@pytest.fixture
def host(kv, rans, monkeypatch):
    """Caches of CPU tensors over a library that only counts."""
    monkeypatch.setattr(rans, "_device", lambda: -1)
    monkeypatch.setattr(rans, "_stream", lambda: 0)

    def make(dtype=torch.float32, answer=0):
        with monkeypatch.context() as m:
            m.setattr(torch.cuda, "is_available", lambda: True)
            m.setattr(torch.Tensor, "is_cuda", True)
            return kv.PagedCache.allocate(8, 2, 64, 16, dtype, track=True, device="cpu", lib=Counted(answer))
    return make


def operations(c):
    """Every operation as a function of one tensor of its arguments."""
    table = torch.zeros(3, 2, dtype=torch.int32)
    n = torch.full((3,), 20, dtype=torch.int32)
    slots = torch.arange(3)
    k = torch.zeros(3, 2, 64, dtype=c.dtype)
    return {
        "attend": (lambda q: c.attend(q, table, n), torch.zeros(3, 4, 64, dtype=c.dtype)),
        "append k": (lambda x: c.append(x, k, slots, n), k),
        "append v": (lambda x: c.append(k, x, slots, n), k.clone()),
        "read": (lambda s: c.read(s), slots),
        "evict": (lambda t: c.evict(t, n, n, 7), table),
    }


NAMES = ("attend", "append k", "append v", "read", "evict")


@pytest.mark.parametrize("name", NAMES)
def test_tracers_are_refused(host, name):
    """A traced call would leave a program without the kernel: uninitialised
    memory in place of its output."""
    from torch.fx.experimental.proxy_tensor import make_fx
    c = host()
    call, x = operations(c)[name]
    call(x)
    assert c.lib.calls == 1
    for trace in (lambda: torch.jit.trace(lambda t: (call(t), t + 1)[1], (x,), check_trace=False),
                  lambda: make_fx(lambda t: (call(t), t + 1)[1])(x)):
        with pytest.raises(ValueError, match="watch"):
            trace()
    assert c.lib.calls == 1


@pytest.mark.parametrize("name", NAMES)
def test_modes_and_levels_are_refused(host, name):
    """Forward mode would drop the tangent, vmap and function and dispatch modes
    would not see the call; the mode of a default device watches nothing."""
    from torch.autograd import forward_ad
    from torch.overrides import TorchFunctionMode
    from torch.utils._python_dispatch import TorchDispatchMode

    class Function(TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    class Dispatch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    c = host()
    call, x = operations(c)[name]
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="watch"):
            call(forward_ad.make_dual(x, torch.ones_like(x)) if x.is_floating_point() else x)
    with pytest.raises(ValueError, match="watch"):
        torch.func.vmap(lambda t: (call(x), t)[1])(torch.zeros(2))
    for mode in (Function, Dispatch):
        with mode(), pytest.raises(ValueError, match="watch"):
            call(x)
    assert c.lib.calls == 0
    with torch.device("cpu"), torch.no_grad():
        call(x)
    with torch.inference_mode():
        call(x)
    assert c.lib.calls == 2


@pytest.mark.parametrize("name", NAMES)
def test_under_the_compiler_calls_run_as_they_are(host, name):
    """A compiled program breaks at a call and makes it."""
    c = host()
    call, x = operations(c)[name]
    run = torch.compile(lambda t: (call(t + 0), t + 1)[1], backend="eager")
    for i in range(1, 4):
        assert torch.equal(run(x), x + 1)
        assert c.lib.calls == i
    torch._dynamo.reset()


@pytest.mark.parametrize("which", ["k", "v", "mass"])
@pytest.mark.parametrize("name", NAMES)
def test_a_cache_that_requires_a_gradient_is_refused(host, name, which):
    """Its output would have no gradient for what it was computed from, and its
    writes pass autograd by; without gradients it is a cache like any other."""
    c = host()
    call, x = operations(c)[name]
    getattr(c, which).requires_grad_()
    with pytest.raises(ValueError, match="gradient"):
        call(x)
    assert c.lib.calls == 0
    with torch.no_grad():
        call(x)
    getattr(c, which).requires_grad_(False)
    call(x)
    assert c.lib.calls == 2


@pytest.mark.parametrize("name", NAMES)
def test_what_the_library_answers_is_raised(host, name):
    """A refusal of the library is a ValueError, an error of HIP a RuntimeError,
    neither an assertion that optimised Python leaves out."""
    call, x = operations(host(answer=EARG))[name]
    with pytest.raises(ValueError, match=str(EARG)):
        call(x)
    call, x = operations(host(answer=2))[name]
    with pytest.raises(RuntimeError, match="HIP error 2"):
        call(x)


@pytest.mark.parametrize("which", ["k", "v", "k_scale", "v_scale", "mass", "position"])
def test_the_tensors_of_a_cache_stay_its_own(host, which):
    """The kernels write where the tensors lay when the cache was made: another
    tensor in the place of one would leave them writing to freed memory."""
    c = host()
    held = getattr(c, which)
    with pytest.raises(AttributeError):
        setattr(c, which, torch.zeros(1) if held is None else torch.zeros_like(held))
    assert getattr(c, which) is held
