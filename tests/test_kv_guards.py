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
