"""The key-value cache's C ABI without a GPU: the library exports what
include/vramc_kv.h declares and refuses bad arguments before any HIP call."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "vramc_kv.h")
EUNSUPPORTED, EWORKSPACE, EARG = -1, -3, -4
P = ctypes.c_void_p(0x10000)  # never dereferenced: every call below returns before launching


@pytest.fixture(scope="module")
def kv(rans):
    import kv_cache
    kv_cache.bind(rans._LIB)
    return kv_cache


def desc(kv, **kw):
    base = dict(pages=8, kv_heads=2, page_size=64, head_dim=128, dtype=1, mx=0, k=0x10000,
                v=0x20000, k_scale=None, v_scale=None, mass=0x30000, position=0x40000)
    return kv.KvCacheDesc(**{**base, **kw})


def test_every_declared_symbol_is_exported(kv, lib):
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = re.findall(r"^(?:int|int64_t|void)\s+(\w+)\s*\(", text, flags=re.M)
    assert set(names) == set(kv.EXPORTS) and len(names) == len(set(names))
    for name in names:
        assert hasattr(lib, name), name


def test_header_compiles_as_c_and_matches_the_mirror(kv, tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None or not os.path.isdir("/opt/rocm/include"):
        pytest.skip("needs gcc and the ROCm headers")
    src = tmp_path / "use.c"
    src.write_text('#include "vramc_kv.h"\n'
                   f"typedef char same[sizeof(vramc_kv_cache) == {ctypes.sizeof(kv.KvCacheDesc)} ? 1 : -1];\n"
                   "int main(void) { return vramc_kv_attend ? 0 : 1; }\n")
    for std, lang in (("c99", "c"), ("c++17", "c++")):
        subprocess.check_call([gcc, f"-std={std}", "-x", lang, "-fsyntax-only",
                               f"-I{os.path.dirname(HEADER)}", "-I/opt/rocm/include",
                               "-D__HIP_PLATFORM_AMD__", str(src)])


BAD_CACHES = [
    (dict(k=None), EARG), (dict(v=None), EARG), (dict(pages=0), EARG), (dict(kv_heads=-1), EARG),
    (dict(page_size=48), EUNSUPPORTED), (dict(page_size=0), EUNSUPPORTED),
    (dict(page_size=512), EUNSUPPORTED), (dict(head_dim=80), EUNSUPPORTED),
    (dict(head_dim=512), EUNSUPPORTED), (dict(dtype=3), EUNSUPPORTED),
    (dict(mx=1, dtype=0, k_scale=0x50000, v_scale=0x60000), EUNSUPPORTED),
    (dict(mx=1), EARG), (dict(mx=1, k_scale=0x50000), EARG), (dict(k=0x10008), EARG),
    (dict(mass=None), EARG), (dict(position=None), EARG),
]


@pytest.mark.parametrize("kw,code", BAD_CACHES, ids=[str(k) for k, _ in BAD_CACHES])
def test_bad_caches_are_refused_by_every_entry_point(kv, lib, kw, code):
    c = ctypes.byref(desc(kv, **kw))
    assert lib.vramc_kv_append(c, P, 256, 128, P, 256, 128, P, P, 1, None) == code
    assert lib.vramc_kv_read(c, P, 1, P, P, None) == code
    assert lib.vramc_kv_attend_workspace(c, 4, 8, 1, 0) == code
    assert lib.vramc_kv_attend(c, P, 512, 128, 4, P, 8, 8, P, 1, 0.1, 0, P, P, 1 << 40, None) == code
    assert lib.vramc_kv_evict_workspace(c, 8, 1, 64, 0) == code
    assert lib.vramc_kv_evict(c, P, 8, 8, P, P, 1, 64, 0, None, 0, 0, P, P, 1 << 40, None) == code


def test_append_and_read_refuse(kv, lib):
    c = ctypes.byref(desc(kv))
    ok = [c, P, 256, 128, P, 256, 128, P, P, 4, None]
    for i, value in ((0, None), (1, None), (4, None), (7, None), (8, None), (9, -1), (9, 1 << 60)):
        bad = list(ok)
        bad[i] = value
        assert lib.vramc_kv_append(*bad) == EARG, i
    assert lib.vramc_kv_append(c, None, 0, 0, None, 0, 0, None, None, 0, None) == 0  # no tokens
    for bad in ((None, P, 4, P, P), (c, None, 4, P, P), (c, P, -1, P, P), (c, P, 4, None, P),
                (c, P, 4, P, None), (c, P, 4, ctypes.c_void_p(0x10008), P), (c, P, 1 << 60, P, P)):
        assert lib.vramc_kv_read(*bad, None) == EARG
    assert lib.vramc_kv_read(c, None, 0, None, None, None) == 0


def test_attend_refuses(kv, lib):
    c = ctypes.byref(desc(kv))
    plain = ctypes.byref(desc(kv, mass=None, position=None))
    for heads, width, batch in ((0, 8, 1), (3, 8, 1), (-2, 8, 1), (4, -1, 1), (4, 1 << 30, 1),
                                (4, 8, -1), (4, 8, 1 << 30)):
        assert lib.vramc_kv_attend_workspace(c, heads, width, batch, 1) == EARG
        assert lib.vramc_kv_attend(c, P, 512, 128, heads, P, 8, width, P, batch, 0.1, 1, P, P,
                                   1 << 60, None) == EARG
    need = lib.vramc_kv_attend_workspace(c, 4, 8, 3, 1)
    assert need > 0
    ok = [c, P, 512, 128, 4, P, 8, 8, P, 3, 0.1, 1, P, P, need, None]
    for i, value, code in ((1, None, EARG), (5, None, EARG), (8, None, EARG), (12, None, EARG),
                           (0, plain, EARG), (13, None, EWORKSPACE), (14, need - 1, EWORKSPACE)):
        bad = list(ok)
        bad[i] = value
        assert lib.vramc_kv_attend(*bad) == code, i
    ok[9] = 0  # no sequences
    assert lib.vramc_kv_attend(*ok) == 0


def test_evict_refuses(kv, lib):
    c = ctypes.byref(desc(kv))
    plain = ctypes.byref(desc(kv, mass=None, position=None))
    for width, batch, budget in ((-1, 1, 64), (8, -1, 64), (8, 1, 0), (8, 1, -5), (1 << 30, 1, 64),
                                 (8, 1 << 30, 64)):
        assert lib.vramc_kv_evict_workspace(c, width, batch, budget, 0) == EARG
        assert lib.vramc_kv_evict(c, P, 8, width, P, P, batch, budget, 0, None, 0, 0, P, P, 1 << 60,
                                  None) == EARG
    need = lib.vramc_kv_evict_workspace(c, 8, 3, 100, 1)
    assert need > 0
    ok = [c, P, 8, 8, P, P, 3, 100, 5, P, 2, 2, P, P, need, None]
    for i, value, code in ((0, plain, EARG), (1, None, EARG), (4, None, EARG), (5, None, EARG),
                           (8, -1, EARG), (11, 1, EARG), (12, None, EARG), (13, None, EWORKSPACE),
                           (14, need - 1, EWORKSPACE)):
        bad = list(ok)
        bad[i] = value
        assert lib.vramc_kv_evict(*bad) == code, i
    ok[6] = 0  # no sequences
    assert lib.vramc_kv_evict(*ok) == 0


def test_fails_loudly_without_gpu(kv):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    with pytest.raises(RuntimeError):
        kv.PagedCache.allocate(4, 2, 128)
    with pytest.raises(RuntimeError):
        kv.PagedCache(torch.zeros(4, 2, 64, 128), torch.zeros(4, 2, 64, 128), torch.float32)


def test_refuses_what_no_grid_holds(kv, lib):
    """A launch has fewer than 2^32 threads: what would need more is an argument
    refused, not a failed launch."""
    c = ctypes.byref(desc(kv))
    assert lib.vramc_kv_append(c, P, 256, 128, P, 256, 128, P, P, 1 << 28, None) == EARG
    assert lib.vramc_kv_read(c, P, 1 << 28, P, P, None) == EARG
    for heads, width, batch in ((2, 1, (1 << 21) + 1), (4, 1 << 17, 1 << 13)):
        assert lib.vramc_kv_attend_workspace(c, heads, width, batch, 1) == EARG
    assert lib.vramc_kv_attend_workspace(c, 2, 1, 1 << 21, 0) > 0
    assert lib.vramc_kv_evict_workspace(c, 1 << 24, 1, 1 << 30, 1) == EARG
    assert lib.vramc_kv_evict_workspace(c, 1 << 23, 1, 1 << 29, 1) > 0


def test_slots_of_padding(kv):
    """Indexes without a page have no slot: negative ones, those beyond the
    table, those of a table without pages."""
    import types

    import torch
    cache = types.SimpleNamespace(page_size=16)
    table = torch.tensor([[3, -1, 5], [0, 2, 7]], dtype=torch.int32)
    sequence = torch.tensor([0, 0, 0, 0, 0, 1, 1, 1, 1], dtype=torch.int32)
    index = torch.tensor([0, 15, 16, 47, 48, -1, -16, -17, 20], dtype=torch.int32)
    got = kv.PagedCache.slots(cache, table, sequence, index)
    assert got.dtype is torch.int64
    assert got.tolist() == [48, 63, -1, 95, -1, -1, -1, -1, 36]
    assert kv.PagedCache.slots(cache, table[:, :0], sequence, index).tolist() == [-1] * 9
