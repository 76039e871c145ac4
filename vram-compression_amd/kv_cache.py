"""The key-value cache of a served model on MI355X: pages of keys and values
in the model's type or in 4 bits, the attention of one new token over them, and
eviction by accumulated attention weight.

The weights are one part of a served model's memory, the cache of past tokens
the other; the reference stops at the weights (README.md:39 names model
integration as its next step), so nothing here has a counterpart there.
PagedCache holds that cache:

    cache = kv_cache.PagedCache.allocate(pages, kv_heads, head_dim, mx=True, track=True)
    cache.append(k, v, cache.slots(table, sequence, index), positions)  # new tokens
    out = cache.attend(q, table, lengths)                 # one new token of each sequence
    lengths = cache.evict(table, lengths, seen, budget, recent)

A sequence's tokens lie in the pages that its row of `table` names, in order;
which pages are free is the program's to keep.  Every operation is a
hand-written HIP kernel in librans_hip.so (include/vramc_kv.h), runs on the
current stream and allocates from torch.  There is no CPU fallback, and nothing
that torch could watch: calls under a gradient, forward mode, vmap, a tracer, a
dispatch or a function mode are refused (a compiled program breaks at a call
and makes it).
"""
import ctypes

import torch

import rans
from rans_linear import _watched

MX_BLOCK = 32  # columns that share a scale byte
PAGE_SIZES = (16, 32, 64, 128, 256)
HEAD_DIMS = (64, 96, 128, 192, 256)
_DTYPES = rans._X_CODES

EXPORTS = ("vramc_kv_append", "vramc_kv_read", "vramc_kv_attend_workspace", "vramc_kv_attend",
           "vramc_kv_evict_workspace", "vramc_kv_evict")


class KvCacheDesc(ctypes.Structure):
    """ctypes mirror of vramc_kv_cache (include/vramc_kv.h)."""
    _fields_ = [("pages", ctypes.c_int32), ("kv_heads", ctypes.c_int32),
                ("page_size", ctypes.c_int32), ("head_dim", ctypes.c_int32),
                ("dtype", ctypes.c_int32), ("mx", ctypes.c_int32),
                ("k", ctypes.c_void_p), ("v", ctypes.c_void_p),
                ("k_scale", ctypes.c_void_p), ("v_scale", ctypes.c_void_p),
                ("mass", ctypes.c_void_p), ("position", ctypes.c_void_p)]


def bind(lib):
    """Sets the argument types of the cache's entry points on a handle of
    librans_hip.so and returns it; raises AttributeError if one is missing."""
    if getattr(lib, "_kv_bound", False):
        return lib
    P, I32, I64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64
    D = ctypes.POINTER(KvCacheDesc)
    sig = {
        "vramc_kv_append": ([D, P, I64, I64, P, I64, I64, P, P, I64, P], I32),
        "vramc_kv_read": ([D, P, I64, P, P, P], I32),
        "vramc_kv_attend_workspace": ([D, I32, I32, I32, I32], I64),
        "vramc_kv_attend": ([D, P, I64, I64, I32, P, I64, I32, P, I32, ctypes.c_float, I32, P, P,
                             I64, P], I32),
        "vramc_kv_evict_workspace": ([D, I32, I32, I32, I32], I64),
        "vramc_kv_evict": ([D, P, I64, I32, P, P, I32, I32, I32, P, I64, I32, P, P, I64, P], I32),
    }
    for name, (args, res) in sig.items():
        f = getattr(lib, name)
        f.argtypes = args
        f.restype = res
    lib._kv_bound = True
    return lib


def _check(ok, message):
    if not ok:
        raise ValueError(message)


def _failed(name, rc):
    """Raises what a return value of the library says."""
    if rc < 0:
        raise ValueError(f"{name}: refused by the library ({rc}): more than one launch holds, or a tensor "
                         "less aligned than the kernels read")
    raise RuntimeError(f"{name}: HIP error {rc}")


class PagedCache:
    """Keys and values of past tokens in pages on the GPU.

    k, v: (pages, kv_heads, page_size, head_dim) of dtype (bf16, f16 or f32),
    or, with k_scale and v_scale, 4-bit codes: uint8 (.., head_dim / 2) and a
    scale byte for every 32 columns, uint8 (.., head_dim / 32) (bf16 or f16
    values; the MXFP4 format, 4.25 bits a value).  mass (f32) and position
    (int32), (pages, kv_heads, page_size), where tokens' accumulated weights are
    tracked.  The tensors are used as they are, not copied, and a cache keeps those
    that it was made of."""

    # The descriptor holds their addresses: not to be assigned.
    k = property(lambda self: self._k)
    v = property(lambda self: self._v)
    k_scale = property(lambda self: self._k_scale)
    v_scale = property(lambda self: self._v_scale)
    mass = property(lambda self: self._mass)
    position = property(lambda self: self._position)

    def __init__(self, k, v, dtype=torch.bfloat16, k_scale=None, v_scale=None, mass=None,
                 position=None, lib=None):
        if not torch.cuda.is_available():
            raise RuntimeError("PagedCache needs a ROCm GPU (gfx950); no CPU fallback exists")
        _check(k.dim() == 4, "k must be (pages, kv_heads, page_size, head_dim)")
        _check(dtype in _DTYPES, f"no cache of {dtype}: bf16, f16 or f32")
        self.mx = k_scale is not None
        _check(self.mx == (v_scale is not None), "k_scale and v_scale come together")
        _check(not (self.mx and dtype is torch.float32), "4-bit storage takes bf16 or f16 values")
        self.pages, self.kv_heads, self.page_size, width = k.shape
        self.head_dim = width * 2 if self.mx else width
        _check(self.pages > 0 and self.kv_heads > 0, "an empty cache")
        _check(self.page_size in PAGE_SIZES, f"page size {self.page_size}: one of {PAGE_SIZES}")
        _check(self.head_dim in HEAD_DIMS, f"head dimension {self.head_dim}: one of {HEAD_DIMS}")
        held = torch.uint8 if self.mx else dtype
        lead = tuple(k.shape[:3])
        want = [("k", k, held, (*lead, width)), ("v", v, held, (*lead, width))]
        if self.mx:
            scales = (*lead, self.head_dim // MX_BLOCK)
            want += [("k_scale", k_scale, torch.uint8, scales),
                     ("v_scale", v_scale, torch.uint8, scales)]
        _check((mass is None) == (position is None), "mass and position come together")
        if mass is not None:
            want += [("mass", mass, torch.float32, lead), ("position", position, torch.int32, lead)]
        for name, t, dt, shape in want:
            if not (t.is_cuda and t.device == k.device and t.dtype is dt and t.shape == shape
                    and t.is_contiguous()):
                raise ValueError(f"{name} must be a contiguous {dt} tensor {shape} on {k.device}, got "
                                 f"{t.dtype} {tuple(t.shape)} on {t.device}")
            if t.data_ptr() % 16 and not name.endswith("scale"):
                raise ValueError(f"{name} must be 16-byte aligned")
        self._k, self._v, self._k_scale, self._v_scale = k, v, k_scale, v_scale
        self._mass, self._position, self.dtype, self.device = mass, position, dtype, k.device
        self._index = k.get_device()
        self.lib = bind(lib or rans._host_lib())
        ptr = {n: t.data_ptr() for n, t, _, _ in want}
        self._desc = KvCacheDesc(pages=self.pages, kv_heads=self.kv_heads,
                                 page_size=self.page_size, head_dim=self.head_dim,
                                 dtype=_DTYPES[dtype], mx=int(self.mx), **ptr)
        self._ref = ctypes.byref(self._desc)
        self.nbytes = sum(t.numel() * t.element_size() for _, t, _, _ in want)

    @classmethod
    def allocate(cls, pages, kv_heads, head_dim, page_size=64, dtype=torch.bfloat16, mx=False,
                 track=False, device="cuda", lib=None):
        """A cache of `pages` free pages.  mx: 4-bit storage; track: with mass
        and position, which evict needs and attend and append then keep."""
        if not torch.cuda.is_available():
            raise RuntimeError("PagedCache needs a ROCm GPU (gfx950); no CPU fallback exists")
        lead = (pages, kv_heads, page_size)

        def zeros(dt, *last):
            return torch.zeros(*lead, *last, dtype=dt, device=device)

        _check(head_dim in HEAD_DIMS, f"head dimension {head_dim}: one of {HEAD_DIMS}")
        if mx:
            k, v = (zeros(torch.uint8, head_dim // 2) for _ in range(2))
            scales = [zeros(torch.uint8, head_dim // MX_BLOCK) for _ in range(2)]
        else:
            k, v = (zeros(dtype, head_dim) for _ in range(2))
            scales = [None, None]
        more = [zeros(torch.float32), zeros(torch.int32)] if track else [None, None]
        return cls(k, v, dtype, *scales, *more, lib=lib)

    # ------------------------------------------------------------- arguments
    # The checks run on every token step: messages are made only for a failure.
    def _stream(self):
        """The current stream, for a call that nothing watches."""
        if _watched():
            raise ValueError("forward mode, vmap, a tracer or a dispatch or function mode watches this "
                             "call, and the cache's operations are hidden from them")
        if torch.is_grad_enabled() and (self._k.requires_grad or self._v.requires_grad or (
                self._mass is not None and self._mass.requires_grad)):
            raise ValueError("the cache's tensors require a gradient, and its operations have none: "
                             "detach them or use torch.no_grad()")
        if rans._device() != self._index:
            raise ValueError(f"the cache is on {self.device}, the current device is another")
        return rans._stream()

    def _ints(self, name, t, dtype, shape):
        """Checks integers of a shape (None for any size) whose last dimension
        is dense."""
        got = t.shape
        if (t.dtype is not dtype or t.get_device() != self._index or len(got) != len(shape)
                or (got[0] != shape[0] and shape[0] is not None)
                or (got[-1] > 1 and t.stride(-1) != 1)):
            want = tuple("n" if n is None else n for n in shape)
            raise ValueError(f"{name} must be {want} of {dtype} on {self.device}, its last dimension "
                             f"dense; got {tuple(got)} of {t.dtype} on {t.device}, strides {t.stride()}")

    def _rows(self, name, t, heads):
        """Checks rows x heads x head_dim values; a last dimension that is not
        dense is copied."""
        got = t.shape
        if (len(got) != 3 or got[2] != self.head_dim or t.dtype is not self.dtype
                or t.get_device() != self._index or (heads is not None and got[1] != heads)):
            raise ValueError(f"{name} must be (n, {heads or 'heads'}, {self.head_dim}) of {self.dtype} "
                             f"on {self.device}, got {tuple(got)} of {t.dtype} on {t.device}")
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} requires a gradient; the cache has none: detach it or use "
                             "torch.no_grad()")
        return t if t.stride(2) == 1 else t.contiguous()

    def slots(self, table, sequence, index):
        """The slots (int64) of tokens `index` of sequences `sequence` (rows of
        table), -1 where the table has no page for them (a negative index, as of
        padding, among them)."""
        index, width = index.long(), table.shape[1]
        if width == 0:
            return torch.full_like(index, -1)
        page = torch.div(index, self.page_size, rounding_mode="floor")
        known = (page >= 0) & (page < width)
        page = table[sequence.long(), page.clamp(0, width - 1)].long()
        slot = page * self.page_size + index % self.page_size
        return torch.where(known & (page >= 0), slot, -1)

    # ------------------------------------------------------------ operations
    def append(self, k, v, slots, positions=None):
        """Writes the keys and values of new tokens, (tokens, kv_heads,
        head_dim) at any strides, into slots (int64; page * page_size + place,
        -1 for none).  positions (int32): the tokens' positions, for a tracked
        cache, whose mass starts at 0."""
        stream = self._stream()
        k, v = self._rows("k", k, self.kv_heads), self._rows("v", v, self.kv_heads)
        n = k.shape[0]
        if v.shape[0] != n:
            raise ValueError(f"{n} keys and {v.shape[0]} values")
        self._ints("slots", slots, torch.int64, (n,))
        at = None
        if self._mass is not None:
            if positions is None:
                raise ValueError("a tracked cache needs the tokens' positions")
            self._ints("positions", positions, torch.int32, (n,))
            at = positions.data_ptr()
        rc = self.lib.vramc_kv_append(self._ref, k.data_ptr(), k.stride(0), k.stride(1),
                                      v.data_ptr(), v.stride(0), v.stride(1), slots.data_ptr(), at,
                                      n, stream)
        if rc:
            _failed("append", rc)

    def read(self, slots):
        """The keys and values in slots (int64), (tokens, kv_heads, head_dim)
        of the cache's dtype; zeros for a slot outside the cache."""
        stream = self._stream()
        self._ints("slots", slots, torch.int64, (None,))
        n = slots.shape[0]
        k = torch.empty((n, self.kv_heads, self.head_dim), dtype=self.dtype, device=self.device)
        v = torch.empty_like(k)
        rc = self.lib.vramc_kv_read(self._ref, slots.data_ptr(), n, k.data_ptr(), v.data_ptr(), stream)
        if rc:
            _failed("read", rc)
        return k, v

    def attend(self, q, table, lengths, scale=None, track=None):
        """Attention of one new token of each sequence over its cached tokens:
        q (sequences, q_heads, head_dim) of the cache's dtype, table (sequences,
        pages; int32, -1 for none), lengths (int32).  Returns (sequences,
        q_heads, head_dim); a sequence without tokens gets zeros.  scale:
        head_dim**-0.5 unless given.  track: whether every token's weight,
        summed over the query heads of its kv head, is added to mass; by default
        where the cache has it.  The table's width bounds the lengths: one cut
        to the pages in use (table[:, :n]) spares what longer ones would need."""
        stream = self._stream()
        q = self._rows("q", q, None)
        batch, heads, _ = q.shape
        if heads <= 0 or heads % self.kv_heads:
            raise ValueError(f"{heads} query heads are no multiple of {self.kv_heads} kv heads")
        self._ints("table", table, torch.int32, (batch, None))
        self._ints("lengths", lengths, torch.int32, (batch,))
        if track is None:
            track = self._mass is not None
        elif track and self._mass is None:
            raise ValueError("the cache was made without track")
        width = table.shape[1]
        out = torch.empty_like(q) if q.is_contiguous() else \
            torch.empty((batch, heads, self.head_dim), dtype=self.dtype, device=self.device)
        need = self.lib.vramc_kv_attend_workspace(self._ref, heads, width, batch, track)
        if need < 0:
            raise ValueError(f"{batch} sequences of {heads} heads over {width} pages: too many ({need})")
        work = torch.empty(need, dtype=torch.uint8, device=self.device)
        rc = self.lib.vramc_kv_attend(
            self._ref, q.data_ptr(), q.stride(0), q.stride(1), heads, table.data_ptr(),
            table.stride(0), width, lengths.data_ptr(), batch,
            self.head_dim ** -0.5 if scale is None else scale, track, out.data_ptr(),
            work.data_ptr(), need, stream)
        if rc:
            _failed("attend", rc)
        return out

    def evict(self, table, lengths, seen, budget, recent=0, into=None):
        """Cuts every sequence longer than budget to that many tokens, each kv
        head by itself: those with position >= seen - recent (seen: int32, the
        tokens that each sequence has seen so far) are kept first, then those of
        the largest mass, ties to the lower index; tokens without a page are
        never kept, and where places have none as many fewer tokens are.  Returns
        the new lengths, min(lengths, budget).  By default in place: tokens kept
        beyond the budget move into the freed places below it, so the pages must
        belong to one sequence alone; the pages beyond the new lengths are free.
        into: a table of other pages, which all kept tokens are copied to in
        order, while the sequences' own pages stay as they are; a new length is
        less where tokens without a page leave fewer."""
        if self._mass is None:
            raise ValueError("the cache was made without track")
        stream = self._stream()
        self._ints("table", table, torch.int32, (None, None))
        batch, width = table.shape
        self._ints("lengths", lengths, torch.int32, (batch,))
        self._ints("seen", seen, torch.int32, (batch,))
        if not 0 < budget < 2 ** 31:
            raise ValueError(f"budget {budget}: a positive number of tokens")
        if not 0 <= recent <= budget:
            raise ValueError(f"recent {recent}: 0 to the budget")
        other, row, wide = None, 0, 0
        if into is not None:
            self._ints("into", into, torch.int32, (batch, None))
            other, row, wide = into.data_ptr(), into.stride(0), into.shape[1]
            if wide * self.page_size < min(budget, width * self.page_size):
                raise ValueError(f"into has no room for {budget} tokens")
        need = self.lib.vramc_kv_evict_workspace(self._ref, width, batch, budget, into is not None)
        if need < 0:
            raise ValueError(f"{batch} sequences over {width} pages: too many ({need})")
        work = torch.empty(need, dtype=torch.uint8, device=self.device)
        out = torch.empty(batch, dtype=torch.int32, device=self.device)
        rc = self.lib.vramc_kv_evict(
            self._ref, table.data_ptr(), table.stride(0), width, lengths.data_ptr(),
            seen.data_ptr(), batch, budget, recent, other, row, wide, out.data_ptr(),
            work.data_ptr(), need, stream)
        if rc:
            _failed("evict", rc)
        return out
