"""Which pages of a key-value cache are free, kept on the GPU: a step's block table
and slots are made there from the sequences' lengths, with no word to the host.

    pool = kv_pages.PagePool(cache.pages, cache.page_size)
    step = pool.extend(table, lengths, new, tokens)       # room for new tokens
    cache.append(k, v, step.slots, step.positions)
    out = cache.attend(q, table, step.lengths)
    ...
    pool.release(table, lengths)                          # pages behind lengths

Each operation is a hand-written HIP kernel in librans_hip.so
(include/vramc_pages.h) on the current stream, as kv_cache's are, and there is no
CPU fallback.
"""
import collections
import ctypes

import torch

import kv_cache
import rans

EXPORTS = ("vramc_pages_extend", "vramc_pages_release_workspace", "vramc_pages_release")
MOST_SEQUENCES = 4096

# What extend returns.
Step = collections.namedtuple("Step", "slots positions filled starts lengths")


class PagesDesc(ctypes.Structure):
    """ctypes mirror of vramc_pages (include/vramc_pages.h)."""
    _fields_ = [("pages", ctypes.c_int32), ("page_size", ctypes.c_int32), ("free", ctypes.c_void_p),
                ("count", ctypes.c_void_p), ("ticket", ctypes.c_void_p)]


def bind(lib):
    """Sets the argument types of the pool's entry points on a handle of
    librans_hip.so and returns it; raises AttributeError if one is missing."""
    if not getattr(lib, "_pages_bound", False):
        P, I32, I64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64
        D = ctypes.POINTER(PagesDesc)
        kv_cache.set_types(lib, {
            "vramc_pages_extend": ([D, P, I64, I32, P, P, P, I32, I64, P, P, P, P, P, P], I32),
            "vramc_pages_release_workspace": ([D, I32, I32], I64),
            "vramc_pages_release": ([D, P, I64, I32, P, I32, P, I64, P], I32),
        })
        lib._pages_bound = True
    return lib


class PagePool(kv_cache.Calls):
    """The free pages of a cache, as a stack on the GPU: free (int32, one place for
    every page of the cache) holds them in its first count (int32, one value), the
    next to be taken last.  All pages are free unless both are given, which are then
    used as they are.  A page belongs to one row of one table at a time.  Calls that
    change a pool run one after the other (one stream, or events between them)."""

    free = property(lambda self: self._free)
    count = property(lambda self: self._count)

    def __init__(self, pages, page_size=64, free=None, count=None, device="cuda", lib=None):
        if not torch.cuda.is_available():
            raise RuntimeError("PagePool needs a ROCm GPU (gfx950); no CPU fallback exists")
        if not 0 < pages < 2 ** 31 or page_size not in kv_cache.PAGE_SIZES:
            raise ValueError(f"{pages} pages of {page_size} tokens: a positive number of pages of one of "
                             f"{kv_cache.PAGE_SIZES}")
        if (free is None) != (count is None):
            raise ValueError("free and count come together")
        if free is None:
            free = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=device)
            count = torch.full((1,), pages, dtype=torch.int32, device=device)
        for name, t, n in (("free", free, pages), ("count", count, 1)):
            if not (t.is_cuda and t.device == free.device and t.dtype is torch.int32 and t.shape == (n,)
                    and t.is_contiguous()):
                raise ValueError(f"{name} must be {n} dense int32 values on a GPU, got {t.dtype} "
                                 f"{tuple(t.shape)} on {t.device}")
        self.pages, self.page_size = pages, page_size
        self._free, self._count, self.device, self._index = free, count, free.device, free.get_device()
        self._ticket = torch.zeros(1, dtype=torch.int32, device=free.device)
        self._long = torch.empty(0, dtype=torch.int64, device=free.device)  # what slots are made like
        # of calls that run one after the other
        self._work = torch.empty(MOST_SEQUENCES + 1, dtype=torch.int32, device=free.device)
        self.lib = bind(lib or rans._host_lib())
        self._desc = PagesDesc(pages, page_size, free.data_ptr(), count.data_ptr(), self._ticket.data_ptr())
        self._ref = ctypes.byref(self._desc)

    def _table(self, table, rows):
        self._ints("table", table, torch.int32, (rows, None))
        batch, width = table.shape
        if batch > MOST_SEQUENCES or (batch > 1 and table.stride(0) < width):
            raise ValueError(f"table: at most {MOST_SEQUENCES} rows, none over another; got "
                             f"{tuple(table.shape)}, strides {table.stride()}")
        return batch, width

    def extend(self, table, lengths, new, tokens, seen=None):
        """Room for new[b] (int32) more tokens of each sequence, which holds lengths[b]
        (int32) in the pages of its row of table (int32, written in place): all new
        tokens, sequence behind sequence, are the first rows of a batch of `tokens`.
        Returns, on the GPU,
        - slots (int64, tokens): where each row's keys and values go, -1 for rows that
          are no token or have no room;
        - positions (int32, tokens): seen[b] (int32; lengths[b] unless given) and on,
          0 for rows that are no token;
        - filled (int32, tokens): the page that the row's token makes full, or -1 (for
          PagedCache.bound);
        - starts (int32, sequences + 1): each sequence's first row, and the end;
        - lengths (int32): with the new tokens.
        A sequence whose tokens do not fit its row of the table or the batch, or whose
        pages, behind those that earlier sequences want, the pool does not have, gets
        none of them: its length stays."""
        batch, width = self._table(table, None)
        stream = self._stream()
        self._ints("lengths", lengths, torch.int32, (batch,))
        self._ints("new", new, torch.int32, (batch,))
        if seen is not None:
            self._ints("seen", seen, torch.int32, (batch,))
        if not 0 <= tokens < 2 ** 31 - 1:
            raise ValueError(f"{tokens} rows: 0 to 2**31 - 2")
        slots = self._long.new_empty(tokens)
        # one allocation for what has 32 bits: positions, filled, starts, lengths
        rest = self._ticket.new_empty(2 * (tokens + batch) + 1)
        positions, filled, starts, lengths_out = rest.split_with_sizes((tokens, tokens, batch + 1, batch))
        rc = self.lib.vramc_pages_extend(
            self._ref, table.data_ptr(), table.stride(0), width, lengths.data_ptr(), new.data_ptr(),
            None if seen is None else seen.data_ptr(), batch, tokens, slots.data_ptr(),
            positions.data_ptr(), filled.data_ptr(), starts.data_ptr(), lengths_out.data_ptr(), stream)
        if rc:
            kv_cache._failed("extend", rc)
        return Step(slots, positions, filled, starts, lengths_out)

    def release(self, table, lengths):
        """Puts the pages behind lengths (int32) tokens of each sequence back, in order
        of the table (int32), and -1 in their entries: of a sequence that is done (length
        0), was cut by an eviction, or had tokens that were refused."""
        batch, width = self._table(table, None)
        stream = self._stream()
        self._ints("lengths", lengths, torch.int32, (batch,))
        rc = self.lib.vramc_pages_release(self._ref, table.data_ptr(), table.stride(0), width,
                                          lengths.data_ptr(), batch, self._work.data_ptr(),
                                          4 * (MOST_SEQUENCES + 1), stream)
        if rc:
            kv_cache._failed("release", rc)
