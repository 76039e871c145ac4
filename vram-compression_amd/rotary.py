"""Rotation of queries and keys by their tokens' positions, with the RMS norms of
each head that newer models put before it, in one pass over them:

    turn = rotary.Rotary(head_dim, base=1e6)
    q, k = turn.rotate(q, k, positions, q_weight, k_weight)
    q = turn.append(cache, q, k, v, slots, positions, q_weight, k_weight)

append writes the rotated keys and the values straight into the pages of a
kv_cache.PagedCache.  Hand-written HIP kernels in librans_hip.so
(include/vramc_rotary.h) on the current stream; no CPU fallback, no gradient.
"""
import ctypes
import math

import torch

import kv_cache
import rans

EXPORTS = ("vramc_rotary_apply", "vramc_rotary_append")
_DTYPES = rans._X_CODES
_check = kv_cache._check


class RotaryDesc(ctypes.Structure):
    """ctypes mirror of vramc_rotary (include/vramc_rotary.h)."""
    _fields_ = [("head_dim", ctypes.c_int32), ("pairs", ctypes.c_int32), ("interleaved", ctypes.c_int32),
                ("amplitude", ctypes.c_float), ("turns", ctypes.c_void_p)]


class RowsDesc(ctypes.Structure):
    """ctypes mirror of vramc_rotary_rows (include/vramc_rotary.h)."""
    _fields_ = [("q", ctypes.c_void_p), ("k", ctypes.c_void_p),
                ("q_token", ctypes.c_int64), ("q_head", ctypes.c_int64),
                ("k_token", ctypes.c_int64), ("k_head", ctypes.c_int64),
                ("q_heads", ctypes.c_int32), ("k_heads", ctypes.c_int32),
                ("q_weight", ctypes.c_void_p), ("k_weight", ctypes.c_void_p),
                ("dtype", ctypes.c_int32), ("weight_dtype", ctypes.c_int32), ("eps", ctypes.c_float),
                ("positions", ctypes.c_void_p), ("tokens", ctypes.c_int64)]


def bind(lib):
    """Sets the argument types of the rotation's entry points on a handle of
    librans_hip.so and returns it; raises AttributeError if one is missing."""
    if not getattr(lib, "_rotary_bound", False):
        P, I64 = ctypes.c_void_p, ctypes.c_int64
        D, R = ctypes.POINTER(RotaryDesc), ctypes.POINTER(RowsDesc)
        C = ctypes.POINTER(kv_cache.KvCacheDesc)
        kv_cache.set_types(lib, {
            "vramc_rotary_apply": ([D, R, P, P, P], ctypes.c_int),
            "vramc_rotary_append": ([D, R, C, P, I64, I64, P, P, P], ctypes.c_int),
        })
        lib._rotary_bound = True
    return lib


class Rotary(kv_cache.Calls):
    """The rotation of a model's heads of head_dim columns (64, 96, 128, 192 or 256):
    the first rotary_dim of them (all unless given; a multiple of 16) rotate in pairs,
    column i with i + rotary_dim / 2, or, interleaved, 2i with 2i + 1, by position *
    base**(-2i / rotary_dim).  inverse: other frequencies (radians a position, a value
    for each pair, taken in 64 bits), as models that stretch their positions have them,
    in place of base and rotary_dim; amplitude: a factor of what rotates, as they have
    beside them."""

    def __init__(self, head_dim, base=10000.0, rotary_dim=None, interleaved=False, inverse=None,
                 amplitude=1.0, device="cuda", lib=None):
        if not torch.cuda.is_available():
            raise RuntimeError("Rotary needs a ROCm GPU (gfx950); no CPU fallback exists")
        _check(head_dim in kv_cache.HEAD_DIMS, f"head dimension {head_dim}: one of {kv_cache.HEAD_DIMS}")
        if inverse is None:
            rotary_dim = head_dim if rotary_dim is None else rotary_dim
            _check(rotary_dim % 2 == 0 and base > 0, f"rotary_dim {rotary_dim}, base {base}: even, positive")
            inverse = torch.tensor([base ** (-2 * i / rotary_dim) for i in range(rotary_dim // 2)],
                                   dtype=torch.float64)
        else:
            inverse = inverse.detach().double()
            _check(inverse.dim() == 1 and rotary_dim in (None, 2 * inverse.numel()),
                   f"inverse: a value for each pair of columns, got {tuple(inverse.shape)}")
        self.head_dim, self.rotary_dim, self.interleaved = head_dim, 2 * inverse.numel(), bool(interleaved)
        _check(0 < self.rotary_dim <= head_dim and self.rotary_dim % 16 == 0,
               f"{self.rotary_dim} columns that rotate: a multiple of 16, at most {head_dim}")
        self._turns = (inverse / (2 * math.pi)).to(device).contiguous()  # full turns a position
        _check(self._turns.is_cuda, f"device {device}: a ROCm GPU")
        self.device, self._index = self._turns.device, self._turns.get_device()
        self.lib = bind(lib or rans._host_lib())
        self._desc = RotaryDesc(head_dim, inverse.numel(), int(self.interleaved), amplitude,
                                self._turns.data_ptr())
        self._ref = ctypes.byref(self._desc)

    def _refuse(self, tokens, dtype, index, **rows):
        """Says which of the rows is not as it has to be."""
        _check(dtype in _DTYPES, f"no rotation of {dtype}: bf16, f16 or f32")
        for name, t in rows.items():
            got = tuple(t.shape)
            if (len(got) != 3 or got[2] != self.head_dim or t.dtype is not dtype or got[0] != tokens
                    or t.get_device() != index):
                raise ValueError(f"{name} must be ({tokens}, heads, {self.head_dim}) of {dtype} on "
                                 f"{self.device}, got {got} of {t.dtype} on {t.device}")

    def _weight(self, name, w, dtype):
        """Checks a norm's weight; its address and type."""
        kind = w.dtype
        if (w.shape != (self.head_dim,) or not w.is_contiguous() or w.get_device() != self._index
                or (kind is not dtype and kind is not torch.float32) or w.data_ptr() % 16):
            raise ValueError(f"{name} must be {self.head_dim} dense values of {dtype} or torch.float32 on "
                             f"{self.device}, aligned to 16 bytes; got {tuple(w.shape)} of {kind} on {w.device}")
        if w.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} requires a gradient; the rotation has none: detach it or use "
                             "torch.no_grad()")
        return w.data_ptr(), kind

    def _taken(self, q, k, positions, q_weight, k_weight, eps):
        """Checks the arguments; the descriptor of the rows, and q and k as they are
        read (a last dimension that is not dense is copied)."""
        dtype, index, qs, ks = q.dtype, self._index, q.shape, k.shape
        tokens = qs[0] if qs else 0
        if (dtype not in _DTYPES or len(qs) != 3 or len(ks) != 3 or qs[2] != self.head_dim
                or ks[2] != self.head_dim or ks[0] != tokens or k.dtype is not dtype
                or q.get_device() != index or k.get_device() != index):
            self._refuse(tokens, dtype, index, q=q, k=k)
        if (q.requires_grad or k.requires_grad) and torch.is_grad_enabled():
            raise ValueError("q or k requires a gradient; the rotation has none: detach it or use "
                             "torch.no_grad()")
        self._ints("positions", positions, torch.int32, (tokens,))
        q_at = k_at = None
        kind = dtype
        if q_weight is not None:
            q_at, kind = self._weight("q_weight", q_weight, dtype)
        if k_weight is not None:
            k_at, k_kind = self._weight("k_weight", k_weight, dtype)
            if q_at is not None and k_kind is not kind:
                raise ValueError(f"the weights are of {kind} and {k_kind}: one type for both")
            kind = k_kind
        if not eps >= 0:
            raise ValueError(f"eps {eps}: not negative")
        q_token, q_head, q_column = q.stride()
        k_token, k_head, k_column = k.stride()
        if q_column != 1:
            q = q.contiguous()
            q_token, q_head, _ = q.stride()
        if k_column != 1:
            k = k.contiguous()
            k_token, k_head, _ = k.stride()
        rows = RowsDesc(q.data_ptr(), k.data_ptr(), q_token, q_head, k_token, k_head, qs[1], ks[1], q_at, k_at,
                        _DTYPES[dtype], _DTYPES[kind], eps, positions.data_ptr(), tokens)
        return rows, q, k

    def rotate(self, q, k, positions, q_weight=None, k_weight=None, eps=1e-6):
        """The queries (tokens, heads, head_dim) and keys (tokens, kv heads, head_dim; bf16,
        f16 or f32, any strides) of tokens at positions (int32), rotated, as new tensors.
        Where a weight (head_dim) is given, a head is first x * weight / sqrt(mean(x^2) +
        eps).  Computed in f32, angles in 64 bits, rounded once."""
        stream = self._stream()
        rows, q, k = self._taken(q, k, positions, q_weight, k_weight, eps)
        q_out, k_out = q.new_empty(q.shape), k.new_empty(k.shape)
        rc = self.lib.vramc_rotary_apply(self._ref, ctypes.byref(rows), q_out.data_ptr(), k_out.data_ptr(),
                                         stream)
        if rc:
            kv_cache._failed("rotate", rc)
        return q_out, k_out

    def append(self, cache, q, k, v, slots, positions, q_weight=None, k_weight=None, eps=1e-6):
        """rotate, with the keys and the values v (as k, any strides) written into slots
        (int64) of a cache, as PagedCache.append writes them; a tracked one takes the
        positions too.  Returns the queries, also of tokens without a slot (-1).  What is
        read lies in none of the cache's tensors."""
        if cache.head_dim != self.head_dim or cache.dtype is not q.dtype or cache._index != self._index:
            raise ValueError(f"a cache of {cache.dtype} heads of {cache.head_dim} on {cache.device} takes no "
                             f"{q.dtype} of {self.head_dim} on {self.device}")
        stream = cache._stream()
        rows, q, k = self._taken(q, k, positions, q_weight, k_weight, eps)
        shape = k.shape
        tokens = shape[0]
        if shape[1] != cache.kv_heads:
            raise ValueError(f"keys of {shape[1]} heads and a cache of {cache.kv_heads}")
        if v.shape != shape or v.dtype is not q.dtype or v.get_device() != self._index:
            raise ValueError(f"v must be {tuple(shape)} of {q.dtype} on {self.device}, got {tuple(v.shape)} of "
                             f"{v.dtype} on {v.device}")
        if v.requires_grad and torch.is_grad_enabled():
            raise ValueError("v requires a gradient; the cache has none: detach it or use torch.no_grad()")
        self._ints("slots", slots, torch.int64, (tokens,))
        v_token, v_head, v_column = v.stride()
        if v_column != 1:
            v = v.contiguous()
            v_token, v_head, _ = v.stride()
        q_out = q.new_empty(q.shape)
        rc = self.lib.vramc_rotary_append(self._ref, ctypes.byref(rows), cache._ref, v.data_ptr(), v_token,
                                          v_head, slots.data_ptr(), q_out.data_ptr(), stream)
        if rc:
            kv_cache._failed("append", rc)
        return q_out
