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

    def _rows(self, name, t, tokens, dtype, heads=None):
        """Checks tokens x heads x head_dim values; a last dimension that is not dense
        is copied."""
        got = t.shape
        if (len(got) != 3 or got[2] != self.head_dim or t.dtype is not dtype or dtype not in _DTYPES
                or got[0] != tokens or t.get_device() != self._index or (heads is not None and got[1] != heads)):
            raise ValueError(f"{name} must be ({tokens}, {heads or 'heads'}, {self.head_dim}) of bf16, f16 or "
                             f"f32, all of one type, on {self.device}, got {tuple(got)} of {t.dtype} on {t.device}")
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} requires a gradient; the rotation has none: detach it or use "
                             "torch.no_grad()")
        return t if t.stride(2) == 1 else t.contiguous()

    def _taken(self, q, k, positions, q_weight, k_weight, eps):
        """Checks the arguments; the descriptor of the rows, and q and k as read."""
        tokens, dtype = q.shape[0], q.dtype
        q = self._rows("q", q, tokens, dtype)
        k = self._rows("k", k, tokens, dtype)
        self._ints("positions", positions, torch.int32, (tokens,))
        kind, at = dtype, [None, None]
        for i, w in enumerate((q_weight, k_weight)):
            if w is None:
                continue
            if (w.shape != (self.head_dim,) or not w.is_contiguous() or w.get_device() != self._index
                    or (w.dtype is not dtype and w.dtype is not torch.float32)
                    or (at[0] is not None and w.dtype is not kind) or w.data_ptr() % 16):
                raise ValueError(f"weights must be {self.head_dim} dense values on {self.device}, both of "
                                 f"{dtype} or both of torch.float32, aligned to 16 bytes; got {w.dtype} "
                                 f"{tuple(w.shape)} on {w.device}")
            if w.requires_grad and torch.is_grad_enabled():
                raise ValueError("the weights require a gradient; the rotation has none: detach them or use "
                                 "torch.no_grad()")
            kind, at[i] = w.dtype, w.data_ptr()
        if not eps >= 0:
            raise ValueError(f"eps {eps}: not negative")
        rows = RowsDesc(q.data_ptr(), k.data_ptr(), q.stride(0), q.stride(1), k.stride(0), k.stride(1),
                        q.shape[1], k.shape[1], at[0], at[1], _DTYPES[dtype], _DTYPES[kind], eps,
                        positions.data_ptr(), tokens)
        return rows, q, k

    def rotate(self, q, k, positions, q_weight=None, k_weight=None, eps=1e-6):
        """The queries (tokens, heads, head_dim) and keys (tokens, kv heads, head_dim; bf16,
        f16 or f32, any strides) of tokens at positions (int32), rotated, as new tensors.
        Where a weight (head_dim) is given, a head is first x * weight / sqrt(mean(x^2) +
        eps).  Computed in f32, angles in 64 bits, rounded once."""
        stream = self._stream()
        rows, q, k = self._taken(q, k, positions, q_weight, k_weight, eps)
        q_out = torch.empty(q.shape, dtype=q.dtype, device=self.device)
        k_out = torch.empty(k.shape, dtype=k.dtype, device=self.device)
        rc = self.lib.vramc_rotary_apply(self._ref, ctypes.byref(rows), q_out.data_ptr(), k_out.data_ptr(),
                                         stream)
        if rc:
            kv_cache._failed("rotate", rc)
        return q_out, k_out

    def append(self, cache, q, k, v, slots, positions, q_weight=None, k_weight=None, eps=1e-6):
        """rotate, with the keys and the values v (as k, any strides) written into slots
        (int64) of a cache, as PagedCache.append writes them; a tracked one takes the
        positions too.  Returns the queries, also of tokens without a slot (-1)."""
        _check(cache.head_dim == self.head_dim and cache.dtype is q.dtype and cache._index == self._index,
               f"a cache of {cache.dtype} heads of {cache.head_dim} on {cache.device} takes no {q.dtype} of "
               f"{self.head_dim} on {self.device}")
        stream = cache._stream()
        rows, q, k = self._taken(q, k, positions, q_weight, k_weight, eps)
        tokens, heads = k.shape[0], cache.kv_heads
        if k.shape[1] != heads:
            raise ValueError(f"keys of {k.shape[1]} heads and a cache of {heads}")
        v = self._rows("v", v, tokens, q.dtype, heads)
        self._ints("slots", slots, torch.int64, (tokens,))
        q_out = torch.empty(q.shape, dtype=q.dtype, device=self.device)
        rc = self.lib.vramc_rotary_append(self._ref, ctypes.byref(rows), cache._ref, v.data_ptr(), v.stride(0),
                                          v.stride(1), slots.data_ptr(), q_out.data_ptr(), stream)
        if rc:
            kv_cache._failed("append", rc)
        return q_out
