"""Device tensors without a tensor library: a pointer-stable buffer plus shape/dtype.

The reference hands torch.Tensor objects to its binding; callers of this backend may do the same
(anything with data_ptr()/shape/stride()/dtype works), or use this class, which needs only NumPy.
bf16 has no NumPy dtype: host arrays carry it as uint16 bit patterns. The 8-bit floats ('f8e4m3', 'f8e5m2': the values
of a block-scaled matrix) are carried as uint8 bit patterns.
"""
from __future__ import annotations

import ctypes as C
from typing import Sequence

import numpy as np

from ._lib import check, lib

DTYPE_CODES = {"f32": 1, "f16": 2, "bf16": 3, "i32": 4, "f8e4m3": 5, "f8e5m2": 6}
DTYPE_SIZES = {"f32": 4, "f16": 2, "bf16": 2, "i32": 4, "f8e4m3": 1, "f8e5m2": 1}
_NP_OF = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16, "i32": np.int32, "f8e4m3": np.uint8, "f8e5m2": np.uint8}


def f32_to_bf16_bits(x: np.ndarray) -> np.ndarray:
    """Round-to-nearest-even fp32 -> bf16, returned as uint16 bit patterns (NaN stays NaN)."""
    u = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32)
    rounded = (u + np.uint32(0x7FFF) + ((u >> np.uint32(16)) & np.uint32(1))) >> np.uint32(16)
    nan = (u & np.uint32(0x7FFFFFFF)) > np.uint32(0x7F800000)
    return np.where(nan, (u >> np.uint32(16)) | np.uint32(0x40), rounded).astype(np.uint16)


def bf16_bits_to_f32(b: np.ndarray) -> np.ndarray:
    return (np.ascontiguousarray(b, dtype=np.uint16).astype(np.uint32) << np.uint32(16)).view(np.float32)


def _f8_values(dtype: str) -> np.ndarray:
    """float32 value of each of the 256 bit patterns of 'f8e4m3' (bias 7, no infinity) or 'f8e5m2' (bias 15, IEEE-like)."""
    mant, bias = {"f8e4m3": (3, 7), "f8e5m2": (2, 15)}[dtype]
    b = np.arange(256)
    m, e = b & ((1 << mant) - 1), (b & 0x7F) >> mant
    v = np.where(e == 0, np.ldexp(m.astype(np.float64), 1 - bias - mant),
                 np.ldexp(1.0 + m / float(1 << mant), e - bias))
    if dtype == "f8e4m3":
        v[(b & 0x7F) == 0x7F] = np.nan
    else:
        v[(b & 0x7F) == 0x7C] = np.inf
        v[(b & 0x7F) > 0x7C] = np.nan
    return np.where(b & 0x80, -v, v).astype(np.float32)


_F8_TABLES = {d: _f8_values(d) for d in ("f8e4m3", "f8e5m2")}


def f8_bits_to_f32(b: np.ndarray, dtype: str) -> np.ndarray:
    return _F8_TABLES[dtype][np.ascontiguousarray(b, dtype=np.uint8)]


def f32_to_f8_bits(x: np.ndarray, dtype: str) -> np.ndarray:
    """Round to nearest even, saturating at the largest finite value (NaN stays NaN), as uint8 bit patterns."""
    x = np.asarray(x, np.float64)
    top = 448.0 if dtype == "f8e4m3" else 57344.0
    grid = _F8_TABLES[dtype][:128].astype(np.float64)
    grid = grid[np.isfinite(grid)]  # ascending; the index is the bit pattern of the magnitude
    mag = np.minimum(np.abs(np.where(np.isnan(x), 0.0, x)), top)
    hi = np.clip(np.searchsorted(grid, mag, side="left"), 0, len(grid) - 1)
    lo = np.maximum(hi - 1, 0)
    dl, dh = mag - grid[lo], grid[hi] - mag
    pick_lo = (dl < dh) | ((dl == dh) & (lo % 2 == 0))
    bits = np.where(pick_lo, lo, hi) | np.where(np.signbit(x), 0x80, 0)
    return np.where(np.isnan(x), 0x7F, bits).astype(np.uint8)


class Tensor:
    """Contiguous device buffer. Owns its memory unless built with `ptr=`."""

    def __init__(self, shape: Sequence[int], dtype: str, ptr: int | None = None):
        if dtype not in DTYPE_CODES:
            raise ValueError(f"unsupported dtype {dtype!r}")
        self.shape = tuple(int(s) for s in shape)
        if len(self.shape) > 4:
            raise ValueError("rank must be <= 4")
        self.dtype = dtype
        self.numel = int(np.prod(self.shape, dtype=np.int64)) if self.shape else 1
        self.nbytes = self.numel * DTYPE_SIZES[dtype]
        self._owned = ptr is None
        if ptr is None:
            p = C.c_void_p()
            check(lib.aicf_b200_malloc(C.byref(p), max(self.nbytes, 1)), "malloc")
            ptr = p.value
        self.ptr = int(ptr)

    # --- duck-typing surface shared with torch.Tensor -------------------------------------------
    def data_ptr(self) -> int:
        return self.ptr

    def stride(self) -> tuple[int, ...]:
        st, acc = [], 1
        for s in reversed(self.shape):
            st.append(acc)
            acc *= s
        return tuple(reversed(st))

    def is_contiguous(self) -> bool:
        return True

    def dim(self) -> int:
        return len(self.shape)

    # --- construction / transfer -----------------------------------------------------------------
    @classmethod
    def empty(cls, shape, dtype="f32") -> "Tensor":
        return cls(shape, dtype)

    @classmethod
    def zeros(cls, shape, dtype="f32") -> "Tensor":
        t = cls(shape, dtype)
        t.zero_()
        return t

    @classmethod
    def from_numpy(cls, arr: np.ndarray, dtype: str | None = None) -> "Tensor":
        """dtype=None infers f32/f16/i32 from the array; dtype='bf16' accepts float32 (rounded to
        nearest even) or uint16 bit patterns, the 8-bit floats accept float32 (rounded, saturating) or uint8 bit patterns."""
        arr = np.asarray(arr)
        if dtype is None:
            dtype = {np.dtype(np.float32): "f32", np.dtype(np.float16): "f16", np.dtype(np.int32): "i32"}.get(arr.dtype)
            if dtype is None:
                raise ValueError(f"cannot infer device dtype from {arr.dtype}")
        if dtype == "bf16":
            host = arr.astype(np.uint16) if arr.dtype == np.uint16 else f32_to_bf16_bits(arr.astype(np.float32))
        elif dtype in _F8_TABLES:
            host = arr if arr.dtype == np.uint8 else f32_to_f8_bits(arr, dtype)
        else:
            host = arr.astype(_NP_OF[dtype])
        host = np.ascontiguousarray(host)
        t = cls(arr.shape, dtype)
        t.copy_from_host(host)
        return t

    def copy_from_host(self, host: np.ndarray, stream: int = 0) -> None:
        host = np.ascontiguousarray(host)
        if host.nbytes != self.nbytes:
            raise ValueError(f"size mismatch: host {host.nbytes} B vs device {self.nbytes} B")
        check(lib.aicf_b200_memcpy_h2d(self.ptr, host.ctypes.data, self.nbytes, stream), "memcpy_h2d")
        check(lib.aicf_b200_stream_sync(stream), "stream_sync")

    def numpy(self, stream: int = 0) -> np.ndarray:
        """Device -> host copy. bf16 comes back as uint16 bit patterns (see bf16_bits_to_f32), the 8-bit floats as uint8."""
        out = np.empty(self.shape, dtype=_NP_OF[self.dtype])
        if self.nbytes:
            check(lib.aicf_b200_memcpy_d2h(out.ctypes.data, self.ptr, self.nbytes, stream), "memcpy_d2h")
            check(lib.aicf_b200_stream_sync(stream), "stream_sync")
        return out

    def float_numpy(self) -> np.ndarray:
        """Host copy widened to float32 (int32 tensors are returned unchanged)."""
        a = self.numpy()
        if self.dtype == "bf16":
            return bf16_bits_to_f32(a).reshape(self.shape)
        if self.dtype in _F8_TABLES:
            return f8_bits_to_f32(a, self.dtype)
        return a.astype(np.float32) if self.dtype == "f16" else a

    def zero_(self) -> "Tensor":
        check(lib.aicf_b200_memset(self.ptr, 0, self.nbytes, 0), "memset")
        check(lib.aicf_b200_stream_sync(0), "stream_sync")
        return self

    def view(self, shape) -> "Tensor":
        v = Tensor(shape, self.dtype, ptr=self.ptr)
        if v.nbytes != self.nbytes:
            raise ValueError("view changes the number of bytes")
        v._base = self  # keep the owner alive
        return v

    def __del__(self):
        if getattr(self, "_owned", False) and getattr(self, "ptr", 0):
            try:
                lib.aicf_b200_free(self.ptr)
            except Exception:
                pass
            self.ptr = 0

    def __repr__(self) -> str:
        return f"aicf_cuda.Tensor(shape={self.shape}, dtype={self.dtype}, ptr=0x{self.ptr:x})"
