"""Helpers of the block-scaled 8-bit and distillation tests: strided operands, calls, and error bounds."""
import numpy as np

from aicf_cuda import _C, Tensor
from aicf_cuda._C import OpKind

EPS_HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # half a step, relative to the value
TOP = {"f8e4m3": 448.0, "f8e5m2": 57344.0}


class Strided:
    """A 2-D view with strides of its own into a device buffer filled with a known pattern."""

    def __init__(self, base: Tensor, shape, stride, offset=0):
        self.base, self.shape, self._stride, self.dtype = base, tuple(shape), tuple(stride), base.dtype
        self.offset = offset

    def data_ptr(self):
        from aicf_cuda.tensor import DTYPE_SIZES
        return self.base.data_ptr() + self.offset * DTYPE_SIZES[self.dtype]

    def stride(self):
        return self._stride

    def is_contiguous(self):
        return self._stride == (self.shape[1], 1)

    def _index(self):
        r, c = np.arange(self.shape[0])[:, None], np.arange(self.shape[1])[None, :]
        return self.offset + r * self._stride[0] + c * self._stride[1]

    def numpy(self):
        return self.base.numpy().reshape(-1)[self._index()]

    def float_numpy(self):
        return self.base.float_numpy().reshape(-1)[self._index()]

    def rest_is(self, pattern):
        """True when no byte outside the view has changed from the fill."""
        a = self.base.numpy().reshape(-1)
        keep = np.ones(a.size, bool)
        keep[self._index()] = False
        return bool(np.all(a.view(np.uint8).reshape(a.size, -1)[keep] == pattern))


def strided(arr, dtype, stride=None, offset=0, slack=0, fill=0xA5):
    """`arr` on the device under `stride` (elements), the gaps filled with a byte pattern. arr None + shape via tuple."""
    shape = arr if isinstance(arr, tuple) else np.shape(arr)
    stride = stride or (shape[1], 1)
    n = offset + (shape[0] - 1) * stride[0] + (shape[1] - 1) * stride[1] + 1 + slack
    t = Tensor((n,), dtype)
    host = np.full(t.nbytes, fill, np.uint8)
    if not isinstance(arr, tuple):
        packed = Tensor.from_numpy(np.ascontiguousarray(arr), dtype).numpy()
        flat = host.view(packed.dtype)
        idx = offset + np.arange(shape[0])[:, None] * stride[0] + np.arange(shape[1])[None, :] * stride[1]
        flat[idx] = packed
    t.copy_from_host(host)
    return Strided(t, shape, stride, offset)


def blocks(n):
    return -(-n // 128)


def call(kind, ins, outs, schema=0, payload=b"", stream=0):
    _C.op_call(kind, ins, outs, schema, payload, stream)
    _C.device_sync()


def scale_shape(stored, trans_k_first, per):
    """Shape of a scale matrix for a stored operand: the summed extent divided by 128, the other one by `per`."""
    k = 0 if trans_k_first else 1
    s = list(stored)
    s[k] = blocks(s[k])
    s[1 - k] = s[1 - k] if per == 1 else blocks(s[1 - k])
    return tuple(s)


def gemm_bound(A, B, K, want, out):
    """|error| allowed for C = A @ B (fp64 dequantised operands) accumulated in fp32 by blocks of 128 of K. With S the sum of
    the |products|: inside a block at most 128 additions, each off by at most 2^-23 of S (a tensor core may truncate: a
    whole step); one rounding for the scale product, one for the scaling; one per block added (2^-24 S each); the scale
    matrix product itself 2^-24. An ordinary fp32 chain is inside the same bound. Then half a step of the output type."""
    S = np.abs(A) @ np.abs(B)
    inner = min(K, 128) * 2.0 ** -23 + (blocks(K) + 4) * 2.0 ** -24
    tiny = 2.0 ** -24 if out == "f16" else 1e-37
    return S * inner * (1 + 2.0 ** -7) + np.abs(want) * EPS_HALF[out] + tiny


__all__ = ["Strided", "strided", "blocks", "call", "scale_shape", "gemm_bound", "EPS_HALF", "TOP", "OpKind", "Tensor", "np"]
