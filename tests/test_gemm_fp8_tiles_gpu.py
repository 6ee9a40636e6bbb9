"""8-bit products with every tile shape and K split forced in turn: several tiles per CTA, several groups of scales, ragged
edges, and the operators of a layer one after the other on a stream of their own."""
import functools

import numpy as np
import pytest

import oracle
from aicf_cuda import _C, pack_attrs
from aicf_cuda._lib import lib
from fp8_util import OpKind, Tensor, blocks, gemm_bound, call
from test_gemm_fp8_gpu import check, operands

pytestmark = pytest.mark.gpu

M, N, K = 2600, 2111, 1100  # nine blocks of K: two groups of scales; more tiles than SMs or pairs at every tile shape


@functools.lru_cache(maxsize=2)
def case(form):
    ta, tb, per_b = {"fwd": (False, True, 128), "dw": (True, False, 1)}[form]
    dev, dA, dB = operands(M, N, K, ta, tb, 1, per_b, "f8e4m3", "f8e5m2", seed=31)
    want = dA @ dB
    return dev, (ta, tb), want, gemm_bound(dA, dB, K, want, "bf16")


@pytest.mark.parametrize("tile", ["2256", "1256", "1128", "164"])
@pytest.mark.parametrize("form", ["fwd", "dw"])
def test_many_tiles_of_each_shape(gpu, form, tile, monkeypatch):
    monkeypatch.setenv("AICF_FP8_TILE", tile)
    (A, B, SA, SB), (ta, tb), want, bound = case(form)
    y = np.maximum(np.random.default_rng(3).standard_normal((M, N)), 0).astype(np.float32)
    Y, C, D = Tensor.from_numpy(y, "bf16"), Tensor.empty((M, N), "bf16"), Tensor.empty((M, N), "bf16")
    attrs = pack_attrs("gemm", {"transA": ta, "transB": tb})
    call(OpKind.Gemm, [A, B, SA, SB], [C], *attrs)
    check(C.float_numpy(), want, bound)
    call(OpKind.GemmReluBwd, [A, B, Y, SA, SB], [D], *attrs)
    check(D.float_numpy(), np.where(y > 0, want, 0.0), bound)
    assert _C.gemm_status() == 0


@pytest.mark.parametrize("splits", ["2", "4", "8"])
@pytest.mark.parametrize("tile", ["1128", "164"])
def test_splits_of_k(gpu, tile, splits, monkeypatch):
    monkeypatch.setenv("AICF_FP8_TILE", tile)
    monkeypatch.setenv("AICF_FP8_SPLITK", splits)
    m, n, k = 67, 203, 2900
    (A, B, SA, SB), dA, dB = operands(m, n, k, False, True, 1, 128, "f8e4m3", "f8e4m3", seed=9)
    bias, C = np.random.default_rng(1).standard_normal(n).astype(np.float32), Tensor.empty((m, n))
    call(OpKind.GemmEpilogue, [A, B, Tensor.from_numpy(bias), SA, SB], [C], *pack_attrs("gemm_epilogue", {"transB": True, "relu": True}))
    want = dA @ dB + bias
    bound = gemm_bound(dA, dB, k, want, "f32") + (np.abs(bias) + 8 * np.abs(want)) * 2.0 ** -24  # the bias, up to eight parts
    check(C.numpy(), np.maximum(want, 0), bound)
    assert _C.gemm_status() == 0


def test_a_layer_on_a_stream_of_its_own(gpu):
    """Quantise both operands, multiply (unaligned rows: with the copies in the workspace), distil, all on one stream."""
    import ctypes
    rng = np.random.default_rng(17)
    b, n, k, top = 130, 301, 205, 7
    x, w = rng.standard_normal((b, k)).astype(np.float32), rng.standard_normal((n, k)).astype(np.float32)
    ids = np.argsort(rng.random((b, n)), axis=1)[:, :top].astype(np.int32)
    t = rng.standard_normal((b, top)).astype(np.float32)
    X, W, I, T = (Tensor.from_numpy(a) for a in (x, w, ids, t))
    QX, SX, QW, SW = Tensor.empty((b, k), "f8e4m3"), Tensor.empty((b, blocks(k))), Tensor.empty((n, k), "f8e4m3"), Tensor.empty((blocks(n), blocks(k)))
    Z, L = Tensor.empty((b, n)), Tensor.empty((b,))
    _C.device_sync()
    stream = ctypes.c_uint64()
    assert lib.aicf_b200_stream_create(ctypes.byref(stream)) == 0
    s = stream.value
    _C.op_call(OpKind.QuantFp8, [X], [QX, SX], 0, b"", s)
    _C.op_call(OpKind.QuantFp8, [W], [QW, SW], 0, b"", s)
    _C.op_call(OpKind.Gemm, [QX, QW, SX, SW], [Z], *pack_attrs("gemm", {"transB": True}), s)
    _C.op_call(OpKind.DistillCE, [Z, I, T], [Z, L], *pack_attrs("distill_ce", {"scale": 1.0, "temperature": 2.0}), s)
    _C.device_sync()
    assert lib.aicf_b200_stream_destroy(stream) == 0
    (qx, sx), (qw, sw) = oracle.quant_fp8(x, "rows", "f8e4m3"), oracle.quant_fp8(w, "tiles", "f8e4m3")
    z = oracle.gemm_fp8(qx, qw, sx, sw, False, True)
    err = gemm_bound(oracle.dequant_fp8(qx, sx), oracle.dequant_fp8(qw, sw).T, k, z, "f32").max()
    wd, wl = oracle.distill_ce(z, ids, t, None, 1.0, 2.0)
    # a logit off by err moves q by err / T of itself at most twice over (its own exponential, the sum), the loss by T * 2 err
    assert np.abs(Z.numpy() - wd).max() <= 2 * 2.0 * err + 256 * 2.0 ** -23
    assert np.abs(L.numpy() - wl).max() <= 2 * 2.0 * err + 4 * 32 * 256 * 2.0 ** -23
    assert _C.gemm_status() == 0 and _C.wait_status() == 0
