"""Products of block-scaled 8-bit matrices against their 64-bit definition, element by element."""
import numpy as np
import pytest

import oracle
from aicf_cuda import _C, pack_attrs
from fp8_util import EPS_HALF, OpKind, Tensor, blocks, call, gemm_bound, scale_shape, strided

pytestmark = pytest.mark.gpu


def operands(m, n, k, ta, tb, per_a, per_b, fa, fb, seed, pitch16=True):
    """Stored operands and their scales: values over the whole format, scales over three decades."""
    rng = np.random.default_rng(seed)
    sha, shb = ((k, m) if ta else (m, k)), ((n, k) if tb else (k, n))
    A = oracle.fp8_round(rng.standard_normal(sha) * 100.0, fa)
    B = oracle.fp8_round(rng.standard_normal(shb) * 100.0, fb)
    SA = np.exp(rng.standard_normal(scale_shape(sha, ta, per_a))).astype(np.float32) * np.float32(1e-3)
    SB = np.exp(rng.standard_normal(scale_shape(shb, not tb, per_b))).astype(np.float32) * np.float32(1e-3)
    pa, pb = ((x + 15) // 16 * 16 if pitch16 else x for x in (sha[1], shb[1]))
    dev = (strided(A, fa, (pa, 1), fill=0x7F), strided(B, fb, (pb, 1), fill=0x7F), Tensor.from_numpy(SA), Tensor.from_numpy(SB))
    dA, dB = oracle.dequant_fp8(A, SA), oracle.dequant_fp8(B, SB)
    return dev, (dA.T if ta else dA), (dB.T if tb else dB)


def check(got, want, bound):
    assert not np.isnan(got).any()
    off = np.abs(got - want) - bound
    assert off.max() <= 0, f"{int((off > 0).sum())} of {off.size} elements off; worst {np.abs(got - want).max():.3e}"


SIZES = [(1, 1, 1), (1, 256, 512), (3, 130, 100), (64, 256, 784), (127, 129, 127), (128, 128, 128), (129, 300, 129),
         (200, 1000, 333), (256, 512, 1024), (300, 272, 2200), (513, 777, 260)]


@pytest.mark.parametrize("ta,tb", [(False, True), (False, False), (True, False), (True, True)])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_all_transposes_and_scale_shapes(gpu, m, n, k, ta, tb):
    for per_a, per_b in ((1, 128), (1, 1), (128, 128), (128, 1)):
        (A, B, SA, SB), dA, dB = operands(m, n, k, ta, tb, per_a, per_b, "f8e4m3", "f8e4m3", seed=m + n + k)
        C = strided((m, n), "f32", slack=5)
        call(OpKind.Gemm, [A, B, SA, SB], [C], *pack_attrs("gemm", {"transA": ta, "transB": tb}))
        want = dA @ dB
        check(C.float_numpy(), want, gemm_bound(dA, dB, k, want, "f32"))
        assert C.rest_is(0xA5)
    assert _C.gemm_status() == 0


@pytest.mark.parametrize("fa,fb", [("f8e4m3", "f8e5m2"), ("f8e5m2", "f8e4m3"), ("f8e5m2", "f8e5m2")])
@pytest.mark.parametrize("out", ["f32", "bf16", "f16"])
def test_formats_and_output_types(gpu, fa, fb, out):
    m, n, k = 150, 260, 400
    (A, B, SA, SB), dA, dB = operands(m, n, k, False, True, 1, 128, fa, fb, seed=3)
    C = Tensor.empty((m, n), out)
    call(OpKind.Gemm, [A, B, SA, SB], [C], *pack_attrs("gemm", {"transB": True}))
    want = dA @ dB
    check(C.float_numpy(), want, gemm_bound(dA, dB, k, want, out))


@pytest.mark.parametrize("bias", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("relu", [True, False])
@pytest.mark.parametrize("m,n,k", [(1, 1000, 640), (140, 257, 300), (300, 512, 256)])
def test_bias_and_relu(gpu, m, n, k, relu, bias):
    (A, B, SA, SB), dA, dB = operands(m, n, k, False, True, 1, 128, "f8e4m3", "f8e4m3", seed=4)
    b = Tensor.from_numpy(np.random.default_rng(1).standard_normal(n).astype(np.float32) * 30, bias)
    C = Tensor.empty((m, n), "bf16")
    call(OpKind.GemmEpilogue, [A, B, b, SA, SB], [C], *pack_attrs("gemm_epilogue", {"transB": True, "epilogue": "bias_relu" if relu else "bias"}))
    want = dA @ dB + b.float_numpy().astype(np.float64)
    bound = gemm_bound(dA, dB, k, want, "bf16") + np.abs(want) * 2.0 ** -24 * 2
    check(C.float_numpy(), np.maximum(want, 0) if relu else want, bound)


@pytest.mark.parametrize("out", ["bf16", "f32", "f16"])
@pytest.mark.parametrize("m,n,k", [(1, 130, 200), (140, 257, 300), (260, 512, 1000)])
def test_relu_backward_mask(gpu, m, n, k, out):
    (A, B, SA, SB), dA, dB = operands(m, n, k, False, False, 1, 128, "f8e5m2", "f8e4m3", seed=5)
    rng = np.random.default_rng(2)
    y = np.maximum(rng.standard_normal((m, n)), 0).astype(np.float32)
    y[0, 0], y[-1, -1] = np.nan, -0.0  # neither is > 0
    Y = strided(y, out, (n + 8, 1))
    C = strided((m, n), out, (n + 3, 1))
    call(OpKind.GemmReluBwd, [A, B, Y, SA, SB], [C], *pack_attrs("gemm_relu_bwd", {}))
    want = np.where(y > 0, dA @ dB, 0.0)
    check(C.float_numpy(), want, gemm_bound(dA, dB, k, want, out))
    assert C.rest_is(0xA5)


@pytest.mark.parametrize("ta,tb", [(False, True), (True, False)])
def test_packed_odd_rows_and_k_block_major_scales(gpu, ta, tb):
    """Operands whose rows do not start on 16 bytes, and scales stored the other way round."""
    m, n, k = 133, 201, 301
    (A, B, SA, SB), dA, dB = operands(m, n, k, ta, tb, 1, 1, "f8e4m3", "f8e4m3", seed=6, pitch16=False)
    sa, sb = SA.numpy(), SB.numpy()
    SAt, SBt = strided(sa, "f32", (1, sa.shape[0])), strided(sb, "f32", (1, sb.shape[0]))
    C = Tensor.empty((m, n))
    call(OpKind.Gemm, [A, B, SAt, SBt], [C], *pack_attrs("gemm", {"transA": ta, "transB": tb}))
    want = dA @ dB
    check(C.float_numpy(), want, gemm_bound(dA, dB, k, want, "f32"))


def test_doubly_strided_operands(gpu):
    """Neither stride is one."""
    m, n, k = 70, 90, 140
    rng = np.random.default_rng(7)
    A, B = (oracle.fp8_round(rng.standard_normal(s) * 50, "f8e4m3") for s in ((m, k), (n, k)))
    SA, SB = np.full((m, 2), 0.5, np.float32), np.full((1, 2), 0.25, np.float32)
    dev = [strided(A, "f8e4m3", (2 * k, 2)), strided(B, "f8e4m3", (3 * k, 3)), Tensor.from_numpy(SA), Tensor.from_numpy(SB)]
    C = Tensor.empty((m, n))
    call(OpKind.Gemm, dev, [C], *pack_attrs("gemm", {"transB": True}))
    dA, dB = oracle.dequant_fp8(A, SA), oracle.dequant_fp8(B, SB).T
    check(C.float_numpy(), dA @ dB, gemm_bound(dA, dB, k, dA @ dB, "f32"))


def test_scales_far_apart_and_zero_blocks(gpu):
    """Scales whose product leaves fp32 meet blocks of zeros (0 stays 0), and blocks 2^60 apart add up."""
    m, n, k = 130, 128, 512
    rng = np.random.default_rng(8)
    A, B = (oracle.fp8_round(rng.standard_normal(s) * 100, "f8e4m3") for s in ((m, k), (n, k)))
    A[:, 128:256] = 0.0
    SA = np.full((m, 4), 2.0 ** -10, np.float32)
    SB = np.full((1, 4), 2.0 ** -10, np.float32)
    SA[:, 1], SB[:, 1] = 1e30, 1e30
    SA[:, 2] = 2.0 ** -70
    SA[:, 3] = 2.0 ** 50
    C = Tensor.empty((m, n))
    call(OpKind.Gemm, [Tensor.from_numpy(A, "f8e4m3"), Tensor.from_numpy(B, "f8e4m3"), Tensor.from_numpy(SA), Tensor.from_numpy(SB)], [C],
         *pack_attrs("gemm", {"transB": True}))
    dA, dB = oracle.dequant_fp8(A, SA), oracle.dequant_fp8(B, SB).T
    check(C.float_numpy(), dA @ dB, gemm_bound(dA, dB, k, dA @ dB, "f32"))


def test_a_nan_scale_spoils_its_own_rows_only(gpu):
    m, n, k = 140, 130, 256
    (A, B, SA, SB), dA, dB = operands(m, n, k, False, True, 1, 128, "f8e4m3", "f8e4m3", seed=9)
    sa = SA.numpy()
    sa[5, 1] = np.nan
    SA.copy_from_host(sa)
    C = Tensor.empty((m, n))
    call(OpKind.Gemm, [A, B, SA, SB], [C], *pack_attrs("gemm", {"transB": True}))
    got = C.float_numpy()
    assert np.isnan(got[5]).all()
    keep = np.arange(m) != 5
    want = (dA @ dB)[keep]
    check(got[keep], want, gemm_bound(dA, dB, k, dA @ dB, "f32")[keep])


def test_two_runs_give_the_same_bits_and_a_replay_too(gpu):
    m, n, k = 3, 1000, 8192
    (A, B, SA, SB), _, _ = operands(m, n, k, False, True, 1, 128, "f8e4m3", "f8e4m3", seed=10)
    outs = [Tensor.empty((m, n)) for _ in range(3)]
    attrs = pack_attrs("gemm", {"transB": True})
    for C in outs[:2]:
        call(OpKind.Gemm, [A, B, SA, SB], [C], *attrs)
    stream = _C.graph_begin()
    _C.op_call(OpKind.Gemm, [A, B, SA, SB], [outs[2]], *attrs, stream)
    _C.graph_end()
    _C.graph_launch()
    _C.device_sync()
    _C.graph_reset()
    assert np.array_equal(outs[0].numpy(), outs[1].numpy()) and np.array_equal(outs[0].numpy(), outs[2].numpy())


def test_quantise_then_multiply_is_close_to_the_unquantised_product(gpu):
    """The operators in a row, as a layer uses them. A normal value is off by at most 2^-4 of itself (e4m3), below the
    normal range by half the smallest step (2^-10) times the block's scale."""
    m, n, k = 130, 260, 384
    rng = np.random.default_rng(11)
    x, w = rng.standard_normal((m, k)).astype(np.float32), rng.standard_normal((n, k)).astype(np.float32)
    X, W = Tensor.from_numpy(x), Tensor.from_numpy(w)
    qx, sx, qw, sw = Tensor.empty((m, k), "f8e4m3"), Tensor.empty((m, blocks(k))), Tensor.empty((n, k), "f8e4m3"), Tensor.empty((blocks(n), blocks(k)))
    call(OpKind.QuantFp8, [X], [qx, sx])
    call(OpKind.QuantFp8, [W], [qw, sw])
    C = Tensor.empty((m, n))
    call(OpKind.Gemm, [qx, qw, sx, sw], [C], *pack_attrs("gemm", {"transB": True}))
    ex = np.abs(x) * 2.0 ** -4 + 2.0 ** -10 * oracle.dequant_fp8(np.ones_like(x), sx.numpy())
    ew = np.abs(w) * 2.0 ** -4 + 2.0 ** -10 * oracle.dequant_fp8(np.ones_like(w), sw.numpy())
    bound = ex @ np.abs(w).T + np.abs(x) @ ew.T + ex @ ew.T
    assert np.all(np.abs(C.float_numpy() - x.astype(np.float64) @ w.T.astype(np.float64)) <= bound * (1 + 1e-4))
    assert EPS_HALF["bf16"] == 2.0 ** -8
