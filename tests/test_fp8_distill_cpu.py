"""Contracts of quant_fp8, the fp8 products and distill_ce without a GPU: what each id accepts and refuses, the 8-bit host
codecs, attributes, and the definitions against independent forms. `supported` runs the argument checks on descriptors
alone, so nothing here touches a device."""
import struct

import numpy as np
import pytest

import aicf_cuda
import oracle
from aicf_cuda import f8_bits_to_f32, f32_to_f8_bits, pack_attrs
from aicf_cuda._C import OpKind
from aicf_cuda._C_ctypes import _blob, _build_descs


class D:
    """Descriptor of a tensor that does not exist."""

    def __init__(self, shape, dtype, stride=None, ptr=1 << 20):
        self.shape, self.dtype, self.ptr = tuple(shape), dtype, ptr
        st, acc = [], 1
        for s in reversed(self.shape):
            st.append(acc)
            acc *= s
        self._packed = tuple(reversed(st))
        self._stride = tuple(stride) if stride else self._packed

    def data_ptr(self):
        return self.ptr

    def stride(self):
        return self._stride

    def is_contiguous(self):
        return self._stride == self._packed


def supported(kid, kind, ins, outs, schema=0, payload=b""):
    di, ni = _build_descs(ins, "inputs")
    do, no = _build_descs(outs, "outputs")
    blob, _keep = _blob(schema, payload)
    return bool(aicf_cuda.lib.aicf_b200_supported(kid.encode(), int(kind), di, ni, do, no, blob))


def q8(ins, outs):
    return supported("quant_fp8_block128_v0", OpKind.QuantFp8, ins, outs)


def test_quant_contract():
    x, q = D((300, 200), "bf16"), D((300, 200), "f8e4m3")
    rows, cols, tiles = D((300, 2), "f32"), D((3, 200), "f32"), D((3, 2), "f32")
    for s in (rows, cols, tiles):
        assert q8([x], [q, s])
    assert q8([x], [q, rows, D((300, 200), "f8e5m2"), cols])
    assert q8([D((300, 200), "f32", (208, 1))], [D((300, 200), "f8e4m3", (208, 1)), D((300, 2), "f32", (1, 300))])
    for bad in ([q, D((300, 3), "f32")], [q, D((2, 200), "f32")], [q, D((300, 2), "bf16")], [q], [q, rows, q], [q, rows, q, rows],
                [q, cols, q, rows], [q, tiles, q, tiles], [D((300, 200), "bf16"), rows], [D((300, 199), "f8e4m3"), rows],
                [D((300, 200), "f8e4m3", (199, 1)), rows], [D((300, 200), "f8e4m3", (1, 300)), rows], [q, D((300, 2), "f32", (0, 1))],
                [q, D((300,), "f32")]):
        assert not q8([x], bad), bad
    for bad in (D((300, 200), "i32"), D((300, 200), "f8e4m3"), D((300, 200), "bf16", (1, 300)), D((300, 200), "bf16", (100, 1)), D((0, 200), "bf16"),
                D((300,), "bf16")):
        assert not q8([bad], [q, rows])
    assert not q8([x, x], [q, rows])


def gemm_case(m=130, n=200, k=300, ta=False, tb=True):
    A, B = D((k, m) if ta else (m, k), "f8e4m3"), D((n, k) if tb else (k, n), "f8e5m2")
    sa = D((3, m) if ta else (m, 3), "f32")
    sb = D((2, 3) if tb else (3, 2), "f32")
    return A, B, sa, sb, D((m, n), "bf16")


@pytest.mark.parametrize("ta,tb", [(False, True), (False, False), (True, False), (True, True)])
def test_gemm_contract(ta, tb):
    A, B, sa, sb, C = gemm_case(ta=ta, tb=tb)
    attrs = pack_attrs("gemm", {"transA": ta, "transB": tb})

    def ok(ins, out=C, kid="gemm_fp8_block128_out_bf16_v0"):
        return supported(kid, OpKind.Gemm, ins, [out], *attrs)

    assert ok([A, B, sa, sb])
    assert ok([A, B, D((3, 2) if ta else (2, 3), "f32"), D((200, 3) if tb else (3, 200), "f32")])  # 128 and 1
    assert not ok([A, B]) and not ok([A, B, sa]) and not ok([A, B, sa, sb, sb])
    assert not ok([A, B, sb, sa])
    assert not ok([A, B, D((sa.shape[0] + 1, sa.shape[1]), "f32"), sb])
    assert not ok([A, B, sa, D(sb.shape, "bf16")])
    assert not ok([D(A.shape, "bf16"), B, sa, sb])
    assert not ok([A, B, sa, sb], D((130, 201), "bf16")) and not ok([A, B, sa, sb], D((130, 200), "f32"))
    assert not ok([A, B, sa, sb], D((130, 200), "bf16", (1, 130))) and not ok([A, B, sa, sb], D((130, 200), "bf16", (199, 1)))
    assert ok([A, B, sa, sb], D((130, 200), "bf16", (256, 1)))
    assert ok([A, B, sa, sb], D((130, 200), "f16"), "gemm_fp8_block128_out_f16_v0")
    assert ok([A, B, sa, sb], D((130, 200), "f32"), "gemm_fp8_block128_out_f32_v0")


def test_gemm_epilogue_and_relu_backward_contract():
    A, B, sa, sb, C = gemm_case()
    bias = D((200,), "f32")
    attrs = pack_attrs("gemm_epilogue", {"transB": True, "epilogue": "bias"})
    kid = "gemm_bias_relu_fp8_block128_out_bf16_v0"
    assert supported(kid, OpKind.GemmEpilogue, [A, B, bias, sa, sb], [C], *attrs)
    assert supported(kid, OpKind.GemmEpilogue, [A, B, D((200,), "bf16", (3,)), sa, sb], [C], *attrs)
    for b in (D((199,), "f32"), D((200,), "i32"), D((1, 200), "f32"), D((200,), "f8e4m3")):
        assert not supported(kid, OpKind.GemmEpilogue, [A, B, b, sa, sb], [C], *attrs)
    assert not supported(kid, OpKind.GemmEpilogue, [A, B, bias], [C], *attrs)
    A, B, sa, sb, C = gemm_case(tb=False)
    kid = "gemm_relu_bwd_fp8_block128_out_bf16_v0"
    attrs = pack_attrs("gemm_relu_bwd", {})
    assert supported(kid, OpKind.GemmReluBwd, [A, B, C, sa, sb], [C], *attrs)
    for y in (D((130, 200), "f32"), D((130, 199), "bf16"), D((130, 200), "bf16", (1, 130)), D((130, 200), "bf16", (150, 1))):
        assert not supported(kid, OpKind.GemmReluBwd, [A, B, y, sa, sb], [C], *attrs)


def test_16_bit_products_do_not_take_fp8_operands_and_the_other_way_round():
    A, B, sa, sb, C = gemm_case()
    attrs = pack_attrs("gemm", {"transB": True})
    for kid in ("gemm_bf16_tcgen05_out_bf16_v0", "gemm_f32_naive_v0"):
        assert not supported(kid, OpKind.Gemm, [A, B], [C], *attrs) and not supported(kid, OpKind.Gemm, [A, B, sa, sb], [C], *attrs)
    a, b = D((130, 300), "bf16"), D((200, 300), "bf16")
    assert not supported("gemm_fp8_block128_out_bf16_v0", OpKind.Gemm, [a, b], [C], *attrs)


def dce(ins, outs, attrs=None, kid="distill_ce_f32_v0"):
    return supported(kid, OpKind.DistillCE, ins, outs, *(attrs if isinstance(attrs, tuple) else pack_attrs("distill_ce", attrs)))


def test_distill_contract():
    z, ids, t, y, l = D((8, 100), "f32"), D((8, 5), "i32"), D((8, 5), "f32"), D((8,), "i32"), D((8,), "f32")
    half = {"scale": 1.0, "temperature": 2.0, "alpha": 0.5}
    assert dce([z, ids, t], [z, l]) and dce([z, ids, t], [l]) and dce([z, ids, t, y], [z, l], half)
    assert dce([D((8, 100), "f32", (104, 1)), ids, D((8, 5), "bf16")], [D((8, 100), "f32", (128, 1)), l])
    assert not dce([z, ids, t], [z, l], half), "a label term without labels"
    for bad in ({"scale": 1.0, "temperature": 0.0}, {"scale": 1.0, "temperature": -1.0}, {"scale": 1.0, "temperature": float("nan")},
                {"scale": 1.0, "temperature": float("inf")}, {"scale": 1.0, "temperature": 2.0 ** -61}, {"scale": 1.0, "temperature": 2.0 ** 61}, {"scale": 1.0, "alpha": 1.5}, {"scale": 1.0, "alpha": -0.1}, {"scale": 1.0, "alpha": float("nan")}):
        assert not dce([z, ids, t, y], [z, l], bad), bad
    assert not dce([z, ids, t], [z, l], (0x45434D53, struct.pack("<f", 1.0))), "another op's attributes"
    assert not dce([z, ids, t], [z, l], (0x4C545344, struct.pack("<ff", 1.0, 1.0))), "short payload"
    for ins in ([z, ids], [z, D((8, 5), "f32"), t], [z, D((8, 6), "i32"), t], [z, ids, D((8, 5), "i32")], [z, ids, t, D((7,), "i32")],
                [z, ids, t, D((8,), "f32")], [D((8, 100), "f32", (1, 8)), ids, t], [D((8, 100), "f32", (99, 1)), ids, t],
                [z, D((8, 5), "i32", (6, 1)), t], [z, D((8, 1025), "i32"), D((8, 1025), "f32")], [z, D((7, 5), "i32"), D((7, 5), "f32")],
                [D((8, 100), "bf16"), ids, t], [D((8, 0), "f32"), ids, t], [D((800,), "f32"), ids, t]):
        assert not dce(ins, [z, l], {"scale": 1.0}), [(i.shape, i.dtype) for i in ins]
    for outs in ([z], [z, D((7,), "f32")], [z, D((8,), "bf16")], [D((8, 100), "bf16"), l], [D((8, 101), "f32"), l], [z, l, l]):
        assert not dce([z, ids, t], outs)
    with pytest.raises(ValueError, match="scale"):
        pack_attrs("distill_ce", {"temperature": 2.0})
    assert pack_attrs("distill_ce", half) == (0x4C545344, struct.pack("<fff", 1.0, 2.0, 0.5)) and pack_attrs("distill_ce", {}) == (0, b"")


@pytest.mark.parametrize("fmt", ["f8e4m3", "f8e5m2"])
def test_host_codecs_agree_with_rounding_by_arithmetic(fmt):
    bits = np.arange(256, dtype=np.uint8)
    v = f8_bits_to_f32(bits, fmt)
    fin = np.isfinite(v)
    assert np.array_equal(f32_to_f8_bits(v[fin], fmt), bits[fin])  # -0.0 keeps its sign
    rng = np.random.default_rng(0)
    x = rng.standard_normal(20000) * np.exp(4 * rng.standard_normal(20000))
    mids = (np.sort(v[fin])[1:].astype(np.float64) + np.sort(v[fin])[:-1]) / 2  # every tie
    x = np.concatenate([x, mids, [1e9, -1e9, 0.0]])
    assert np.array_equal(f8_bits_to_f32(f32_to_f8_bits(x, fmt), fmt), oracle.fp8_round(x, fmt))
    assert np.isnan(f8_bits_to_f32(f32_to_f8_bits(np.array([np.nan]), fmt), fmt)).all()


def test_definition_of_the_distillation_gradient_by_differences():
    rng = np.random.default_rng(1)
    z, t = rng.standard_normal((2, 9)), rng.standard_normal((2, 4))
    ids, y = np.array([[1, 3, 3, -1], [0, 8, 2, 5]]), np.array([4, -1])
    d, _ = oracle.distill_ce(z, ids, t, y, 1.0, 1.7, 0.4)
    h, num = 1e-5, np.zeros_like(z)
    for r in range(2):
        for c in range(9):
            e = np.zeros_like(z)
            e[r, c] = h
            num[r, c] = (oracle.distill_ce(z + e, ids, t, y, 1.0, 1.7, 0.4)[1] - oracle.distill_ce(z - e, ids, t, y, 1.0, 1.7, 0.4)[1])[r] / (2 * h)
    assert np.abs(num - d).max() < 1e-8


def test_new_ops_are_named_and_registered():
    lib = aicf_cuda.lib
    assert [lib.aicf_b200_op_name(k).decode() for k in (26, 27)] == ["quant_fp8", "distill_ce"]
    import aicf_cuda._C as m
    assert m.kernel_ids(OpKind.QuantFp8) == ["quant_fp8_block128_v0"]
    assert m.kernel_ids(OpKind.DistillCE) == ["distill_ce_f32_v0", "distill_ce_bf16_v0", "distill_ce_f16_v0"]
