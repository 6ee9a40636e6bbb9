"""quant_fp8 against its definition, bit for bit: every rounding of the definition is an IEEE fp32 one."""
import numpy as np
import pytest

import oracle
from aicf_cuda import _C
from fp8_util import OpKind, Tensor, blocks, call, strided

pytestmark = pytest.mark.gpu

FORMS = {"rows": lambda M, N: (M, blocks(N)), "cols": lambda M, N: (blocks(M), N), "tiles": lambda M, N: (blocks(M), blocks(N))}


def matrix(M, N, seed):
    """Channels of different size, a zero row, a zero column, a block of values far below the rest."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((M, N)) * np.exp(0.7 * rng.standard_normal(N))
    x[M // 2] = 0.0
    x[:, N // 2] = 0.0
    x[: M // 3, : N // 3] *= 1e-6
    return x.astype(np.float32)


def quantise(x, dtype, outs_spec, fmts, pitch=None):
    X = Tensor.from_numpy(x, dtype)
    outs = []
    M, N = x.shape
    for form, fmt in zip(outs_spec, fmts):
        q = strided((M, N), fmt, (pitch or N, 1), slack=7)
        outs += [q, strided(FORMS[form](M, N), "f32", slack=3)]
    call(OpKind.QuantFp8, [X], outs)
    return X.float_numpy(), outs


@pytest.mark.parametrize("fmt", ["f8e4m3", "f8e5m2"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", [(1, 1), (1, 300), (300, 1), (64, 784), (127, 129), (128, 128), (129, 136), (257, 1000), (5, 4099)])
def test_every_form_is_the_definition_bit_for_bit(gpu, shape, dtype, fmt):
    x = matrix(*shape, seed=shape[0] * 7 + shape[1])
    for forms in (["rows"], ["cols"], ["tiles"], ["rows", "cols"]):
        xs, outs = quantise(x, dtype, forms, [fmt] * len(forms))
        for form, q, s in zip(forms, outs[0::2], outs[1::2]):
            wq, ws = oracle.quant_fp8(xs, form, fmt)
            assert np.array_equal(s.float_numpy(), ws), (forms, form)
            assert np.array_equal(q.float_numpy(), wq), (forms, form)
            assert q.rest_is(0xA5) and s.rest_is(0xA5), "wrote outside its outputs"


@pytest.mark.parametrize("pitch", [1000, 1008, 1013])
def test_pitched_outputs_and_two_formats_in_one_call(gpu, pitch):
    x = matrix(130, 1000, seed=5)
    xs, outs = quantise(x, "bf16", ["rows", "cols"], ["f8e4m3", "f8e5m2"], pitch=pitch)
    for form, fmt, q, s in (("rows", "f8e4m3", *outs[:2]), ("cols", "f8e5m2", *outs[2:])):
        wq, ws = oracle.quant_fp8(xs, form, fmt)
        assert np.array_equal(s.float_numpy(), ws) and np.array_equal(q.float_numpy(), wq)
        assert q.rest_is(0xA5)


def test_pitched_unaligned_input_and_strided_scales(gpu):
    x = matrix(200, 333, seed=6)
    X = strided(x, "bf16", (337, 1), offset=3)
    q, s = strided((200, 333), "f8e4m3", (336, 1)), strided((200, 3), "f32", (1, 205))  # scale stored k-block major
    call(OpKind.QuantFp8, [X], [q, s])
    wq, ws = oracle.quant_fp8(X.float_numpy(), "rows", "f8e4m3")
    assert np.array_equal(q.float_numpy(), wq) and np.array_equal(s.float_numpy(), ws) and s.rest_is(0xA5)


def test_extreme_values(gpu):
    """Largest, smallest and subnormal magnitudes; a NaN or an infinity spoils its own block and no other."""
    x = np.zeros((4, 512), np.float32)
    x[0, :128], x[0, 128:256], x[0, 256:384] = 3.0e38, 1e-45, np.float32(2.0 ** -110)
    x[0, 384:] = np.linspace(-1, 1, 128)
    x[1, :128] = np.linspace(0, 448, 128)
    x[2, 5], x[2, 200] = np.nan, np.inf
    x[2, 130] = 2.0
    x[3] = 1.0
    xs, (q, s) = quantise(x, "f32", ["rows"], ["f8e4m3"])
    good = np.ones((4, 4), bool)
    good[2, :2] = False
    wq, ws = oracle.quant_fp8(xs, "rows", "f8e4m3")
    gq, gs = q.float_numpy(), s.float_numpy()
    assert np.array_equal(gs[good], ws[good])
    keep = np.repeat(good, 128, axis=1)
    assert np.array_equal(gq[keep], wq[keep])
    assert np.isnan(gs[2, 0]) and np.isinf(gs[2, 1]) and np.isnan(gq[2, 200])


def test_captured_and_replayed(gpu):
    x = matrix(64, 256, seed=8)
    X = Tensor.from_numpy(x, "f32")
    q, s = Tensor.zeros((64, 256), "f8e4m3"), Tensor.zeros((64, 2))
    stream = _C.graph_begin()
    _C.op_call(OpKind.QuantFp8, [X], [q, s], stream=stream)
    _C.graph_end()
    X.copy_from_host(2 * x)
    _C.graph_launch()
    _C.device_sync()
    _C.graph_reset()
    wq, ws = oracle.quant_fp8(2 * x, "rows", "f8e4m3")
    assert np.array_equal(q.float_numpy(), wq) and np.array_equal(s.float_numpy(), ws)


@pytest.mark.parametrize("fmt", ["f8e4m3", "f8e5m2"])
@pytest.mark.parametrize("power", [-100, -60, 0, 60, 127])
def test_quotients_next_to_a_tie_round_to_the_right_side(gpu, fmt, power):
    """Values within half an fp32 step of the midpoint between two values of the format: the fp32 quotient often is the
    midpoint itself, and only the exact one tells the side."""
    rng = np.random.default_rng(power + 200)
    M, N = 256, 1024
    amax = (np.float64(2.0) ** power * rng.uniform(1.0, 1.99, (M, N // 128))).astype(np.float32).astype(np.float64)
    bits = 3 if fmt == "f8e4m3" else 2
    top = 8 if fmt == "f8e4m3" else 15
    mid = (2 ** bits + rng.integers(0, 2 ** bits, (M, N)) + 0.5) * 2.0 ** (rng.integers(-6, top, (M, N)) - bits)
    x = (mid * np.repeat(amax, 128, axis=1) / (448.0 if fmt == "f8e4m3" else 57344.0)).astype(np.float32)
    x *= rng.choice(np.float32([-1, 1]), (M, N))
    x[:, ::128] = amax
    for form in ("rows", "cols", "tiles"):
        xs, (q, s) = quantise(x, "f32", [form], [fmt])
        wq, ws = oracle.quant_fp8(xs, form, fmt)
        assert np.array_equal(s.float_numpy(), ws) and np.array_equal(q.float_numpy(), wq), form
