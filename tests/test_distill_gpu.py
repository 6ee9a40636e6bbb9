"""distill_ce against its 64-bit definition and against differences of its own loss."""
import numpy as np
import pytest

import oracle
from aicf_cuda import _C, pack_attrs
from fp8_util import EPS_HALF, OpKind, Tensor, call, strided

pytestmark = pytest.mark.gpu


def batch(B, C, K, dtype, seed, spread=2.0):
    rng = np.random.default_rng(seed)
    z = (spread * rng.standard_normal((B, C))).astype(np.float32)
    z = Tensor.from_numpy(z, dtype).float_numpy()  # what the device holds
    ids = np.argsort(rng.random((B, C)), axis=1)[:, :K].astype(np.int32)
    t = (np.take_along_axis(z, ids, 1) + rng.standard_normal((B, K)) + 3).astype(np.float32)
    y = rng.integers(0, C, B, dtype=np.int32)
    return z, ids, t, y


def run(z, ids, t, y, dtype, scale, T, alpha, t_dtype="f32", grad=True, ld=None, ld_out=None, offset=0):
    Z = strided(z, dtype, (ld or z.shape[1], 1), offset=offset)
    D = strided(z.shape, dtype, (ld_out or ld or z.shape[1], 1), offset=offset, slack=9)
    L = Tensor.empty((z.shape[0],))
    ins = [Z, Tensor.from_numpy(ids), Tensor.from_numpy(t, t_dtype)] + ([Tensor.from_numpy(y)] if y is not None else [])
    call(OpKind.DistillCE, ins, [D, L] if grad else [L], *pack_attrs("distill_ce", {"scale": scale, "temperature": T, "alpha": alpha}))
    if grad:
        assert D.rest_is(0xA5), "wrote outside its rows"
    return D.float_numpy() if grad else None, L.numpy()


def assert_matches(got_d, got_l, z, ids, t, y, dtype, scale, T, alpha):
    """Exponentials and sums in fp32: an exponential of x is off by (|x| + 4) 2^-23 (its argument's rounding, its own and
    the scaling by 1/T), a sum of C positive terms by at most the same plus 64 2^-23 (thread, warp and block partial sums
    of at most about 64 levels), so p, q and their products by (R + 80) 2^-23 with R the row's range over T; the gradient
    additionally by half a step of its type, the loss by that much of the terms it is made of."""
    wd, wl = oracle.distill_ce(z, ids, t, y, scale, T, alpha)
    R = (z.max(1) - z.min(1)) * max(1.0, 1.0 / T)
    rel = ((R + 100) * 2.0 ** -23)[:, None]
    # the terms the gradient is the difference of
    q = np.exp(z / T - (z / T).max(1, keepdims=True))
    q /= q.sum(1, keepdims=True)
    q1 = np.exp(z - z.max(1, keepdims=True))
    q1 /= q1.sum(1, keepdims=True)
    p = np.zeros_like(z, np.float64)
    ok = (ids >= 0) & (ids < z.shape[1])
    tt = np.where(ok, t / T, -np.inf)
    with np.errstate(invalid="ignore"):
        pk = np.nan_to_num(np.exp(tt - tt.max(1, keepdims=True)) / np.exp(tt - tt.max(1, keepdims=True)).sum(1, keepdims=True))
    np.add.at(p, (np.arange(len(z))[:, None], np.where(ok, ids, 0)), np.where(ok, pk, 0))
    size = np.abs(scale) * ((1 - alpha) * T * (q + p) + alpha * (q1 + (np.arange(z.shape[1])[None, :] == (y if y is not None else -1 + 0 * z[:, 0])[:, None])))
    if got_d is not None:
        tiny = 2.0 ** -25 if dtype == "f16" else 1e-37
        bound = size * rel + np.abs(wd) * EPS_HALF[dtype] * (1 + 2.0 ** -6) + tiny
        off = np.abs(got_d - wd) - bound
        assert off.max() <= 0, f"gradient: {int((off > 0).sum())} off, worst {np.abs(got_d - wd).max():.3e}"
    parts = (1 - alpha) * T * T * (2 * R + 20) + alpha * (R + 20)
    assert np.all(np.abs(got_l - wl) <= parts * (R + 100) * 2.0 ** -23), f"loss off by {np.abs(got_l - wl).max():.3e}"


SHAPES = [(1, 2, 1), (3, 10, 4), (64, 1000, 8), (5, 1001, 33), (130, 257, 100), (7, 4096, 64), (2, 32000, 512), (3, 50001, 128),
          (2, 131072, 20), (2, 160003, 1000)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,C,K", SHAPES)
def test_loss_and_gradient(gpu, B, C, K, dtype):
    z, ids, t, y = batch(B, C, K, dtype, seed=C)
    for T, alpha, lab in ((1.0, 0.0, None), (2.0, 0.5, y), (1.5, 1.0, y)):
        d, l = run(z, ids, t, lab, dtype, 1.0, T, alpha)
        assert_matches(d, l, z, ids, t, lab, dtype, 1.0, T, alpha)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("C,ld,ld_out,offset", [(1000, 1003, None, 0), (1000, 1000, 1016, 0), (999, 999, None, 5), (40001, 40001, 40004, 1), (2000, 2008, None, 4)])
def test_row_pitches_and_alignments(gpu, C, ld, ld_out, offset, dtype):
    z, ids, t, y = batch(9, C, 40, dtype, seed=C + offset)
    d, l = run(z, ids, t, y, dtype, 0.25, 2.0, 0.25, ld=ld, ld_out=ld_out, offset=offset)
    assert_matches(d, l, z, ids, t, y, dtype, 0.25, 2.0, 0.25)


@pytest.mark.parametrize("C", [300, 1003, 40000])
def test_padding_repeated_columns_and_missing_labels(gpu, C):
    B, K = 12, 64
    z, ids, t, y = batch(B, C, K, "f32", seed=2)
    ids[0] = -1                                  # no entries at all
    ids[1, 5:] = -1
    ids[2, ::2] = C                              # outside on the other side
    ids[3, :] = ids[3, 0]                        # one column, K times
    ids[4, 10:20] = ids[4, 3]
    ids[5, -1] = y[5]                            # the label is among the entries
    ids[6, :3] = y[6]                            # and repeated
    t[7, 1:] = -np.inf                           # weight zero
    t[8] = -np.inf                               # every weight zero: no target
    t[1, 5:] = np.nan                            # what padding holds does not matter
    y[9], y[10] = -1, C
    ids[11], y[11] = -7, -1                      # neither term: zero loss, zero gradient
    for T, alpha in ((1.0, 0.0), (2.0, 0.3)):
        d, l = run(z, ids, t, y, "f32", 1.0, T, alpha)
        clean = t.copy()
        clean[1, 5:] = 0.0
        assert_matches(d, l, z, ids, clean, y, "f32", 1.0, T, alpha)
        assert l[11] == 0.0 and not d[11].any()
        if alpha == 0.0:
            assert l[0] == 0.0 and not d[0].any() and l[8] == 0.0 and not d[8].any()


def test_masked_student_columns(gpu):
    """-inf and the type's lowest value in columns the teacher does not list give q = 0 there; listed, an infinite loss."""
    z, ids, t, y = batch(4, 500, 6, "f32", seed=3)
    free = np.setdiff1d(np.arange(500), ids[:3].ravel())
    z[0, free[:200]], z[1, free[:200]] = -np.inf, -3.4028235e38
    z[3, ids[3, 2]] = -np.inf
    d, l = run(z, ids, t, None, "f32", 1.0, 2.0, 0.0)
    wd, wl = oracle.distill_ce(z, ids, t, None, 1.0, 2.0, 0.0)
    assert np.allclose(l[:3], wl[:3], rtol=3e-6, atol=3e-6) and np.isposinf(l[3]) and np.isposinf(wl[3])
    assert np.allclose(d, wd, rtol=1e-5, atol=1e-7) and not d[0, free[:200]].any() and not d[1, free[:200]].any()


def test_nan_and_infinite_rows_stay_in_their_rows(gpu):
    z, ids, t, y = batch(6, 700, 9, "f32", seed=4)
    clean = (z.copy(), t.copy())
    z[1, 3], z[3, 5], t[4, 2] = np.nan, np.inf, np.nan
    d, l = run(z, ids, t, y, "f32", 1.0, 1.0, 0.5)
    for r in (1, 3, 4):
        assert np.isnan(l[r])
    assert np.isnan(d[1]).any() and np.isnan(d[3]).any() and np.isnan(d[4]).any()
    keep = [0, 2, 5]
    wd, wl = oracle.distill_ce(clean[0], ids, clean[1], y, 1.0, 1.0, 0.5)
    assert np.allclose(l[keep], wl[keep], rtol=1e-5) and np.allclose(d[keep], wd[keep], rtol=1e-5, atol=1e-7)


@pytest.mark.parametrize("t_dtype", ["bf16", "f16"])
def test_teacher_types(gpu, t_dtype):
    z, ids, t, y = batch(20, 1000, 30, "bf16", seed=5)
    held = Tensor.from_numpy(t, t_dtype).float_numpy()
    d, l = run(z, ids, t, y, "bf16", 1.0, 2.0, 0.5, t_dtype=t_dtype)
    assert_matches(d, l, z, ids, held, y, "bf16", 1.0, 2.0, 0.5)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("C", [1000, 1003, 33000, 100003])
def test_in_place_and_loss_only(gpu, C, dtype):
    """The gradient over the logits gives the bits of a separate output; the loss alone gives the same loss."""
    z, ids, t, y = batch(5, C, 50, dtype, seed=6)
    ids[2, 7] = ids[2, 8]
    d, l = run(z, ids, t, y, dtype, 0.5, 2.0, 0.25)
    Z = strided(z, dtype)
    L = Tensor.empty((5,))
    call(OpKind.DistillCE, [Z, Tensor.from_numpy(ids), Tensor.from_numpy(t), Tensor.from_numpy(y)], [Z, L],
         *pack_attrs("distill_ce", {"scale": 0.5, "temperature": 2.0, "alpha": 0.25}))
    assert np.array_equal(Z.float_numpy(), d) and np.array_equal(L.numpy(), l)
    _, l2 = run(z, ids, t, y, dtype, 0.5, 2.0, 0.25, grad=False)
    assert np.array_equal(l, l2)


def test_gradient_against_differences_of_the_loss(gpu):
    B, C, K, T, alpha = 3, 40, 7, 2.0, 0.3
    z, ids, t, y = batch(B, C, K, "f32", seed=7, spread=1.0)
    ids[1, 2] = ids[1, 1]
    d, _ = run(z, ids, t, y, "f32", 1.0, T, alpha)
    h = 2.0 ** -6
    up = np.repeat(z[:, None, :], C, 1) + h * np.eye(C, dtype=np.float32)
    dn = np.repeat(z[:, None, :], C, 1) - h * np.eye(C, dtype=np.float32)
    rep = lambda a: np.repeat(a[:, None], C, 1).reshape((B * C,) + a.shape[1:])  # noqa: E731
    lu = run(up.reshape(B * C, C), rep(ids), rep(t), rep(y), "f32", 1.0, T, alpha)[1]
    ld = run(dn.reshape(B * C, C), rep(ids), rep(t), rep(y), "f32", 1.0, T, alpha)[1]
    num = ((lu.astype(np.float64) - ld) / (2 * h)).reshape(B, C)
    # central difference: h^2/6 times a third derivative of at most 1 (T >= 1); the losses' own error of 1e-6 over h
    assert np.abs(num - d).max() <= h * h / 6 + 2e-6 / h


@pytest.mark.parametrize("B,C,K,dtype", [(700, 1000, 16, "bf16"), (300, 5003, 40, "f32"), (40, 70001, 64, "bf16")])
def test_many_rows_twice_and_replayed(gpu, B, C, K, dtype):
    z, ids, t, y = batch(B, C, K, dtype, seed=8)
    ids[::7, 3] = ids[::7, 4]
    d, l = run(z, ids, t, y, dtype, 1.0 / B, 2.0, 0.5)
    assert_matches(d, l, z, ids, t, y, dtype, 1.0 / B, 2.0, 0.5)
    d2, l2 = run(z, ids, t, y, dtype, 1.0 / B, 2.0, 0.5)
    assert np.array_equal(d, d2) and np.array_equal(l, l2)
    Z, D, L = strided(z, dtype), Tensor.empty((B, C), dtype), Tensor.empty((B,))
    I, T_, Y = Tensor.from_numpy(ids), Tensor.from_numpy(t), Tensor.from_numpy(y)
    stream = _C.graph_begin()
    _C.op_call(OpKind.DistillCE, [Z, I, T_, Y], [D, L], *pack_attrs("distill_ce", {"scale": 1.0 / B, "temperature": 2.0, "alpha": 0.5}), stream)
    _C.graph_end()
    for _ in range(2):
        _C.graph_launch()
    _C.device_sync()
    _C.graph_reset()
    assert np.array_equal(D.float_numpy(), d) and np.array_equal(L.numpy(), l)
    assert _C.wait_status() == 0


LOWEST = {"f32": -3.4028235e38, "bf16": -3.3895314e38, "f16": -65504.0}


@pytest.mark.parametrize("T,alpha", [(1.0, 0.0), (1.0, 0.5), (2.0, 0.5), (4.0, 0.25), (1.5, 0.5), (0.25, 0.5)])
@pytest.mark.parametrize("C,K,dtype", [(500, 6, "f32"), (1000, 40, "bf16"), (1000, 8, "f16"), (20000, 12, "bf16"), (40001, 70, "f32")])
def test_rows_that_a_mask_leaves_nothing_of(gpu, C, K, dtype, T, alpha):
    """Every logit of a row (its teacher's, too) replaced by a large negative number: the softmax is that of the differences,
    uniform where the numbers are equal. Differences of equal logits are exact, so no error grows with the logits' size:
    32 2^-23 relative on sums of C and K equal terms and their quotients, and the types' half steps."""
    values = [-1e4, LOWEST[dtype]] if dtype == "f16" else [-1e9, -3e9, -1e15, -1e30, LOWEST[dtype], -LOWEST[dtype]]
    B = 2 * len(values) + 1
    z, ids, t, y = batch(B, C, K, dtype, seed=C + K)
    for i, v in enumerate(values):
        z[2 * i] = z[2 * i + 1] = v
        t[2 * i] = v
    z[1, :: C // 7] *= 1.5 if dtype == "f16" else 2.0  # below the others by a whole factor: weighs nothing
    t[-1] = LOWEST["f32"]
    z, t = Tensor.from_numpy(z, dtype).float_numpy(), t.astype(np.float32)
    d, l = run(z, ids, t, y if alpha else None, dtype, 1.0, T, alpha)
    wd, wl = oracle.distill_ce(z, ids, t, y if alpha else None, 1.0, T, alpha)
    plain = np.arange(B - 1)  # the last row is an ordinary one with a masked teacher
    size = np.abs(wd) + (1 - alpha) * T / np.maximum(1, (t == t.max(1, keepdims=True)).sum(1, keepdims=True)) + alpha
    tiny = 2.0 ** -25 if dtype == "f16" else 1e-37
    listed = np.zeros((B, C), bool)
    np.put_along_axis(listed, ids, True, 1)
    if alpha:
        listed[np.arange(B), y] = True
    bound = np.where(listed, size, np.abs(wd)) * 128 * 2.0 ** -23 + np.abs(wd) * EPS_HALF[dtype] * (1 + 2.0 ** -6) + tiny
    assert np.all(np.abs(d - wd)[plain] <= bound[plain]), f"gradient off by {np.abs(d - wd)[plain].max():.3e}"
    with np.errstate(over="ignore"):
        fits = np.abs(wl) < 3e38
        assert np.all(np.isposinf(l[~fits]))
        assert np.all(np.abs(l - wl)[fits] <= 128 * 2.0 ** -23 * (np.abs(wl[fits]) + 20 * T * T)), (l, wl)
    assert np.abs(d[-1] - wd[-1]).max() <= 128 * 2.0 ** -23 * T + EPS_HALF[dtype] * np.abs(wd[-1]).max()


@pytest.mark.parametrize("C,K,dtype", [(500, 6, "f32"), (20000, 12, "bf16"), (40001, 70, "f32")])
def test_a_listed_column_with_the_lowest_logit_has_a_finite_loss(gpu, C, K, dtype):
    z, ids, t, y = batch(3, C, K, dtype, seed=K)
    z[0, ids[0, 1]] = z[1, y[1]] = LOWEST[dtype]
    d, l = run(z, ids, t, y, dtype, 1.0, 1.0, 0.25)
    wd, wl = oracle.distill_ce(z, ids, t, y, 1.0, 1.0, 0.25)
    assert np.all(np.abs(l - wl) <= 128 * 2.0 ** -23 * (np.abs(wl) + 20)), (l, wl)
    assert np.all(np.abs(d - wd) <= 128 * 2.0 ** -23 + EPS_HALF[dtype] * np.abs(wd))
