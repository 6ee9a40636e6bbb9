"""The operators together: an MLP train step whose linear layers multiply block-scaled 8-bit matrices, and whose student
is distilled from a teacher's top logits, as one captured plan against the same lowered list in 64 bits."""
import numpy as np
import pytest

import oracle
from aicf_cuda import Plan, build_mlp_train_step, f32_to_bf16_bits, plan_from_json, plan_to_json


def lowered(batch, dims, **kw):
    return build_mlp_train_step(batch, dims, **kw)


def host_env(vals, dims, batch, seed=0, top=0):
    params = oracle.mlp_params(dims, seed)
    x, y = oracle.mlp_batch(batch, dims[0], dims[-1], seed)
    rng = np.random.default_rng(seed + 1)
    t = 2 * rng.standard_normal((batch, dims[-1])).astype(np.float32)
    ids = np.argsort(-t, axis=1)[:, :top].astype(np.int32) if top else None
    given = {"x": x, "labels": y}
    if top:
        given.update({"teacher.ids": ids, "teacher.logits": np.take_along_axis(t, ids, 1)})
    env, dtypes = {}, {}
    for v in vals:
        dtypes[v.vid] = v.dtype
        arr = given.get(v.name, params.get(v.name))
        if arr is None and v.name.endswith(".W.lp"):
            arr = oracle.cast(params[v.name[:-3]], v.dtype)
        given_here = arr is not None
        env[v.vid] = np.array(arr if given_here else np.zeros(v.shape), np.int32 if v.dtype == "i32" else np.float32)
        yield v, env[v.vid] if given_here else None, env, dtypes


def test_lowering_of_the_fp8_step():
    vals, ops = lowered(96, [200, 256, 40], compute_dtype="bf16", linear="fp8", fp8_grad="f8e5m2")
    names = [o["op"] for o in ops]
    assert names.count("quant_fp8") == 2 + 2 + 2 and "cast" not in names
    kids = {o["kernel_id"] for o in ops}
    assert {"gemm_bias_relu_fp8_block128_out_bf16_v0", "gemm_relu_bwd_fp8_block128_out_bf16_v0", "gemm_fp8_block128_out_f32_v0"} <= kids
    by = {v.name: v for v in vals}
    assert not any(n.endswith(".lp") for n in by)
    assert by["0.W.s_tiles"].shape == (2, 2) and by["x.s_rows"].shape == (96, 2) and by["x.s_cols"].shape == (1, 200)
    assert by["d_logits.q_cols"].dtype == "f8e5m2" and by["x.q_rows"].dtype == "f8e4m3"
    assert plan_from_json(plan_to_json("p", vals, ops))[2] == ops


def test_lowering_of_the_distillation_step():
    vals, ops = lowered(32, [20, 12], compute_dtype="f32", loss="distill", teacher_top=5, temperature=2.0)
    by = {v.name: v for v in vals}
    assert by["teacher.ids"].dtype == "i32" and by["teacher.logits"].shape == (32, 5) and "labels" not in by
    d = next(o for o in ops if o["op"] == "distill_ce")
    assert d["attrs"] == {"scale": 1 / 32, "temperature": 2.0, "alpha": 0.0} and d["kernel_id"] == "distill_ce_f32_v0"
    assert "labels" in {v.name for v in lowered(32, [20, 12], loss="distill", teacher_top=5, alpha=0.5)[0]}


@pytest.mark.parametrize("kw", [dict(linear="int8"), dict(linear="fp8", compute_dtype="f32"), dict(linear="fp8", data_parallel="fused"),
                                dict(linear="fp8", fp8_grad="f16"), dict(loss="mse"), dict(loss="distill"), dict(loss="distill", teacher_top=2000),
                                dict(loss="distill", teacher_top=4, with_argmax=True), dict(loss="distill", teacher_top=4, alpha=-0.5),
                                dict(loss="distill", teacher_top=4, temperature=0.0)])
def test_lowering_refuses(kw):
    with pytest.raises(ValueError):
        lowered(32, [20, 12], **kw)


def test_steps_without_the_new_options_are_what_they_were():
    for cd in ("f32", "bf16"):
        vals, ops = lowered(64, [784, 256, 10], compute_dtype=cd)
        assert [o["op"] for o in ops if o["op"] in ("quant_fp8", "distill_ce")] == [] and not any(v.dtype.startswith("f8") for v in vals)


CASES = [
    dict(dims=[200, 256, 40], batch=96, kw=dict(linear="fp8")),
    dict(dims=[130, 300, 120, 72], batch=150, kw=dict(linear="fp8", loss="distill", teacher_top=8, temperature=2.0, alpha=0.5)),
    dict(dims=[256, 384, 100], batch=256, kw=dict(linear="fp8", fp8_grad="f8e5m2", loss="distill", teacher_top=40, temperature=1.0)),
    dict(dims=[96, 128, 50], batch=64, kw=dict(loss="distill", teacher_top=10, temperature=4.0, alpha=0.25)),
    dict(dims=[96, 128, 50], batch=64, kw=dict(linear="fp8", fuse_relu_bwd=False, input_f32=False)),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=range(len(CASES)))
def test_captured_step_against_the_same_list_in_64_bits(gpu, case):
    """First step: every parameter gradient and the loss. The device and the 64-bit run round the same quantities to bf16 and
    to 8 bits; where a sum lies at a rounding border the two may round apart, by one 8-bit step (2^-3 of a value for e4m3,
    2^-2 for e5m2) in a few places, so gradients are compared in norm: an element that rounds apart changes it by 2^-2 / sqrt(n).
    Bound 1e-2 (bf16's own half step is 2^-8, three of them in a row along a layer)."""
    dims, batch, kw = case["dims"], case["batch"], case["kw"]
    vals, ops = lowered(batch, dims, compute_dtype="bf16", lr=1e-3, **kw)
    plan = Plan("fp8", vals, ops)
    for v, arr, env, dtypes in host_env(vals, dims, batch, top=kw.get("teacher_top", 0)):
        if arr is not None:
            plan.tensor(v.vid).copy_from_host(f32_to_bf16_bits(arr) if v.dtype == "bf16" else arr)
            if v.dtype == "bf16":
                env[v.vid] = oracle.bf16_round(arr)
    plan.run()
    plan.sync()
    oracle.run_lowered(ops, env, dtypes, np.float64)
    by = plan.by_name
    got, want = float(plan.tensor("loss").numpy()[0]), float(env[by["loss"]][0])
    assert abs(got - want) <= 2e-3 * abs(want), (got, want)
    for i in range(len(dims) - 1):
        m = plan.tensor(f"opt.m.{2 * i}.W").numpy()  # after one step the first moment is (1 - beta1) times the gradient
        w = env[by[f"opt.m.{2 * i}.W"]]
        rel = np.linalg.norm(m.astype(np.float64) - w) / np.linalg.norm(w)
        assert rel <= 1e-2, (i, rel)
    # and captured: the graph holds every launch of the step, the aligned copies of odd-pitched operands among them
    plan.capture()
    plan.replay(30)
    plan.sync()
    assert np.isfinite(float(plan.tensor("loss").numpy()[0]))
    plan.close()
