"""Workloads of the 8-bit block-scaled linear layer and of the distillation loss.

Three operators, as one training step of a student uses them:

  quant     a matrix to 8-bit floating point with one fp32 scale per block of 128 values: along the rows (what a product
            that sums over the columns reads), along the columns (what the weight gradient reads, summing over the rows),
            both from one read, or per 128 x 128 tile (weights)
  linear    the layer's three products on such operands: forward with bias and ReLU, input gradient with the ReLU mask,
            weight gradient in fp32
  distill   loss rows and logit gradient of a student against its teacher's top logits, optionally mixed with the
            cross-entropy of the labels

`own` selects the side: elementary torch operations in fp32, or this repository's operators through `aicf_cuda._C`.
"""
import math
import sys
from pathlib import Path

import torch

own = False

BLOCK = 128
TINY = 2.0 ** -100  # a block whose largest magnitude is below this is scaled as if it were this
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
FORMATS = {"e4m3": (torch.float8_e4m3fn, 448.0), "e5m2": (torch.float8_e5m2, 57344.0)}


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one small batch of the 784-256-10 classifier: launch latency
        dict(name="quant_small", op="quant", rows=64, cols=784, dtype="f32", layout="rows_cols", fmt="e4m3"),
        # a hidden layer's fp32 master weight, once per step
        dict(name="quant_weight", op="quant", rows=8192, cols=8192, dtype="f32", layout="tiles", fmt="e4m3"),
        # a hidden activation of the full batch: the forward product reads one form, the weight gradient the other
        dict(name="quant_activation", op="quant", rows=65536, cols=8192, dtype="bf16", layout="rows_cols", fmt="e4m3"),
        # first layer of the small classifier
        dict(name="linear_small", op="linear", form="fwd", m=64, n=256, k=784, relu=True, fmt="e4m3", out="bf16", packed=False),
        # one sample through a hidden layer: a stream of the weight
        dict(name="linear_one_row", op="linear", form="fwd", m=1, n=8192, k=8192, relu=True, fmt="e4m3", out="bf16", packed=False),
        # a hidden layer of the full batch
        dict(name="linear_hidden", op="linear", form="fwd", m=65536, n=8192, k=8192, relu=True, fmt="e4m3", out="bf16", packed=False),
        # input gradient behind the 1000-class layer: K is no multiple of 128, gradients in the wide-range format
        dict(name="linear_dx_classes", op="linear", form="dx", m=65536, n=8192, k=1000, relu=False, fmt="e5m2", out="bf16", packed=False),
        # weight gradient of the 1000-class layer: both operands scaled along the batch
        dict(name="linear_dw_classes", op="linear", form="dw", m=1000, n=8192, k=65536, relu=False, fmt="e4m3", out="f32", packed=False),
        # a handful of rows, a handful of classes: launch latency
        dict(name="distill_small", op="distill", rows=64, cols=1000, top=8, dtype="f32", temperature=2.0, alpha=0.5, scale=1 / 64, padded=False),
        # the 1000-class student of the full batch, half distillation, half labels
        dict(name="distill_classes", op="distill", rows=65536, cols=1000, top=16, dtype="bf16", temperature=2.0, alpha=0.5, scale=1 / 65536, padded=True),
        # a vocabulary in fp32
        dict(name="distill_vocab", op="distill", rows=8192, cols=32000, top=64, dtype="f32", temperature=1.0, alpha=0.0, scale=1 / 8192, padded=True),
        # a long odd row: no row starts where the one before it did within 16 bytes
        dict(name="distill_long_odd", op="distill", rows=4096, cols=100003, top=128, dtype="bf16", temperature=1.5, alpha=0.25, scale=1 / 4096, padded=True),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["quant", "linear", "linear", "distill", "distill"])
    if op == "quant":
        rows, cols = _log_uniform(rng, 1, 65536), _log_uniform(rng, 16, 32768)
        while rows * cols > 65536 * 8192:
            rows //= 2
        return dict(op=op, rows=rows, cols=cols, dtype=rng.choice(list(DTYPES)), layout=rng.choice(["rows", "cols", "rows_cols", "tiles"]),
                    fmt=rng.choice(list(FORMATS)))
    if op == "linear":
        form = rng.choice(["fwd", "dx", "dw"])
        m, n, k = _log_uniform(rng, 1, 32768), _log_uniform(rng, 8, 16384), _log_uniform(rng, 16, 32768)
        while m * n * k > 2 ** 39:
            m, n, k = (m + 1) // 2, (n + 1) // 2, (k + 1) // 2
        return dict(op=op, form=form, m=m, n=n, k=k, relu=form == "fwd" and rng.random() < 0.7, fmt=rng.choice(list(FORMATS)),
                    out=rng.choice(["f32", "bf16"]) if form == "dw" else rng.choice(["bf16", "bf16", "f16", "f32"]), packed=rng.random() < 0.25)
    rows, cols = _log_uniform(rng, 1, 65536), _log_uniform(rng, 10, 160000)
    while rows * cols > 4096 * 100003:
        rows = (rows + 1) // 2
    dtype = rng.choice(list(DTYPES))
    return dict(op=op, rows=rows, cols=cols, top=min(cols, _log_uniform(rng, 1, 512)), dtype=dtype, temperature=rng.choice([1.0, 1.5, 2.0, 4.0]),
                alpha=rng.choice([0.0, 0.0, 0.1, 0.5]), scale=1.0 if dtype == "f16" else 1.0 / rows, padded=rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------ inputs
def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def _bytes_matrix(rows, cols, packed):
    """An uninitialised 8-bit matrix: rows 16 bytes aligned, or packed."""
    pitch = cols if packed else (cols + 15) // 16 * 16
    return torch.empty((rows, pitch), dtype=torch.uint8, device="cuda")[:, :cols]


def _random_fp8(g, rows, cols, fmt, packed, nonneg):
    """Values as a quantised matrix holds them: a bell curve that reaches the format's largest value, half of it zero behind a ReLU."""
    dt, top = FORMATS[fmt]
    v = torch.randn((rows, cols), generator=g, device="cuda", dtype=torch.float32).mul_(top / 4).clamp_(-top, top)
    if nonneg:
        v.clamp_(min=0.0)
    m = _bytes_matrix(rows, cols, packed).view(dt)
    m.copy_(v)
    return m


def _random_scales(g, shape, fmt):
    return torch.randn(shape, generator=g, device="cuda").mul_(0.5).exp_().mul_(1.0 / FORMATS[fmt][1])


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    s = {"case": case}
    if case["op"] == "quant":
        M, N = case["rows"], case["cols"]
        # activations behind a ReLU (weights: a bell curve), channels of different size, a few all-zero (padding) rows
        x = torch.randn((M, N), generator=g, device="cuda", dtype=torch.float32 if case["dtype"] == "f32" else torch.bfloat16)
        if case["layout"] != "tiles":
            x.clamp_(min=0.0).mul_(torch.randn((N,), generator=g, device="cuda").mul_(0.7).exp_().to(x.dtype))
            x.masked_fill_((torch.rand((M, 1), generator=g, device="cuda") < 0.01), 0.0)
        s["x"] = x.to(DTYPES[case["dtype"]])
        dt = FORMATS[case["fmt"]][0]
        s["out"] = []
        if case["layout"] in ("rows", "rows_cols"):
            s["out"] += [_bytes_matrix(M, N, False).view(dt), torch.empty((M, _blocks(N)), device="cuda")]
        if case["layout"] in ("cols", "rows_cols"):
            s["out"] += [_bytes_matrix(M, N, False).view(dt), torch.empty((_blocks(M), N), device="cuda")]
        if case["layout"] == "tiles":
            s["out"] += [_bytes_matrix(M, N, False).view(dt), torch.empty((_blocks(M), _blocks(N)), device="cuda")]
    elif case["op"] == "linear":
        m, n, k, fmt, packed = case["m"], case["n"], case["k"], case["fmt"], case["packed"]
        if case["form"] == "fwd":    # x [m,k], w [n,k]
            s["a"], s["sa"] = _random_fp8(g, m, k, "e4m3", packed, True), _random_scales(g, (m, _blocks(k)), "e4m3")
            s["b"], s["sb"] = _random_fp8(g, n, k, fmt, packed, False), _random_scales(g, (_blocks(n), _blocks(k)), fmt)
            s["bias"] = torch.randn((n,), generator=g, device="cuda")
        elif case["form"] == "dx":   # dy [m,k], w [k,n], activation y [m,n]
            s["a"], s["sa"] = _random_fp8(g, m, k, fmt, packed, False), _random_scales(g, (m, _blocks(k)), fmt)
            s["b"], s["sb"] = _random_fp8(g, k, n, "e4m3", packed, False), _random_scales(g, (_blocks(k), _blocks(n)), "e4m3")
            s["y"] = torch.randn((m, n), generator=g, device="cuda", dtype=torch.bfloat16).clamp_(min=0.0).to(DTYPES[case["out"]])
        else:                        # dy [k,m], x [k,n]
            s["a"], s["sa"] = _random_fp8(g, k, m, fmt, packed, False), _random_scales(g, (_blocks(k), m), fmt)
            s["b"], s["sb"] = _random_fp8(g, k, n, "e4m3", packed, True), _random_scales(g, (_blocks(k), n), "e4m3")
        s["out"] = torch.empty((m, n), device="cuda", dtype=DTYPES[case["out"]])
    else:
        B, C, K = case["rows"], case["cols"], case["top"]
        z = torch.randn((B, C), generator=g, device="cuda", dtype=torch.bfloat16 if case["dtype"] == "bf16" else torch.float32).mul_(2.0)
        s["z"] = z.to(DTYPES[case["dtype"]])
        # the teacher agrees with the student in part; its K largest logits
        teacher = torch.randn((B, C), generator=g, device="cuda", dtype=z.dtype).add_(z, alpha=0.7)
        t, ids = torch.topk(teacher, K, dim=1)
        s["t"], s["ids"] = t.float(), ids.to(torch.int32)
        s["labels"] = torch.randint(0, C, (B,), generator=g, device="cuda", dtype=torch.int32)
        if case["padded"]:  # rows with fewer entries than K, some with none; rows without a label
            short = torch.rand((B,), generator=g, device="cuda") < 0.25
            count = torch.where(short, torch.randint(0, K + 1, (B,), generator=g, device="cuda"), torch.full((B,), K, device="cuda"))
            gone = torch.arange(K, device="cuda")[None, :] >= count[:, None]
            s["ids"].masked_fill_(gone, -1)
            s["t"].masked_fill_(gone, 0.0)
            s["labels"].masked_fill_(torch.rand((B,), generator=g, device="cuda") < 0.02, -1)
        s["out"] = [torch.empty_like(s["z"]), torch.empty((B,), device="cuda")]
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_quant(x, along, fmt):
    """Per block of 128 along dimension 1 (rows), 0 (cols) or both (tiles): scale = amax / top, value = round(x * (top / amax))."""
    dt, top = FORMATS[fmt]
    M, N = x.shape
    by, bx = (BLOCK if along in ("cols", "tiles") else 1), (BLOCK if along in ("rows", "tiles") else 1)
    x = torch.nn.functional.pad(x.float(), (0, -N % bx, 0, -M % by))
    v = x.view(x.shape[0] // by, by, x.shape[1] // bx, bx)
    amax = v.abs().amax(dim=(1, 3), keepdim=True).clamp_(min=TINY)
    q = (v * (top / amax)).to(dt).view(x.shape)[:M, :N]
    return [q, (amax / top).view(amax.shape[0], amax.shape[2])]


def _dequant(q, s):
    """fp32 values of a quantised matrix whose scale matrix divides each dimension by 1 or by 128."""
    v = q.float()
    if s.shape[0] != q.shape[0]:
        s = s.repeat_interleave(BLOCK, 0)[: q.shape[0]]
    if s.shape[1] != q.shape[1]:
        s = s.repeat_interleave(BLOCK, 1)[:, : q.shape[1]]
    return v.mul_(s)


def _plain_linear(s):
    case = s["case"]
    a, b = _dequant(s["a"], s["sa"]), _dequant(s["b"], s["sb"])
    if case["form"] == "fwd":
        c = (a @ b.t()).add_(s["bias"])
        c = c.clamp_(min=0.0) if case["relu"] else c
    elif case["form"] == "dx":
        c = (a @ b).mul_(s["y"] > 0)
    else:
        c = a.t() @ b
    return c.to(DTYPES[case["out"]])


def _plain_distill(s):
    case = s["case"]
    T, alpha, scale, C = case["temperature"], case["alpha"], case["scale"], case["cols"]
    z = s["z"].float()
    mz = z.amax(dim=1, keepdim=True)
    ez = ((z - mz) / T).exp_()
    sz = ez.sum(dim=1, keepdim=True)
    valid = (s["ids"] >= 0) & (s["ids"] < C)
    ids = s["ids"].clamp(0, C - 1).long()
    has = valid.any(dim=1, keepdim=True)
    t = s["t"].masked_fill(~valid, -math.inf)
    mt = t.amax(dim=1, keepdim=True).masked_fill(~has, 0.0)
    a = (t - mt) / T
    et = a.exp()
    p = et / et.sum(dim=1, keepdim=True).masked_fill(~has, 1.0)
    b = (z.gather(1, ids) - mz) / T
    cross = torch.where(p > 0, p * (a - b), torch.zeros_like(p)).sum(dim=1, keepdim=True)
    soft = torch.where(has, cross - et.sum(dim=1, keepdim=True).log() + sz.log(), torch.zeros_like(cross))
    loss = (1.0 - alpha) * T * T * soft
    g = (ez / sz) * has
    g.scatter_add_(1, ids, -p)
    g.mul_((1.0 - alpha) * T)
    if alpha > 0.0:
        known = (s["labels"] >= 0) & (s["labels"] < C)
        label = s["labels"].clamp(0, C - 1).long()[:, None]
        e1 = (z - mz).exp_()
        s1 = e1.sum(dim=1, keepdim=True)
        hard = s1.log() + mz - z.gather(1, label)
        loss = loss + alpha * hard * known[:, None]
        g.addcmul_(e1, (alpha / s1) * known[:, None])
        g.scatter_add_(1, label, -alpha * known[:, None].float())
    return [g.mul_(scale).to(s["z"].dtype), loss.view(-1)]


# ------------------------------------------------------------------------------------------------ this repository
_PACKAGE = str(Path(__file__).resolve().parents[1] / "ai-compiler-framework_b200" / "python")


def _aicf():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    import aicf_cuda
    return aicf_cuda


def _attrs(s, op, attrs):
    """The operator's packed attributes, kept with the state as a program would keep them."""
    if "attrs" not in s:
        s["attrs"] = _aicf().pack_attrs(op, attrs)
    return s["attrs"]


def _own(s):
    _C = _aicf()._C
    case, stream = s["case"], torch.cuda.current_stream().cuda_stream
    if case["op"] == "quant":
        _C.op_call(_C.OpKind.QuantFp8, [s["x"]], s["out"], stream=stream)
    elif case["op"] == "linear":
        if case["form"] == "fwd":
            schema, payload = _attrs(s, "gemm_epilogue", {"transB": True, "epilogue": "bias_relu" if case["relu"] else "bias"})
            _C.op_call(_C.OpKind.GemmEpilogue, [s["a"], s["b"], s["bias"], s["sa"], s["sb"]], [s["out"]], schema, payload, stream)
        elif case["form"] == "dx":
            schema, payload = _attrs(s, "gemm_relu_bwd", {})
            _C.op_call(_C.OpKind.GemmReluBwd, [s["a"], s["b"], s["y"], s["sa"], s["sb"]], [s["out"]], schema, payload, stream)
        else:
            schema, payload = _attrs(s, "gemm", {"transA": True})
            _C.op_call(_C.OpKind.Gemm, [s["a"], s["b"], s["sa"], s["sb"]], [s["out"]], schema, payload, stream)
    else:
        schema, payload = _attrs(s, "distill_ce", {"scale": case["scale"], "temperature": case["temperature"], "alpha": case["alpha"]})
        labels = [s["labels"]] if case["alpha"] > 0.0 else []
        _C.op_call(_C.OpKind.DistillCE, [s["z"], s["ids"], s["t"]] + labels, s["out"], schema, payload, stream)
    return s["out"]


def run(state):
    if own:
        return _own(state)
    case = state["case"]
    if case["op"] == "quant":
        return [y for along in (["rows", "cols"] if case["layout"] == "rows_cols" else [case["layout"]])
                for y in _plain_quant(state["x"], along, case["fmt"])]
    return _plain_linear(state) if case["op"] == "linear" else _plain_distill(state)


def work(case):
    if case["op"] == "quant":
        M, N = case["rows"], case["cols"]
        size = {"f32": 4, "f16": 2, "bf16": 2}[case["dtype"]]
        forms = {"rows": M * _blocks(N), "cols": _blocks(M) * N, "tiles": _blocks(M) * _blocks(N)}
        made = ["rows", "cols"] if case["layout"] == "rows_cols" else [case["layout"]]
        return {"bytes": M * N * size + sum(M * N + 4 * forms[f] for f in made), "flops": M * N * (1 + 2 * len(made))}
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        osize = 4 if case["out"] == "f32" else 2
        kb = _blocks(k)
        if case["form"] == "fwd":
            extra = 4 * (m * kb + _blocks(n) * kb) + 4 * n
        elif case["form"] == "dx":
            extra = 4 * (m * kb + _blocks(n) * kb) + m * n * osize
        else:
            extra = 4 * kb * (m + n)
        return {"bytes": m * k + n * k + m * n * osize + extra, "flops": 2 * m * n * k}
    B, C, K = case["rows"], case["cols"], case["top"]
    size = 4 if case["dtype"] == "f32" else 2
    return {"bytes": 2 * B * C * size + 8 * B * K + 8 * B, "flops": B * C * (6 if case["alpha"] > 0 else 4)}


# ------------------------------------------------------------------------------------------------ definitions in 64 bits
def _round_to_format(v, fmt):
    """The nearest value of the format (ties to even), as a 64-bit number; |v| is at most the format's largest value."""
    mantissa, lowest = (3, -6) if fmt == "e4m3" else (2, -14)
    exponent = torch.frexp(v).exponent.sub_(1).clamp_(min=lowest)
    step = torch.ldexp(torch.ones((), device=v.device, dtype=torch.float64), exponent - mantissa)
    return torch.round(v / step) * step


def _exact_quant(x, along, fmt):
    top = FORMATS[fmt][1]
    values, scales = torch.empty(x.shape, dtype=torch.float64, device=x.device), []
    axis = {"rows": (1,), "cols": (0,), "tiles": (0, 1)}[along]
    for r0 in range(0, x.shape[0], 64 * BLOCK):  # a band of rows at a time: 64-bit copies are large
        band = x[r0:r0 + 64 * BLOCK].double()
        amax = band.abs()
        for d in axis:
            amax = torch.stack([piece.amax(dim=d) for piece in amax.split(BLOCK, dim=d)], dim=d)
        amax = amax.clamp(min=TINY)
        scales.append(amax / top)
        spread = amax
        for d in axis:
            index = torch.arange(band.shape[d], device=x.device) // BLOCK
            spread = spread.index_select(d, index)
        values[r0:r0 + 64 * BLOCK] = _round_to_format(band * top / spread, fmt)
    return [values, torch.cat(scales)]


def _exact_linear(s):
    case = s["case"]
    a, b = s["a"].double(), s["b"].double()
    sa, sb = s["sa"].double(), s["sb"].double()
    if case["form"] != "dw":  # bring both to [rows, k] and [k, cols] with scales [rows or blocks, k blocks]
        if case["form"] == "fwd":
            b, sb = b.t(), sb.t()
        sb = sb[:, torch.arange(b.shape[1], device=b.device) // BLOCK]
    else:
        a, sa = a.t(), sa.t()
    c = torch.zeros((a.shape[0], b.shape[1]), dtype=torch.float64, device=a.device)
    step = BLOCK * 64
    for k0 in range(0, a.shape[1], step):
        block = torch.arange(k0, min(k0 + step, a.shape[1]), device=a.device) // BLOCK
        c += (a[:, k0:k0 + step] * sa[:, block]) @ (b[k0:k0 + step] * sb[block])
    if case["form"] == "fwd":
        c += s["bias"].double()
        if case["relu"]:
            c = torch.relu(c)
    elif case["form"] == "dx":
        c[s["y"] <= 0] = 0.0
    return c


def _exact_distill(s):
    case = s["case"]
    T, alpha, C = case["temperature"], case["alpha"], case["cols"]
    grad, loss = torch.empty(s["z"].shape, dtype=torch.float64, device=s["z"].device), []
    for r0 in range(0, s["z"].shape[0], 512):
        z, t, ids, labels = (s[n][r0:r0 + 512] for n in ("z", "t", "ids", "labels"))
        z, t, ids, labels = z.double(), t.double(), ids.long(), labels.long()
        ok = (ids >= 0) & (ids < C)
        some = ok.any(dim=1)
        logq = z / T - torch.logsumexp(z / T, dim=1, keepdim=True)
        tt = torch.where(ok, t / T, torch.full_like(t, -math.inf))
        tt[~some] = 0.0
        logp = tt - torch.logsumexp(tt, dim=1, keepdim=True)
        p = torch.where(ok & some[:, None], logp.exp(), torch.zeros_like(logp))
        terms = p * (logp - logq.gather(1, torch.where(ok, ids, torch.zeros_like(ids))))
        soft = torch.where(p > 0, terms, torch.zeros_like(terms)).sum(dim=1) * T * T
        target = torch.zeros_like(z).scatter_add_(1, torch.where(ok, ids, torch.zeros_like(ids)), p)
        g = (1 - alpha) * T * (logq.exp() * some[:, None] - target)
        row_loss = (1 - alpha) * soft
        if alpha > 0:
            rows = torch.nonzero((labels >= 0) & (labels < C)).view(-1)
            log1 = z[rows] - torch.logsumexp(z[rows], dim=1, keepdim=True)
            one = torch.zeros_like(log1)
            one[torch.arange(len(rows), device=z.device), labels[rows]] = 1.0
            g[rows] += alpha * (log1.exp() - one)
            row_loss[rows] -= alpha * (log1 * one).sum(dim=1)
        grad[r0:r0 + 512] = g * case["scale"]
        loss.append(row_loss)
    return [grad, torch.cat(loss)]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quant":
        return [y for along in (["rows", "cols"] if case["layout"] == "rows_cols" else [case["layout"]])
                for y in _exact_quant(s["x"], along, case["fmt"])]
    return _exact_linear(s) if case["op"] == "linear" else _exact_distill(s)
