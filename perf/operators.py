"""The 8-bit (W8A8) operators of the decoder layer, as a user calls them.

Cases are dicts: ``op`` ("norm": add-residual RMSNorm to int8 rows, "rows":
rows to int8, "swiglu": SwiGLU to int8 rows, "linear": int8 product with a
scale per token and per output channel), its sizes and ``dtype``, the type of
the activations. ``run`` computes a case in plain torch operations, or with
``own`` through llama2_b200.ops. int8 results come back as the values they
stand for (q * scale), in the activations' type, next to their scales.
"""
import math

import torch

own = False
device = "cuda"

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # one token of a batch-1 decode step, 7B width: latency
        dict(name="norm 1x4096 bf16", op="norm", rows=1, dim=4096, add=True, dtype="bf16"),
        # a decode batch at 13B width
        dict(name="norm 64x5120 f16", op="norm", rows=64, dim=5120, add=True, dtype="f16"),
        # the first layer's norm (nothing to add), fp32, an odd width: rows of no alignment
        dict(name="norm 333x1023 f32", op="norm", rows=333, dim=1023, add=False, dtype="f32"),
        # 8 prompts of 2048 tokens
        dict(name="norm 16384x4096 bf16", op="norm", rows=16384, dim=4096, add=True, dtype="bf16"),
        # the attention output of a decode batch, before the O projection
        dict(name="rows 64x4096 bf16", op="rows", rows=64, dim=4096, dtype="bf16"),
        # gate/up weights [out, in] from an fp32 checkpoint, one scale per output channel
        dict(name="rows 22016x4096 f32", op="rows", rows=22016, dim=4096, dtype="f32"),
        # a decode batch's gate/up product
        dict(name="swiglu 64x11008 bf16", op="swiglu", rows=64, dim=11008, dtype="bf16"),
        # a prompt batch of odd length at 13B width
        dict(name="swiglu 4099x13824 f16", op="swiglu", rows=4099, dim=13824, dtype="f16"),
        # the O projection of one token: latency
        dict(name="linear 1x4096x4096 bf16", op="linear", rows=1, n=4096, dim=4096, dtype="bf16"),
        # the gate/up projection of a decode batch: the weights' bytes
        dict(name="linear 64x22016x4096 bf16", op="linear", rows=64, n=22016, dim=4096, dtype="bf16"),
        # a short ragged prompt through a projection of odd width, fp32 activations
        dict(name="linear 257x1003x2064 f32", op="linear", rows=257, n=1003, dim=2064, dtype="f32"),
        # the QKV projection of 8 prompts of 2048 tokens: the tensor cores' rate
        dict(name="linear 16384x12288x4096 bf16", op="linear", rows=16384, n=12288, dim=4096, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "rows", "swiglu", "linear", "linear"])
    if op == "linear":
        # row lengths of int8 operands are multiples of 16 in every layer; tokens and channels are not
        dim = 16 * _log_int(rng, 4, 864)
        n = _log_int(rng, 16, 32000)
        rows = _log_int(rng, 1, min(16384, 16384 * 12288 * 4096 // (n * dim)))
        return dict(op=op, rows=rows, n=n, dim=dim, dtype=rng.choice(["f32", "f16", "bf16"]))
    dim = _log_int(rng, 64, 16384)
    if rng.random() < 0.7:
        dim = (dim + 15) // 16 * 16
    rows = _log_int(rng, 1, min(22016, 4099 * 13824 // dim))
    # a gate/up product has 16 bits
    dtype = rng.choice(["f16", "bf16"] if op == "swiglu" else ["f32", "f16", "bf16"])
    case = dict(op=op, rows=rows, dim=dim, dtype=dtype)
    if op == "norm":
        case["add"] = rng.random() < 0.8
    return case


def work(case):
    m, d, es = case["rows"], case["dim"], 4 if case["dtype"] == "f32" else 2
    out = m * d + 4 * m  # int8 rows and their scales
    if case["op"] == "norm":
        return {"bytes": es * (m * d * (3 if case["add"] else 1) + d) + out, "flops": m * d * (7 if case["add"] else 6)}
    if case["op"] == "rows":
        return {"bytes": es * m * d + out, "flops": 3 * m * d}
    if case["op"] == "swiglu":
        return {"bytes": 2 * es * m * d + out, "flops": 8 * m * d}
    n = case["n"]
    return {"bytes": m * d + n * d + 4 * (m + n) + es * m * n, "flops": 2 * m * n * d}


# --------------------------------------------------------------- the inputs
def prepare(case, seed):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    m, d, t = case["rows"], case["dim"], DTYPES[case["dtype"]]
    randn = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
    s = {"case": case}
    if case["op"] == "linear":
        n = case["n"]
        # rows of normal values quantised by their largest (about 4.2 standard deviations at these widths)
        s["a"] = randn(m, d).mul_(30).round_().clamp_(-127, 127).to(torch.int8)
        s["b"] = randn(n, d).mul_(30).round_().clamp_(-127, 127).to(torch.int8)
        s["a_scales"] = torch.rand(m, generator=g, device=device).add_(0.5).mul_(4.2 / 127)
        s["b_scales"] = torch.rand(n, generator=g, device=device).add_(0.5).mul_(4.2 / 127 / math.sqrt(d))
        s["c"] = torch.empty(m, n, dtype=t, device=device)
        return s
    if case["op"] == "swiglu":
        s["x"] = randn(m, 2 * d).to(t)
    else:
        x = randn(m, d)
        if case["op"] == "norm":
            x[:, torch.randint(0, d, (4,), generator=g, device=device)] *= 20  # the residual stream's outlier channels
            s["w"] = (torch.rand(d, generator=g, device=device) + 0.5).to(t)
            s["residual"] = randn(m, d).to(t)
        if m >= 64:
            x[m // 64::64] = 0  # padding
            if case["op"] == "norm":
                s["residual"][m // 64::64] = 0
        s["x"] = x.to(t)
    s["q"] = torch.empty(m, d, dtype=torch.int8, device=device)
    s["scales"] = torch.empty(m, dtype=torch.float32, device=device)
    return s


# ------------------------------------------------------------ the plain form
def _quantised(y):
    """Row-wise 8-bit values of y (64 bits: values next to a border) and a / 127, a the row's largest magnitude."""
    a = y.abs().amax(1, keepdim=True)
    q = (y * 127 / torch.where(a > 0, a, 1.0)).round()
    return q, a / 127


def _plain(s):
    case = s["case"]
    t = DTYPES[case["dtype"]]
    if case["op"] == "linear":
        acc = s["a"].float() @ s["b"].float().T
        return {"c": (acc * (s["a_scales"][:, None] * s["b_scales"])).to(t)}
    x = s["x"]
    if case["op"] == "rows":
        q, scale = _quantised(x.double())
        return {"y": (q * scale).to(t), "scales": scale[:, 0].float()}
    if case["op"] == "swiglu":
        gate, up = x.double().chunk(2, dim=1)
        q, scale = _quantised(gate / (1 + torch.exp(-gate)) * up)
        return {"y": (q * scale).to(t), "scales": scale[:, 0].float()}
    if case["add"]:
        x.copy_(x.float() + s["residual"].float())
    inv_rms = torch.rsqrt(x.float().square().mean(1, keepdim=True) + 1e-5).double()
    q, scale = _quantised(x.double() * s["w"].double())
    return {"x": x, "y": (q * (scale * inv_rms)).to(t), "scales": (scale * inv_rms)[:, 0].float()}


# ------------------------------------------------------- the framework's form
def _own(s):
    from llama2_b200 import ops

    case = s["case"]
    if case["op"] == "linear":
        ops.launch_linear_int8(s["a"], s["a_scales"], s["b"], s["b_scales"], s["c"])
        return {"c": s["c"]}
    q, scales = s["q"], s["scales"]
    if case["op"] == "rows":
        ops.launch_quantize_rows_int8(s["x"], q, scales)
    elif case["op"] == "swiglu":
        ops.launch_swiglu_int8(s["x"], q, scales)
    else:
        ops.launch_fused_add_residual_rmsnorm_int8(s["w"], s["x"], s["residual"], q, scales, case["add"])
    y = torch.empty(q.shape, dtype=s["x"].dtype, device=q.device)
    torch.mul(q, scales[:, None], out=y)  # the values the bytes stand for
    return {"x": s["x"], "y": y, "scales": scales} if case["op"] == "norm" else {"y": y, "scales": scales}


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    f = torch.float64
    if case["op"] == "linear":
        product = torch.matmul(s["a"].to(f), s["b"].to(f).t())
        return {"c": product.mul_(s["a_scales"].to(f).unsqueeze(1)).mul_(s["b_scales"].to(f).unsqueeze(0))}
    out, inv_rms = {}, 1.0
    if case["op"] == "rows":
        y = s["x"].to(f)
    elif case["op"] == "swiglu":
        gate, up = s["x"][:, : case["dim"]].to(f), s["x"][:, case["dim"]:].to(f)
        y = gate * torch.sigmoid(gate) * up
    else:
        x = s["x"].to(f)
        if case["add"]:
            x = x + s["residual"].to(f)
        out["x"] = x
        stored = x.to(torch.float32).to(s["x"].dtype).to(f)  # the norm is of the stored row
        inv_rms = 1.0 / (stored.pow(2).sum(1, keepdim=True) / case["dim"] + 1e-5).sqrt()
        y = stored * s["w"].to(f)  # 1 / rms cancels in the 8-bit values and stays in their scale
    top = y.abs().max(1, keepdim=True).values
    out["y"] = torch.round(127 * y / top.clamp_min(1e-300)) * top * inv_rms / 127
    out["scales"] = (top * inv_rms / 127).squeeze(1)
    return out
