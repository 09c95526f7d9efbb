"""Operators of 8-bit inference as they are measured: the matrix product of 8-bit integers with a
scale for each token and each channel, and the three ways a program makes its 8-bit operands -- rows
quantised as they are, after a root-mean-square norm with the residual's addition, and after a gated
activation.

With ``own`` false the operators run in their plain form, elementary torch operations in 32 bits (64
for the long sums of the integer product); with ``own`` true through this framework's entry points.
An 8-bit float result comes back as the float8 tensor it is, an 8-bit integer one as bfloat16 (every
integer up to 256 is a bfloat16 number), each next to its fp32 scales.
"""
import torch

own = False

DEV = "cuda"
EPS = 1e-6
FLOATS = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EIGHT = {"i8": torch.int8, "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
QMAX = {"i8": 127.0, "e4m3": 448.0, "e5m2": 57344.0}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1, "e4m3": 1, "e5m2": 1}
TINY = 2.0 ** -126   # the smallest scale of a row


def listed():
    return [
        # --- C = scale_a[m] * scale_b[n] * (A . B^T), int8 operands with K innermost
        # one sequence decoding one token: the weights are read once for a single row
        {"name": "gemm one token", "op": "gemm", "m": 1, "n": 4096, "k": 4096, "out": "bf16"},
        # a decode batch of 16 against a square weight matrix
        {"name": "gemm 16 tokens", "op": "gemm", "m": 16, "n": 8192, "k": 8192, "out": "bf16"},
        # a ragged batch against a layer whose sizes fit no tile, rows not on 16-byte boundaries
        {"name": "gemm ragged", "op": "gemm", "m": 333, "n": 1000, "k": 4099, "out": "f32"},
        # a prompt of 2048 tokens through one projection
        {"name": "gemm prompt 2048", "op": "gemm", "m": 2048, "n": 4096, "k": 8192, "out": "f16"},
        # a full batch of prompts, the size at which the tensor pipes set the time
        {"name": "gemm prompts 8192", "op": "gemm", "m": 8192, "n": 8192, "k": 8192, "out": "bf16"},
        # --- h = x + residual; 8-bit rows and scales of h / rms(h) * weight, and h itself
        # one token between two layers of a decoder
        {"name": "norm one token", "op": "rmsnorm", "rows": 1, "cols": 4096, "in": "bf16", "q": "e4m3", "residual": True},
        # a ragged decode batch, no residual yet (a first layer), an odd width
        {"name": "norm ragged", "op": "rmsnorm", "rows": 1023, "cols": 5001, "in": "f16", "q": "i8", "residual": False},
        # a full batch of prompts: memory traffic alone
        {"name": "norm prompts 8192", "op": "rmsnorm", "rows": 8192, "cols": 8192, "in": "bf16", "q": "e4m3", "residual": True},
        # --- 8-bit rows and scales of silu(gate) * up, gate and up side by side in one buffer
        # a decode batch between the two halves of a gated feed-forward block
        {"name": "gate 16 tokens", "op": "silu_mul", "rows": 16, "cols": 16384, "in": "bf16", "q": "e4m3"},
        # the same block on prompts
        {"name": "gate prompts 4096", "op": "silu_mul", "rows": 4096, "cols": 16384, "in": "bf16", "q": "e4m3"},
        # --- 8-bit rows and scales of a matrix as it is
        # one projection's weights, a scale for each output channel, from a master copy in 32 bits
        {"name": "quantise weights", "op": "plain", "rows": 8192, "cols": 8192, "in": "f32", "q": "e4m3", "pitch": 0},
        # attention outputs of a batch, a slice of a wider buffer, an odd width
        {"name": "quantise slice", "op": "plain", "rows": 2047, "cols": 4095, "in": "bf16", "q": "i8", "pitch": 6150},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["gemm", "gemm", "rmsnorm", "silu_mul", "plain"])
    if op == "gemm":
        m, n, k = _log_int(rng, 1, 8192), _log_int(rng, 64, 16384), _log_int(rng, 64, 16384)
        if rng.random() < 0.6:   # most layers are multiples of 64, some programs' are not
            n, k = -(-n // 64) * 64, -(-k // 64) * 64
        while m * n * k > 8192 ** 3:
            m = -(-m // 2)
        return {"op": op, "m": m, "n": n, "k": k, "out": rng.choice(["bf16", "f16", "f32"])}
    rows, cols = _log_int(rng, 1, 8192), _log_int(rng, 64, 32768)
    if rng.random() < 0.6:
        cols = -(-cols // 64) * 64
    while rows * cols > (1 << 25):
        rows = -(-rows // 2)
    c = {"op": op, "rows": rows, "cols": cols, "in": rng.choice(["bf16", "bf16", "f16", "f32"]), "q": rng.choice(["e4m3", "i8", "e5m2"])}
    if op == "rmsnorm":
        c["residual"] = rng.random() < 0.7
    if op == "plain":
        c["pitch"] = 0 if rng.random() < 0.5 else cols + rng.randrange(1, 4096)
    return c


# ---------------------------------------------------------------------------------- inputs
def _normal(g, *shape):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)


def _activations(g, rows, cols, spread=0.5):
    """Normal values with channels of different spread, as activations have."""
    return _normal(g, rows, cols).mul_(torch.exp(spread * _normal(g, 1, cols)))


def _int8_rows(x):
    scale = x.abs().amax(1).div_(127.0).clamp_(min=TINY)
    return x.div_(scale[:, None]).round_().to(torch.int8), scale


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case)
    if case["op"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        s["A"], s["scale_a"] = _int8_rows(_activations(g, m, k))
        s["B"], s["scale_b"] = _int8_rows(_normal(g, n, k).mul_(0.02))   # weights, one row per channel
        s["C"] = torch.empty((m, n), dtype=FLOATS[case["out"]], device=DEV)
        if own:
            from frisk_b200 import runtime as R, workloads as W
            s["plan"] = R.GemmPlan(m, n, k, W.I8, _code(W, case["out"]), transB=True, scales=True)
            s["workspace"] = torch.empty(s["plan"].workspace_bytes, dtype=torch.uint8, device=DEV) if s["plan"].workspace_bytes else None
        return s
    rows, cols, dt = case["rows"], case["cols"], FLOATS[case["in"]]
    s["q_out"] = torch.empty((rows, cols), dtype=EIGHT[case["q"]], device=DEV)
    s["scale"] = torch.empty((rows,), dtype=torch.float32, device=DEV)
    pitch = 0
    if case["op"] == "rmsnorm":
        s["x"] = _activations(g, rows, cols).to(dt)
        s["weight"] = _normal(g, cols).mul_(0.2).add_(1.0).to(dt)
        s["residual_in"] = _activations(g, rows, cols).mul_(4.0).to(dt) if case["residual"] else None
        s["sum"] = torch.empty((rows, cols), dtype=dt, device=DEV) if case["residual"] else None
    elif case["op"] == "silu_mul":
        s["x"] = _activations(g, rows, 2 * cols, 0.2).to(dt)
    else:
        pitch = case["pitch"]
        s["x"] = _activations(g, rows, pitch or cols).to(dt)[:, :cols]
    if own:
        from frisk_b200 import runtime as R, workloads as W
        s["desc"] = R.quant_desc(rows, cols, _code(W, case["in"]), _code(W, case["q"]), case["op"], eps=EPS, ldx=pitch)
    return s


def _code(W, name):
    return {"f32": W.F32, "f16": W.F16, "bf16": W.BF16, "i8": W.I8, "e4m3": W.E4M3, "e5m2": W.E5M2}[name]


# ---------------------------------------------------------------------------------- one pass
def _rows_in_8_bits(v, q):
    """The plain form of the 8-bit rows: v in 32 bits -> (q as stored, scales)."""
    scale = torch.clamp(v.abs().amax(1) / QMAX[q], min=TINY)
    r = torch.clamp(v / scale[:, None], -QMAX[q], QMAX[q])
    return (torch.round(r) if q == "i8" else r).to(EIGHT[q]), scale


def _values(q):
    """8-bit integers as numbers of a floating type that holds them exactly."""
    return q.to(torch.bfloat16) if q.dtype == torch.int8 else q


def run(s):
    if own:
        from frisk_b200 import runtime as R
        stream = torch.cuda.current_stream().cuda_stream
        if s["op"] == "gemm":
            s["plan"].run(s["A"], s["B"], s["C"], s["scale_a"], s["scale_b"], workspace=s["workspace"], stream=stream)
            return s["C"]
        if s["op"] == "rmsnorm":
            R.quant_run(s["desc"], s["x"], s["q_out"], s["scale"], weight=s["weight"], residual=s["residual_in"], sum_out=s["sum"], stream=stream)
            return {"q": _values(s["q_out"]), "scale": s["scale"], "sum": s["sum"]}
        R.quant_run(s["desc"], s["x"], s["q_out"], s["scale"], stream=stream)
        return {"q": _values(s["q_out"]), "scale": s["scale"]}
    if s["op"] == "gemm":
        # sums of products of 8-bit integers pass 2^24: 64 bits keep them whole
        acc = s["A"].double() @ s["B"].double().t()
        s["C"].copy_(acc * s["scale_a"].double()[:, None] * s["scale_b"].double())
        return s["C"]
    if s["op"] == "rmsnorm":
        h = s["x"].float()
        if s["residual_in"] is not None:
            h = h + s["residual_in"].float()
        n = h * torch.rsqrt(h.square().mean(1, keepdim=True) + EPS) * s["weight"].float()
        q, scale = _rows_in_8_bits(n, s["q"])
        return {"q": _values(q), "scale": scale, "sum": h.to(s["x"].dtype) if s["sum"] is not None else None}
    x = s["x"].float()
    if s["op"] == "silu_mul":
        gate, up = x[:, : s["cols"]], x[:, s["cols"]:]
        x = gate / (1.0 + torch.exp(-gate)) * up
    q, scale = _rows_in_8_bits(x, s["q"])
    return {"q": _values(q), "scale": scale}


# ---------------------------------------------------------------------------------- what it takes
def work(case):
    if case["op"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + m * n * SIZE[case["out"]] + 4 * (m + n), "flops": 2 * m * n * k}
    rows, cols, es = case["rows"], case["cols"], SIZE[case["in"]]
    e = rows * cols
    if case["op"] == "rmsnorm":
        return {"bytes": e * es * (3 if case["residual"] else 1) + cols * es + e + 4 * rows, "flops": 6 * e}
    if case["op"] == "silu_mul":
        return {"bytes": e * es * 2 + e + 4 * rows, "flops": 8 * e}
    return {"bytes": e * es + e + 4 * rows, "flops": 3 * e}


# ---------------------------------------------------------------------------------- in 64 bits
def _on_grid(v, q):
    """Nearest number of the 8-bit type to each of v (64 bits, |v| within the type's range), ties to even."""
    if q == "i8":
        return v.round()
    mantissa, least = (3, -6) if q == "e4m3" else (2, -14)
    exponent = torch.frexp(v)[1].to(torch.int64) - 1          # v = f * 2^exponent, 1 <= |f| < 2
    step = torch.ldexp(torch.ones_like(v), exponent.clamp(min=least) - mantissa)
    return (v / step).round() * step


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "gemm":
        # products of 512 terms at a time are whole in any order of a 32-bit sum (512 * 127^2 < 2^24)
        k, acc = case["k"], torch.zeros((case["m"], case["n"]), dtype=torch.float64, device=DEV)
        for k0 in range(0, k, 512):
            a, b = s["A"][:, k0:k0 + 512].float(), s["B"][:, k0:k0 + 512].float()
            acc += torch.einsum("mk,nk->mn", a, b)
        return acc.mul_(s["scale_a"].double().outer(s["scale_b"].double()))
    out = {"sum": None}
    v = s["x"].to(torch.float64)
    if case["op"] == "rmsnorm":
        if case["residual"]:
            v = v.add(s["residual_in"].to(torch.float64))
            out["sum"] = v
        rms = (torch.linalg.vector_norm(v, dim=1).square() / case["cols"] + EPS).sqrt()
        v = v / rms.unsqueeze(1) * s["weight"].to(torch.float64)
    elif case["op"] == "silu_mul":
        gate, up = v.chunk(2, dim=1)
        v = gate * torch.special.expit(gate) * up
    scale = torch.linalg.vector_norm(v, ord=float("inf"), dim=1) / QMAX[case["q"]]
    scale = torch.maximum(scale, torch.full_like(scale, TINY))
    out["q"] = _on_grid(v / scale.unsqueeze(1), case["q"])
    out["scale"] = scale
    return out if case["op"] == "rmsnorm" else {"q": out["q"], "scale": scale}
