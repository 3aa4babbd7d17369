"""Workloads of the 8-bit layer operators: RMS norm (with the residual's addition and an 8-bit output), its gradient,
row-wise quantisation to 8 bits, and the product of 8-bit operands with a scale for each token and channel.

`run` computes a case either in its plain form (elementary torch operations in 32 bits, `own` false) or through this
repository's Calculator (`own` true). Matrices are torch tensors [rows, columns]; the columns are the fastest dimension.
Codes of an int8 output are whole numbers that the operator's definition fixes (each is the nearest whole number to the
32-bit quotient of the value and its row's step, ties to even), so they come back as they are, beside the steps; fp8
outputs come back as torch's fp8 type.
"""
import torch

own = False

EPS = 1e-5
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32, "int8": torch.int8, "fp8": torch.float8_e4m3fn}
#: largest magnitude of a code: int8 is used symmetrically, fp8 is 1-4-3 with exponent bias 7 (448 is its largest finite value)
TOP = {"int8": 127.0, "fp8": 448.0}
#: the sizes no drawn case goes beyond: elements of a norm or quantiser input, elements of a weight, multiply-adds of a product
MOST_ROWS_X_COLS, MOST_WEIGHT, MOST_MACS = 8192 * 8192, 28672 * 8192, 8192 ** 3


def listed():
    return [
        # ---- RMS norm
        # one token of a running answer: the norm in front of the next 8-bit product, latency is all that counts
        {"name": "norm int8 1x8192", "op": "norm", "rows": 1, "cols": 8192, "x": "bf16", "residual": "bf16", "gamma": "bf16", "out": "int8"},
        # a prompt of 8192 tokens: residual added, stream written back, 8-bit rows for the product
        {"name": "norm int8 8192x8192", "op": "norm", "rows": 8192, "cols": 8192, "x": "bf16", "residual": "bf16", "gamma": "bf16", "out": "int8"},
        # a ragged batch of a model whose width divides by nothing, fp8 rows
        {"name": "norm fp8 1537x4999", "op": "norm", "rows": 1537, "cols": 4999, "x": "bf16", "residual": "bf16", "gamma": "fp32", "out": "fp8"},
        # a training step's forward pass with the residual stream in 32 bits
        {"name": "norm bf16 16384x4096", "op": "norm", "rows": 16384, "cols": 4096, "x": "bf16", "residual": "fp32", "gamma": "fp32", "out": "bf16"},
        # ---- its gradient
        # a short batch of a narrow model
        {"name": "norm grad 200x1000", "op": "norm_grad", "rows": 200, "cols": 1000, "x": "bf16", "gamma": "fp32", "dsum": False},
        # a training step: 16384 tokens, the residual stream's gradient joined in
        {"name": "norm grad 16384x4096", "op": "norm_grad", "rows": 16384, "cols": 4096, "x": "bf16", "gamma": "fp32", "dsum": True},
        # ---- quantisation
        # the inner activations of an MLP projection of a 2048-token prompt, in front of the product back
        {"name": "quantize int8 2048x28672", "op": "quantize", "rows": 2048, "cols": 28672, "x": "bf16", "out": "int8", "transpose": False},
        # a weight stored with its output channels contiguous, laid out once for the 8-bit product
        {"name": "quantize int8 8192x8192 T", "op": "quantize", "rows": 8192, "cols": 8192, "x": "bf16", "out": "int8", "transpose": True},
        # ---- product
        # one token through a square projection: every weight is read once, nothing else matters
        {"name": "product int8 1x8192x8192", "op": "product", "m": 1, "n": 8192, "k": 8192, "type": "int8", "out": "bf16", "bias": False, "dense": False},
        # 37 running answers through the MLP projection: still bound by the weights
        {"name": "product int8 37x28672x8192", "op": "product", "m": 37, "n": 28672, "k": 8192, "type": "int8", "out": "bf16", "bias": False, "dense": False},
        # a prompt through a square projection: bound by the tensor cores
        {"name": "product int8 8192x8192x8192", "op": "product", "m": 8192, "n": 8192, "k": 8192, "type": "int8", "out": "bf16", "bias": False, "dense": False},
        # a ragged batch through a projection with odd sizes, fp8 operands, a bias, 32-bit result
        {"name": "product fp8 777x5001x4100", "op": "product", "m": 777, "n": 5001, "k": 4100, "type": "fp8", "out": "fp32", "bias": True, "dense": False},
    ]


def _spread(rng, low, high):
    """A whole number from low to high, spread over its logarithm; one in three is a multiple of 64 where there is room."""
    v = low * (high / low) ** rng.random()
    n = max(low, min(high, int(round(v))))
    return max(low, n // 64 * 64) if n >= 128 and rng.random() < 1 / 3 else n


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_grad", "quantize", "product", "product", "product"])
    if op == "product":
        while True:
            m, n, k = _spread(rng, 1, 8192), _spread(rng, 64, 28672), _spread(rng, 64, 28672)
            if n * k <= MOST_WEIGHT and m * n * k <= MOST_MACS:
                break
        return {"op": op, "m": m, "n": n, "k": k, "type": rng.choice(["int8", "int8", "fp8"]), "out": rng.choice(["bf16", "bf16", "fp32"]),
                "bias": rng.random() < 0.5, "dense": rng.random() < 0.25}
    while True:
        rows, cols = _spread(rng, 1, 16384), _spread(rng, 64, 28672)
        if rows * cols <= MOST_ROWS_X_COLS:
            break
    if op == "norm":
        return {"op": op, "rows": rows, "cols": cols, "x": rng.choice(["bf16", "bf16", "fp32"]), "residual": rng.choice(["none", "bf16", "fp32"]),
                "gamma": rng.choice(["bf16", "fp32"]), "out": rng.choice(["int8", "int8", "fp8", "bf16", "fp32"])}
    if op == "norm_grad":
        return {"op": op, "rows": rows, "cols": cols, "x": rng.choice(["bf16", "bf16", "fp32"]), "gamma": rng.choice(["bf16", "fp32"]), "dsum": rng.random() < 0.5}
    return {"op": op, "rows": rows, "cols": cols, "x": rng.choice(["bf16", "bf16", "fp32"]), "out": rng.choice(["int8", "int8", "fp8"]), "transpose": rng.random() < 0.5}


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    s = {"case": case, "kept": {}}
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        # rows 16 bytes apart, or one behind the other where the case says dense
        pitch = k if case["dense"] else -(-k // 16) * 16

        def codes(rows, spread):
            c = torch.zeros(rows, pitch, dtype=TYPES[case["type"]], device="cuda")
            v = normal(rows, k).mul_(spread)
            c[:, :k] = (v.round_().clamp_(-127, 127) if case["type"] == "int8" else v.clamp_(-448, 448)).to(c.dtype)
            return c[:, :k]

        # codes as a quantiser leaves them: a row's largest is near the end of the type's range, four spreads out
        s["x"], s["w"] = codes(m, TOP[case["type"]] / 4), codes(n, TOP[case["type"]] / 4)
        s["x_scale"] = normal(m).mul_(0.5).exp_().mul_(4 / TOP[case["type"]])
        s["w_scale"] = normal(n).mul_(0.25).exp_().mul_(0.08 / TOP[case["type"]])
        s["bias"] = normal(n) if case["bias"] else None
        s["out"] = torch.empty(m, n, dtype=TYPES[case["out"]], device="cuda")
        return s
    rows, cols = case["rows"], case["cols"]
    t = TYPES[case["x"]]
    # activations of a language model: channels of different spread, a few of them far out
    spread = torch.exp(0.5 * normal(cols))
    spread[:: max(1, cols // 5)] *= 20
    s["x"] = normal(rows, cols).mul_(spread).to(t)
    if case["op"] == "quantize":
        s["out"] = torch.empty((cols, rows) if case["transpose"] else (rows, cols), dtype=TYPES[case["out"]], device="cuda")
        s["scale"] = torch.empty(cols if case["transpose"] else rows, device="cuda")
        return s
    s["gamma"] = (1 + 0.3 * normal(cols)).to(TYPES[case["gamma"]])
    if case["op"] == "norm":
        if case["residual"] != "none":
            s["residual"] = (normal(rows, cols) * spread * 3).to(TYPES[case["residual"]])
            s["sum"] = torch.empty_like(s["residual"])
        s["out"] = torch.empty(rows, cols, dtype=TYPES[case["out"]], device="cuda")
        if case["out"] in TOP:
            s["scale"] = torch.empty(rows, device="cuda")
        return s
    s["dy"] = normal(rows, cols).to(t)
    s["dsum"] = normal(rows, cols).to(t) if case["dsum"] else None
    s["dx"] = torch.empty(rows, cols, dtype=t, device="cuda")
    s["dgamma"] = torch.empty(cols, device="cuda")
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _codes(v, kind):
    """(codes, steps) of the rows of v in 32 bits."""
    step = v.abs().amax(-1, keepdim=True)
    step = step / torch.full_like(step, TOP[kind])
    t = torch.where(step > 0, v / step, torch.zeros_like(v)).clamp(-TOP[kind], TOP[kind])
    return (t.round() if kind == "int8" else t).to(TYPES[kind]), step


def _plain(s):
    case, x = s["case"], s["x"].float()
    if case["op"] == "product":
        y = x @ s["w"].float().T * s["x_scale"][:, None] * s["w_scale"]
        return {"out": (y if s["bias"] is None else y + s["bias"]).to(TYPES[case["out"]])}
    if case["op"] == "quantize":
        codes, step = _codes(x.T.contiguous() if case["transpose"] else x, case["out"])
        return {"out": codes, "scale": step[:, 0]}
    gamma = s["gamma"].float()
    if case["op"] == "norm":
        got = {}
        if "residual" in s:
            got["sum"] = (x + s["residual"].float()).to(s["residual"].dtype)
            x = got["sum"].float()   # the norm sees the stream as it is kept
        inverse = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS)
        v = x * gamma
        if case["out"] not in TOP:
            return got | {"out": (v * inverse).to(TYPES[case["out"]])}
        codes, step = _codes(v, case["out"])
        return got | {"out": codes, "scale": (step * inverse)[:, 0]}
    inverse = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS)
    dy, unit = s["dy"].float(), x * inverse
    a = dy * gamma
    dx = (a - unit * (a * unit).mean(-1, keepdim=True)) * inverse
    if s["dsum"] is not None:
        dx = dx + s["dsum"].float()
    return {"dx": dx.to(s["x"].dtype), "dgamma": (dy * unit).sum(0)}


# ------------------------------------------------------------------------------------------------ this repository's calls
_calculator = None


def _own(s):
    global _calculator
    from intel_gaudi3_software_b200 import Calculator, abi

    if _calculator is None:
        _calculator = Calculator(device=torch.cuda.current_device())
    calc, case, kept = _calculator, s["case"], s["kept"]
    calc.set_stream(torch.cuda.current_stream().cuda_stream or abi.STREAM_LEGACY)
    if not kept:
        kinds = {torch.bfloat16: abi.BF16, torch.float32: abi.FP32, torch.int8: abi.INT8, torch.float8_e4m3fn: abi.FP8_143}
        for name, t in s.items():
            if isinstance(t, torch.Tensor):
                fp8 = {"fp_bias": 7, "inf_nan_mode": abi.INFNAN_MINIMAL} if t.dtype == torch.float8_e4m3fn else {}
                kept[name] = abi.make_tensor(t.data_ptr(), kinds[t.dtype], reversed(t.shape), reversed(t.stride()), mem_space=abi.MEM_DEVICE, **fp8)
    if case["op"] == "product":
        calc.scaled_gemm(kept["out"], kept["x"], kept["x_scale"], kept["w"], kept["w_scale"], bias=kept.get("bias"))
        return {"out": s["out"]}
    if case["op"] == "quantize":
        calc.quantize(kept["out"], kept["scale"], kept["x"], abi.OP_TRANS if case["transpose"] else abi.OP_MEMCPY)
        return {"out": s["out"], "scale": s["scale"]}
    if case["op"] == "norm":
        calc.rms_norm(kept["out"], kept["x"], kept["gamma"], EPS, residual=kept.get("residual"), sum=kept.get("sum"), scale=kept.get("scale"))
        return {name: s[name] for name in ("sum", "out", "scale") if name in s}
    calc.rms_norm_grad(kept["dx"], kept["dgamma"], kept["dy"], kept["x"], kept["gamma"], EPS, dsum=kept.get("dsum"))
    return {"dx": s["dx"], "dgamma": s["dgamma"]}


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = {"bf16": 2, "fp32": 4, "int8": 1, "fp8": 1, "none": 0}
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + m * n * size[case["out"]] + 4 * (m + n + n * case["bias"]), "flops": 2 * m * n * k}
    n = case["rows"] * case["cols"]
    if case["op"] == "quantize":
        return {"bytes": n * (size[case["x"]] + 1) + 4 * (case["cols"] if case["transpose"] else case["rows"]), "flops": 3 * n}
    gamma = case["cols"] * size[case["gamma"]]
    if case["op"] == "norm":
        eight = case["out"] in TOP
        # the stream is read and written, x read, the result written
        return {"bytes": n * (size[case["x"]] + 2 * size[case["residual"]] + size[case["out"]]) + gamma + 4 * case["rows"] * eight, "flops": (7 if eight else 5) * n}
    return {"bytes": n * size[case["x"]] * (4 if case["dsum"] else 3) + gamma + 4 * case["cols"], "flops": 10 * n}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """The formulas in 64 bits. The whole numbers of an int8 output have no value here; an fp8 output's is the quotient it rounds."""
    s = prepare(case, seed)
    x = s["x"].double()
    if case["op"] == "product":
        y = torch.einsum("mk,nk->mn", x * s["x_scale"].double().unsqueeze(1), s["w"].double() * s["w_scale"].double().unsqueeze(1))
        return {"out": y if s["bias"] is None else y + s["bias"].double().unsqueeze(0)}

    def eight(v):
        largest = v.abs().max(dim=1).values
        return (None if case["out"] == "int8" else v * (TOP[case["out"]] / largest).unsqueeze(1)), largest / TOP[case["out"]]

    if case["op"] == "quantize":
        codes, step = eight(x.t() if case["transpose"] else x)
        return {"out": codes, "scale": step}
    gamma, got = s["gamma"].double(), {}
    if case["op"] == "norm" and "residual" in s:
        got["sum"] = x + s["residual"].double()
        x = got["sum"].to(s["residual"].dtype).double()
    size = torch.linalg.vector_norm(x, dim=1, keepdim=True)
    rms = torch.sqrt(size ** 2 / case["cols"] + EPS)
    if case["op"] == "norm":
        if case["out"] not in TOP:
            return got | {"out": x / rms * gamma}
        codes, step = eight(x * gamma)
        return got | {"out": codes, "scale": step / rms.squeeze(1)}
    dy = s["dy"].double()
    d = dy * gamma
    dx = d / rms - x * torch.einsum("rc,rc->r", d, x).unsqueeze(1) / (case["cols"] * rms ** 3)
    return {"dx": dx if s["dsum"] is None else dx + s["dsum"].double(), "dgamma": torch.einsum("rc,rc->c", dy, x / rms)}
