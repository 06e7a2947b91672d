"""The low-precision operators' measured cases: what they compute, on which sizes, in a plain form and through the package.

Three operators.  `quantize_i8` turns each column of a matrix (a token's activations, a channel's weights) into 8-bit
integers with a scale of its own.  `linear` is what a serving program does with it: the activations of this step
quantised, then `gemm_i8` on weights that were quantised when the model was loaded.  `newton_schulz` orthogonalises a
batch of update matrices, as an optimiser does once per step.

A case's `run` is the plain form in elementary torch operations, or, where `own` is true, the package's calls.
"""
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
EPS = 1e-7


def listed():
    return [
        # one token's activations before a projection: pure latency
        {"name": "quantize_1x4096_bf16", "op": "quantize_i8", "type": "bf16", "batch": 1, "cols": 1, "k": 4096},
        # a float weight matrix with odd sizes, quantised by channel when a model is loaded
        {"name": "quantize_5003x4097_f32", "op": "quantize_i8", "type": "f32", "batch": 1, "cols": 5003, "k": 4097},
        # one token through a square projection: the smallest call of a decoding loop
        {"name": "linear_t1_4096x4096_bf16", "op": "linear", "type": "bf16", "batch": 1, "cols": 1, "rows": 4096, "k": 4096},
        # sixteen sequences decoding side by side through a wide projection
        {"name": "linear_t16_16384x4096_bf16", "op": "linear", "type": "bf16", "batch": 1, "cols": 16, "rows": 16384, "k": 4096},
        # a batch of experts, each with its own share of the tokens
        {"name": "linear_b32_t96_1000x2048_f16", "op": "linear", "type": "f16", "batch": 32, "cols": 96, "rows": 1000, "k": 2048},
        # odd everything, float activations: no row but the first starts on a 16-byte boundary
        {"name": "linear_t777_4099x1003_f32", "op": "linear", "type": "f32", "batch": 1, "cols": 777, "rows": 4099, "k": 1003},
        # a long prompt through large square weights: the tensor pipe's case
        {"name": "linear_t8192_8192x8192_bf16", "op": "linear", "type": "bf16", "batch": 1, "cols": 8192, "rows": 8192, "k": 8192},
        # the heads of one layer, orthogonalised one by one: many small matrices
        {"name": "orthogonal_b64_128x128_bf16", "op": "newton_schulz", "type": "bf16", "batch": 64, "cols": 128, "rows": 128, "steps": 5},
        # the square projections of a layer
        {"name": "orthogonal_b4_1024x1024_bf16", "op": "newton_schulz", "type": "bf16", "batch": 4, "cols": 1024, "rows": 1024, "steps": 5},
        # odd sizes in float, taller than wide
        {"name": "orthogonal_1501x1000_f32", "op": "newton_schulz", "type": "f32", "batch": 1, "cols": 1000, "rows": 1501, "steps": 5},
        # two rectangular matrices held in half precision, wider than tall
        {"name": "orthogonal_b2_1024x4096_f16", "op": "newton_schulz", "type": "f16", "batch": 2, "cols": 4096, "rows": 1024, "steps": 5},
        # a large feed-forward projection
        {"name": "orthogonal_4096x16384_bf16", "op": "newton_schulz", "type": "bf16", "batch": 1, "cols": 4096, "rows": 16384, "steps": 5},
    ]


def _log_size(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    op = rng.choice(["quantize_i8", "linear", "linear", "newton_schulz", "newton_schulz"])
    kind = rng.choice(["f32", "f16", "bf16"])
    if op == "quantize_i8":
        case = {"op": op, "type": kind, "batch": rng.randint(1, 4), "cols": _log_size(rng, 1, 8192), "k": _log_size(rng, 16, 16384)}
        while case["batch"] * case["cols"] * case["k"] > 5003 * 4097:
            case["cols"] = max(1, case["cols"] // 2)
        return case
    if op == "linear":
        batch = rng.choice([1, 1, 1, _log_size(rng, 2, 32)])
        case = {"op": op, "type": kind, "batch": batch, "cols": _log_size(rng, 1, 8192), "rows": _log_size(rng, 64, 16384),
                "k": _log_size(rng, 64, 16384)}
        while case["batch"] * case["rows"] * case["k"] > 1 << 28:
            case["batch"], case["rows"] = (case["batch"] + 1) // 2, max(64, case["rows"] // 2)
        while case["batch"] * case["cols"] * case["rows"] * case["k"] > 1 << 38:
            case["cols"] = max(1, case["cols"] // 2)
        return case
    case = {"op": op, "type": kind, "batch": rng.choice([1, 1, _log_size(rng, 2, 64)]), "cols": _log_size(rng, 24, 4096),
            "rows": _log_size(rng, 24, 8192), "steps": rng.randint(3, 6)}
    while work(case)["flops"] > 5e11:
        case["batch"], case["rows"] = (case["batch"] + 1) // 2, max(24, case["rows"] * 3 // 4)
    return case


def work(case):
    es, batch = BYTES[case["type"]], case["batch"]
    if case["op"] == "quantize_i8":
        n = batch * case["cols"]
        return {"bytes": n * case["k"] * (es + 1) + 4 * n, "flops": 3 * n * case["k"]}
    if case["op"] == "linear":
        t, m, k = case["cols"], case["rows"], case["k"]
        return {"bytes": batch * (t * k * es + m * k + 4 * m + t * m * es), "flops": 2 * batch * t * m * k}
    p, q = sorted((case["cols"], case["rows"]))
    # a Gram matrix and its square have p(p+1)/2 different entries
    step = p * (p + 1) * q + p * (p + 1) * p + 2 * p * p * q
    return {"bytes": 2 * batch * p * q * es, "flops": batch * case["steps"] * step}


def _plain_quantize(x):
    """Whole numbers (as float) and scales, by rows of the last axis; a row without a finite non-zero scale gets zeros."""
    x = x.float()
    scale = x.abs().amax(-1) / 127.0
    usable = (scale > 0) & torch.isfinite(scale)
    q = torch.round(x / torch.where(usable, scale, torch.ones_like(scale)).unsqueeze(-1))
    q = torch.where(usable.unsqueeze(-1), q.clamp(-127, 127), torch.zeros_like(q))
    return q, scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)
    kind, batch = TYPES[case["type"]], case["batch"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    state = {"case": case}
    if case["op"] in ("quantize_i8", "linear"):
        x = normal(batch, case["cols"], case["k"])
        # activations after a norm: a few channels are much larger than the rest, and tokens differ in size
        wide = torch.rand(case["k"], generator=g, device="cuda") < 0.01
        x = x * torch.where(wide, 12.0, 1.0) * torch.exp(0.5 * normal(batch, case["cols"], 1))
        state["x"] = x.to(kind)
        state["q"] = torch.empty(x.shape, dtype=torch.int8, device="cuda")
        state["scale"] = torch.empty(x.shape[:2], dtype=torch.float32, device="cuda")
    if case["op"] == "linear":
        w = normal(batch, case["rows"], case["k"]) * case["k"] ** -0.5
        wq, ws = _plain_quantize(w)
        state["w"], state["w_scale"] = wq.to(torch.int8), ws
        state["y"] = torch.empty(batch, case["cols"], case["rows"], dtype=kind, device="cuda")
    if case["op"] == "newton_schulz":
        c, r = case["cols"], case["rows"]
        # a momentum buffer: a few strong directions over a floor of noise, small in absolute value
        rank = max(1, min(c, r) // 8)
        strong = torch.bmm(normal(batch, c, rank) * torch.linspace(1.0, 0.1, rank, device="cuda"), normal(batch, rank, r))
        state["g"] = (1e-3 * (strong * rank ** -0.5 + 0.5 * normal(batch, c, r))).to(kind)
        state["out"] = torch.empty_like(state["g"])
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    import batchlas_b200 as bl
    case = state["case"]
    if case["op"] == "newton_schulz":
        return bl.newton_schulz(state["g"], state["out"], steps=case["steps"], coefficients=COEFFICIENTS, eps=EPS)
    bl.quantize_i8(state["x"], state["q"], state["scale"])
    if case["op"] == "quantize_i8":
        return {"values": state["q"] * state["scale"].unsqueeze(-1), "scale": state["scale"]}
    return bl.gemm_i8(state["w"], state["q"], state["y"], state["w_scale"], state["scale"])


def _run_plain(state):
    case = state["case"]
    if case["op"] == "newton_schulz":
        g = state["g"].float()
        x = g / (g.square().sum((-2, -1), keepdim=True).sqrt() + EPS)
        tall = x.shape[-2] > x.shape[-1]
        if tall:
            x = x.transpose(-2, -1)
        a, b, c = COEFFICIENTS
        for _ in range(case["steps"]):
            gram = x @ x.transpose(-2, -1)
            x = a * x + (b * gram + c * (gram @ gram)) @ x
        if tall:
            x = x.transpose(-2, -1)
        return x.to(state["g"].dtype).contiguous()
    q, scale = _plain_quantize(state["x"])
    if case["op"] == "quantize_i8":
        return {"values": q * scale.unsqueeze(-1), "scale": scale}
    acc = q @ state["w"].float().transpose(-2, -1)
    return (acc * state["w_scale"].unsqueeze(-2) * scale.unsqueeze(-1)).to(TYPES[case["type"]])


def exact(case, seed):
    """The definitions in 64 bits.  The scale and the quotient of a quantised value are 32-bit numbers by definition
    (a value halfway between two steps is common, so the rounding it goes through is part of the operator); they
    are formed here in 64 bits and rounded to 32, everything else stays in 64."""
    with torch.no_grad():
        state = prepare(case, seed)
        if case["op"] == "newton_schulz":
            x = state["g"].double()
            norm = torch.linalg.vector_norm(x.flatten(1), dim=1)
            x = x / (norm + EPS)[:, None, None]
            a, b, c = (float(v) for v in COEFFICIENTS)
            one = torch.eye(min(x.shape[1:]), dtype=torch.float64, device=x.device)
            for _ in range(case["steps"]):
                if x.shape[1] <= x.shape[2]:
                    gram = torch.matmul(x, x.mT)
                    x = torch.matmul(a * one + torch.matmul(gram, b * one + c * gram), x)
                else:
                    gram = torch.matmul(x.mT, x)
                    x = torch.matmul(x, a * one + torch.matmul(gram, b * one + c * gram))
            return x
        x = state["x"].double()
        scale = (torch.maximum(x.amax(-1), -x.amin(-1)) / 127).to(torch.float32).double()
        divisor = torch.where(scale == 0, 1.0, scale)
        q = torch.round((x / divisor[..., None]).to(torch.float32).double()).clamp(-127, 127)
        q[scale == 0] = 0
        if case["op"] == "quantize_i8":
            return {"values": q * scale[..., None], "scale": scale}
        total = torch.einsum("btk,bmk->btm", q, state["w"].double())
        return total * state["w_scale"].double()[:, None, :] * scale[..., None]
