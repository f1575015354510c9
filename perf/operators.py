"""Cases for the operators around the block-scaled e4m3 Linear: the product itself (one fp32 scale for each row and
128 columns of K of the activation, one for each 128 x 128 block of the weight), the residual addition + RMSNorm that
leaves its result as e4m3 rows with scales, and the quantisers that make both kinds of operand.

`own` chooses what `run` calls: the plain form (elementary torch operations in fp32, rounded once at the end) or this
package's HIP operators.  `exact` gives the values in 64 bits, before their rounding to the output's type."""
import math

import torch

own = False

BLOCK = 128          # columns of K (and rows of a weight) that share a scale
E4M3_MAX = 448.0
AMAX_FLOOR = 1e-12   # a group of zeros gets the scale 1e-12 / 448
EPS = 1e-6


# ---------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one token: the time projection of a denoising step, [1, 5120] -> the six modulation vectors
        {"name": "gemm 1x30720x5120", "op": "gemm", "m": 1, "n": 30720, "k": 5120, "epi": "none"},
        # a handful of rows: per-request embeddings served together
        {"name": "gemm 13x5120x4096", "op": "gemm", "m": 13, "n": 5120, "k": 4096, "epi": "gelu"},
        # the cross-attention keys and values of 512 text tokens, k | v as one product
        {"name": "gemm 512x10240x5120", "op": "gemm", "m": 512, "n": 10240, "k": 5120, "epi": "none"},
        # odd sizes: a last block of K of 48 columns, a last block of N of 8 rows
        {"name": "gemm 1000x2056x1456", "op": "gemm", "m": 1000, "n": 2056, "k": 1456, "epi": "gelu"},
        # first FFN product of the small video model at 480p, 81 frames
        {"name": "gemm 32760x8960x1536", "op": "gemm", "m": 32760, "n": 8960, "k": 1536, "epi": "gelu"},
        # second FFN product of the large one at 720p, gated and added to the residual stream
        {"name": "gemm 75600x5120x13824", "op": "gemm", "m": 75600, "n": 5120, "k": 13824, "epi": "residual"},
        # one token through a pre-norm
        {"name": "norm 1x5120 group", "op": "norm", "rows": 1, "dim": 5120, "stream": "bf16", "form": "group"},
        # a text encoder's 512 tokens, residual stream kept in fp32, one scale per row
        {"name": "norm 512x4096 row", "op": "norm", "rows": 512, "dim": 4096, "stream": "fp32", "form": "row"},
        # the full 720p sequence, operands of the block-scaled Linear out
        {"name": "norm 75600x5120 group", "op": "norm", "rows": 75600, "dim": 5120, "stream": "bf16", "form": "group"},
        # activations of the second FFN product: 257 image tokens, and the full 720p sequence
        {"name": "quant 257x1280", "op": "quant", "rows": 257, "dim": 1280, "block_rows": 1},
        {"name": "quant 75600x13824", "op": "quant", "rows": 75600, "dim": 13824, "block_rows": 1},
        # a checkpoint weight at load time, 128 x 128 blocks
        {"name": "quant weight 13824x5120", "op": "quant", "rows": 13824, "dim": 5120, "block_rows": BLOCK},
    ]


def _log_int(rng, lo, hi, step=1):
    return max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi)))) // step * step)


def draw(rng):
    op = rng.choice(["gemm", "gemm", "norm", "quant"])
    if op == "gemm":
        while True:
            m, n, k = _log_int(rng, 1, 75600), _log_int(rng, 64, 13824, 8), _log_int(rng, 128, 13824, 16)
            if m * n * k <= 75600 * 5120 * 13824:
                return {"op": op, "m": m, "n": n, "k": k, "epi": rng.choice(["none", "gelu", "residual"])}
    if op == "norm":
        return {"op": op, "rows": _log_int(rng, 1, 75600), "dim": _log_int(rng, 64, 5120, 8), "stream": rng.choice(["bf16", "fp32"]),
                "form": rng.choice(["bf16", "row", "group"])}
    if rng.random() < 0.7:
        return {"op": op, "rows": _log_int(rng, 1, 75600), "dim": _log_int(rng, 64, 13824, 8), "block_rows": 1}
    return {"op": op, "rows": _log_int(rng, 64, 13824, 8), "dim": _log_int(rng, 128, 13824, 16), "block_rows": BLOCK}


def work(case):
    if case["op"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        g = -(-k // BLOCK)
        b = m * k + n * k + 4 * (m * g + -(-n // BLOCK) * g) + 4 * n + 2 * m * n
        if case["epi"] == "residual":
            b += 2 * m * n + 4 * n
        return {"bytes": b, "flops": 2 * m * n * k}
    rows, dim = case["rows"], case["dim"]
    g = -(-dim // BLOCK)
    if case["op"] == "norm":
        stream = 2 if case["stream"] == "bf16" else 4
        out = {"bf16": 2 * rows * dim, "row": rows * dim + 4 * rows, "group": rows * dim + 4 * rows * g}[case["form"]]
        return {"bytes": 2 * stream * rows * dim + 2 * rows * dim + 4 * dim + out, "flops": 6 * rows * dim}
    return {"bytes": 3 * rows * dim + 4 * -(-rows // case["block_rows"]) * g, "flops": 3 * rows * dim}


# ---------------------------------------------------------------------------------------------- inputs
def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def _activation(gen, rows, cols):
    """Rows of an activation: unit variance, with some channels well above the rest, and their own level for each token."""
    x = _randn(gen, rows, cols)
    x *= torch.exp(0.5 * _randn(gen, 1, cols))
    x *= torch.exp(0.3 * _randn(gen, rows, 1))
    return x


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        # both operands as a program holds them before the product: e4m3 values with their scales.  The activation's
        # scales lie group after group ([groups, rows] in memory), the weight's as a checkpoint stores them.
        a, a_scale = _quantise(_activation(gen, m, k), 1)
        w, w_scale = _quantise(_randn(gen, n, k) * 0.02, BLOCK)
        s = {"a": a, "a_scale": a_scale.t().contiguous().t(), "w": w, "w_scale": w_scale.contiguous(), "bias": 0.02 * _randn(gen, n)}
        if case["epi"] == "residual":
            s["resid"] = _activation(gen, m, n).to(torch.bfloat16)
            s["gate"] = 0.1 * _randn(gen, n) + 0.3
    elif case["op"] == "norm":
        rows, dim = case["rows"], case["dim"]
        s = {"x": _activation(gen, rows, dim).to(torch.bfloat16 if case["stream"] == "bf16" else torch.float32),
             "y": (0.2 * _randn(gen, rows, dim)).to(torch.bfloat16),
             "weight": 1.0 + 0.1 * _randn(gen, dim)}
    elif case["block_rows"] == 1:
        s = {"x": _activation(gen, case["rows"], case["dim"]).to(torch.bfloat16)}
    else:
        s = {"x": (_randn(gen, case["rows"], case["dim"]) * 0.02).to(torch.bfloat16)}
    s["case"] = case
    return s


# ---------------------------------------------------------------------------------------------- plain form
def _blocks(x, block_rows):
    """[rows, cols] -> [row blocks, block_rows, groups, 128], zeros past the end."""
    rows, cols = x.shape
    x = torch.nn.functional.pad(x, (0, -cols % BLOCK, 0, -rows % block_rows))
    return x.view(x.shape[0] // block_rows, block_rows, x.shape[1] // BLOCK, BLOCK)


def _scale_of(amax):
    return amax.clamp(min=AMAX_FLOOR) / E4M3_MAX


def _quantise(x, block_rows):
    """fp32 [rows, cols] -> e4m3 [rows, cols] and the scale of each block of `block_rows` x 128."""
    rows, cols = x.shape
    b = _blocks(x, block_rows)
    scale = _scale_of(b.abs().amax(dim=(1, 3)))
    q = (b * scale.reciprocal()[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX)
    return q.reshape(b.shape[0] * block_rows, -1)[:rows, :cols].to(torch.float8_e4m3fn).contiguous(), scale


def _dequantise(q, scale, block_rows):
    rows, cols = q.shape
    b = _blocks(q.float(), block_rows) * scale[:, None, :, None]
    return b.view(b.shape[0] * block_rows, -1)[:rows, :cols]


def _gelu_tanh(v):
    return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))


def _plain_gemm(s):
    epi = s["case"]["epi"]
    v = _dequantise(s["a"], s["a_scale"], 1) @ _dequantise(s["w"], s["w_scale"], BLOCK).t() + s["bias"]
    if epi == "gelu":
        v = _gelu_tanh(v)
    elif epi == "residual":
        v = s["resid"].float() + v * s["gate"]
    return v.to(torch.bfloat16)


def _plain_norm(s):
    form = s["case"]["form"]
    h = s["x"].float() + s["y"].float()
    s["x"].copy_(h)  # the residual stream moves on in place
    v = h * torch.rsqrt(h.square().mean(dim=1, keepdim=True) + EPS) * s["weight"]
    if form == "bf16":
        return s["x"], v.to(torch.bfloat16)
    if form == "group":
        return (s["x"],) + _quantise(v, 1)
    scale = _scale_of(v.abs().amax(dim=1))
    return s["x"], (v * scale.reciprocal()[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale


# ---------------------------------------------------------------------------------------------- one pass
def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "gemm":
        return _plain_gemm(state)
    if op == "norm":
        return _plain_norm(state)
    return _quantise(state["x"].float(), state["case"]["block_rows"])


def _run_own(s):
    from lightx2v_amd import hip

    case = s["case"]
    if case["op"] == "gemm":
        if case["epi"] == "residual":
            return hip.gemm_fp8_block(s["a"], s["a_scale"], s["w"], s["w_scale"], s["bias"], epilogue=hip.EPI_RESIDUAL, resid=s["resid"], gate=s["gate"])
        return hip.gemm_fp8_block(s["a"], s["a_scale"], s["w"], s["w_scale"], s["bias"], epilogue=hip.EPI_GELU_TANH if case["epi"] == "gelu" else hip.EPI_NONE)
    if case["op"] == "norm":
        if case["form"] == "bf16":
            return s["x"], hip.add_rmsnorm_(s["x"], s["y"], s["weight"], eps=EPS)
        r = hip.add_rmsnorm_(s["x"], s["y"], s["weight"], eps=EPS, quant=case["form"])
        return s["x"], r.q, r.scale
    return hip.quant_fp8_group128(s["x"]) if case["block_rows"] == 1 else hip.quant_fp8_block128(s["x"])


# ---------------------------------------------------------------------------------------------- 64 bits
def _grid(scale, rows, cols, tall):
    """The scale of every element in 64 bits, from the scale of its block."""
    r = torch.arange(rows, device=scale.device) // (BLOCK if tall else 1)
    return scale.double()[r][:, torch.arange(cols, device=scale.device) // BLOCK]


def _exact_quant(v, tall):
    """v / scale in 64 bits (not rounded to e4m3) and the scales; `tall`: 128 x 128 blocks."""
    rows, cols = v.shape
    groups = -(-cols // BLOCK)
    a = torch.zeros(rows, groups * BLOCK, dtype=torch.float64, device=v.device)
    a[:, :cols] = v.abs()
    a = a.view(rows, groups, BLOCK).amax(dim=2)
    if tall:
        a = torch.stack([a[i:i + BLOCK].amax(dim=0) for i in range(0, rows, BLOCK)])
    scale = torch.clamp(a, min=AMAX_FLOOR) / E4M3_MAX
    return v / _grid(scale, rows, cols, tall), scale


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        w = s["w"].double() * _grid(s["w_scale"], n, k, True)
        out = torch.empty(m, n, dtype=torch.float64, device="cuda")
        for i in range(0, m, 8192):
            a = s["a"][i:i + 8192].double()
            a = a * _grid(s["a_scale"][i:i + 8192], a.shape[0], k, False)
            v = a @ w.t() + s["bias"].double()
            if case["epi"] == "gelu":
                v = v / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3)))
            elif case["epi"] == "residual":
                v = s["resid"][i:i + 8192].double() + s["gate"].double() * v
            out[i:i + 8192] = v
        return out
    if case["op"] == "quant":
        return _exact_quant(s["x"].double(), case["block_rows"] == BLOCK)
    h = s["x"].double() + s["y"].double()
    v = s["weight"].double() * h / torch.sqrt((h * h).sum(dim=1, keepdim=True) / case["dim"] + EPS)
    if case["form"] == "bf16":
        return h, v
    if case["form"] == "group":
        return (h,) + _exact_quant(v, False)
    scale = torch.clamp(v.abs().amax(dim=1), min=AMAX_FLOOR) / E4M3_MAX
    return h, v / scale[:, None], scale
