"""What is measured of the 8-bit block-scaled linear layers and of the operators around them.

A decoder block's feed-forward half in 8-bit floating point is
`residual add + RMS norm -> fp8`, `fp8 x fp8 product`, `silu(gate) * up -> fp8`, `fp8 x fp8 product`, and backwards the
products over the same weight, the gate's gradient and the norm's. An activation has one float32 scale for every 128
consecutive channels of a row, a weight one for every 128 x 128 block. `run` is one operator of that chain: in elementary
torch operations (`own` false), or as a user calls the framework (`own` true).

Kinds of case:
  linear     x [M, K] 16 bit -> [M, N]: quantize the activation, then the product with the weight [N, K]
  mm         the same product on an activation that is in 8 bits already (what the norm or the gate has written)
  dgrad      g [M, N] 16 bit -> [M, K]: quantize the gradient, then the product with the same weight, untransposed
  norm       x [M, K] (+ residual) -> fp8 codes, their scales, the new residual and 1 / rms
  norm_grad  the norm's backward pass: the gradient of its input (plus the one of the residual stream) and of its weight
  silu       [M, 2 F] -> fp8 codes of silu(gate) * up and their scales
  silu_grad  the gradient of [M, 2 F] from the gradient of silu(gate) * up
"""

import math

import torch

own = False

BLOCK = 128
EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
TOP = {"e4m3": 448.0, "e5m2": 57344.0}


def listed():
    return [
        # one token of one sequence being answered: the weight is read once and nothing else counts
        {"name": "linear_1tok", "kind": "linear", "M": 1, "N": 12288, "K": 4096, "type": "bf16", "out": "bf16", "code": "e4m3", "bias": False},
        # a small batch of sequences being answered, with a bias
        {"name": "linear_24tok", "kind": "linear", "M": 24, "N": 5120, "K": 5120, "type": "fp16", "out": "fp16", "code": "e4m3", "bias": True},
        # a short ragged prompt; neither axis of the weight is a multiple of 128
        {"name": "mm_ragged", "kind": "mm", "M": 777, "N": 3856, "K": 2576, "type": "bf16", "out": "bf16", "code": "e4m3", "bias": False},
        # a training step's or a long prompt's tokens through a gate-and-up projection
        {"name": "mm_large", "kind": "mm", "M": 8192, "N": 12288, "K": 4096, "type": "bf16", "out": "bf16", "code": "e4m3", "bias": False},
        # the gradient of a short batch, in the type with the wider range
        {"name": "dgrad_short", "kind": "dgrad", "M": 200, "N": 5120, "K": 1280, "type": "fp16", "out": "fp16", "code": "e5m2", "bias": False},
        # a training step's gradient through the same kind of projection
        {"name": "dgrad_large", "kind": "dgrad", "M": 4096, "N": 12288, "K": 4096, "type": "bf16", "out": "bf16", "code": "e4m3", "bias": False},
        # one token: the launch is what counts
        {"name": "norm_1tok", "kind": "norm", "M": 1, "K": 5120, "type": "fp16", "code": "e4m3", "residual": True},
        # a training step's tokens
        {"name": "norm_large", "kind": "norm", "M": 8192, "K": 4096, "type": "bf16", "code": "e4m3", "residual": True},
        # a short ragged batch's backward pass
        {"name": "norm_grad_ragged", "kind": "norm_grad", "M": 333, "K": 2576, "type": "fp16", "residual": False},
        # a training step's
        {"name": "norm_grad_large", "kind": "norm_grad", "M": 8192, "K": 4096, "type": "bf16", "residual": True},
        # the gate of a training step's tokens
        {"name": "silu_large", "kind": "silu", "M": 4096, "F": 12288, "type": "bf16", "code": "e4m3"},
        # its backward pass at a ragged batch
        {"name": "silu_grad_ragged", "kind": "silu_grad", "M": 1111, "F": 6160, "type": "bf16"},
    ]


def _log(rng, low, high, step):
    """A multiple of `step` in [low, high], spread over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high))) / step)) * step))


def draw(rng):
    kind = rng.choice(["linear", "mm", "dgrad", "norm", "norm_grad", "silu", "silu_grad"])
    case = {"kind": kind, "M": _log(rng, 1, 8192, 1), "type": rng.choice(["bf16", "fp16"])}
    if kind in ("linear", "mm", "dgrad"):
        case |= {"N": _log(rng, 512, 12288, 16), "K": _log(rng, 512, 4096, 16), "out": rng.choice(["bf16", "fp16"])}
        case |= {"code": rng.choice(["e4m3", "e4m3", "e5m2"]), "bias": kind != "dgrad" and rng.random() < 0.3}
    elif kind in ("norm", "norm_grad"):
        case |= {"K": _log(rng, 256, 8192, 16), "residual": rng.random() < 0.6}
        if kind == "norm":
            case["code"] = rng.choice(["e4m3", "e4m3", "e5m2"])
    else:
        case["F"] = _log(rng, 256, 12288, 16)
        if kind == "silu":
            case["code"] = rng.choice(["e4m3", "e4m3", "e5m2"])
    return case


# ---------------------------------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------------------------------
def _activation(g, rows, width, dtype, size=1.0):
    """Channels of unlike sizes, a few of them far out, and a padded batch's rows of zeros at the end."""
    x = torch.randn(rows, width, generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn(width, generator=g, device="cuda"))
    x[:, torch.randint(0, width, (max(1, width // 512),), generator=g, device="cuda")] *= 12.0
    x[rows - rows // 32 :] = 0
    return (x * size).to(dtype)


def _weight(g, n, k):
    """A weight in e4m3 with a scale for each 128 x 128 block."""
    w = 0.02 * torch.randn(n, k, generator=g, device="cuda")
    w *= torch.exp(0.3 * torch.randn(n, 1, generator=g, device="cuda"))
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    padded = torch.zeros(nb * BLOCK, kb * BLOCK, device="cuda")
    padded[:n, :k] = w
    scale = (padded.view(nb, BLOCK, kb, BLOCK).abs().amax((1, 3)) / 448.0).clamp(min=1e-30)
    q = (w / _spread(scale, n, k)).to(torch.float8_e4m3fn)
    return q, scale


def _spread(scale, n, k):
    """The weight's scales, one for each element."""
    return scale.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, m, dtype = case["kind"], case["M"], TYPES[case["type"]]
    s = {"case": case}
    if kind in ("linear", "mm", "dgrad"):
        n, k = case["N"], case["K"]
        s["w"], s["ws"] = _weight(g, n, k)
        s["bias"] = torch.randn(n, generator=g, device="cuda").to(TYPES[case["out"]]) if case["bias"] else None
        if kind == "dgrad":
            s["x"] = _activation(g, m, n, dtype, 1e-3)
        else:
            s["x"] = _activation(g, m, k, dtype)
        if kind == "mm":
            s["q"], s["s"] = _quantize(s.pop("x").float(), case["code"])
    elif kind in ("norm", "norm_grad"):
        k = case["K"]
        s["x"] = _activation(g, m, k, dtype)
        s["weight"] = (1 + 0.2 * torch.randn(k, generator=g, device="cuda")).to(dtype)
        s["residual"] = _activation(g, m, k, dtype, 3.0) if case["residual"] else None
        if kind == "norm_grad":
            s["grad"] = _activation(g, m, k, dtype, 1e-2)
            s["rstd"] = torch.rsqrt(s["x"].double().square().mean(1) + EPS).float()
            if s["residual"] is not None:  # here: the gradient that comes down the residual stream
                s["residual"] = _activation(g, m, k, dtype, 1e-2)
    else:
        f = case["F"]
        s["gate_up"] = _activation(g, m, 2 * f, dtype)
        if kind == "silu_grad":
            s["grad"] = _activation(g, m, f, dtype, 1e-2)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# The plain forms, in 32 bits
# ---------------------------------------------------------------------------------------------------------------------
def _quantize(x, code):
    """Codes [M, K] and scales [ceil(K / 128), M] of a float32 activation."""
    m, k = x.shape
    kb = -(-k // BLOCK)
    if k % BLOCK:
        padded = x.new_zeros(m, kb * BLOCK)
        padded[:, :k] = x
    else:
        padded = x
    blocks = padded.view(m, kb, BLOCK)
    top = blocks.abs().amax(2).clamp(min=1e-30 * TOP[code])
    # one inverse a block and a product an element: 16-bit inputs meet ties, and both sides have to see the same ones
    q = (blocks * (TOP[code] / top)[:, :, None]).view(m, kb * BLOCK)[:, :k].to(TYPES[code]).contiguous()
    return q, (top / TOP[code]).t().contiguous()


def _values(q, scale):
    """What an activation's codes stand for, float32."""
    m, k = q.shape
    return q.float() * scale.t().repeat_interleave(BLOCK, 1)[:, :k]


def _plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind in ("linear", "mm", "dgrad"):
        q, scale = (s["q"], s["s"]) if kind == "mm" else _quantize(s["x"].float(), case["code"])
        w = s["w"].float() * _spread(s["ws"], *s["w"].shape)
        out = _values(q, scale) @ (w if kind == "dgrad" else w.t())
        if s["bias"] is not None:
            out = out + s["bias"].float()
        return out.to(TYPES[case["out"]])
    if kind == "norm":
        h = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(s["x"].dtype)
        v = h.float()
        rstd = torch.rsqrt(v.square().mean(1) + EPS)
        q, scale = _quantize(v * rstd[:, None] * s["weight"].float(), case["code"])
        return q, scale, h, rstd
    if kind == "norm_grad":
        normed = s["x"].float() * s["rstd"][:, None]
        grad = s["grad"].float()
        inner = grad * s["weight"].float()
        gx = (inner - normed * (inner * normed).mean(1, keepdim=True)) * s["rstd"][:, None]
        if s["residual"] is not None:
            gx = gx + s["residual"].float()
        return gx.to(s["x"].dtype), (grad * normed).sum(0)
    f = case["F"]
    gate, up = s["gate_up"][:, :f].float(), s["gate_up"][:, f:].float()
    if kind == "silu":
        return _quantize(gate / (1 + torch.exp(-gate)) * up, case["code"])
    grad = s["grad"].float()
    sig = 1 / (1 + torch.exp(-gate))
    return torch.cat([grad * up * sig * (1 + gate * (1 - sig)), grad * gate * sig], 1).to(s["gate_up"].dtype)


# ---------------------------------------------------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------------------------------------------------
def _own(s):
    import feather_ops_b200 as fo

    case = s["case"]
    kind = case["kind"]
    if kind == "linear":
        return fo.fp8_block_linear(s["x"], s["w"], s["ws"], s["bias"], TYPES[case["out"]], TYPES[case["code"]])
    if kind == "mm":
        return fo.fp8_block_mm(s["q"], s["s"], s["w"], s["ws"], s["bias"], TYPES[case["out"]])
    if kind == "dgrad":
        return fo.fp8_block_dgrad(s["x"], s["w"], s["ws"], TYPES[case["out"]], TYPES[case["code"]])
    if kind == "norm":
        return fo.rms_norm_quantize_fp8(s["x"], s["weight"], s["residual"], EPS, TYPES[case["code"]])
    if kind == "norm_grad":
        return fo.rms_norm_dgrad(s["grad"], s["x"], s["weight"], s["rstd"], s["residual"])
    if kind == "silu":
        return fo.silu_mul_quantize_fp8(s["gate_up"], TYPES[case["code"]])
    return fo.silu_mul_dgrad(s["grad"], s["gate_up"])


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------------------------------
# What a pass cannot do without, and its result in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    kind, m = case["kind"], case["M"]
    if kind in ("linear", "mm", "dgrad"):
        n, k = case["N"], case["K"]
        depth, width = (n, k) if kind == "dgrad" else (k, n)
        weight = n * k + 4 * -(-n // BLOCK) * -(-k // BLOCK)
        act = m * depth + 4 * m * -(-depth // BLOCK) if kind == "mm" else 2 * m * depth
        return {"bytes": weight + act + 2 * m * width + (2 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    if kind == "norm":
        k = case["K"]
        streams = 3 if case["residual"] else 1  # x in; the residual in and out
        return {"bytes": m * k * (2 * streams + 1) + 4 * m * -(-k // BLOCK) + 4 * m + 2 * k, "flops": 8 * m * k}
    if kind == "norm_grad":
        k = case["K"]
        streams = 4 if case["residual"] else 3
        return {"bytes": 2 * m * k * streams + 4 * m + 6 * k, "flops": 10 * m * k}
    f = case["F"]
    if kind == "silu":
        return {"bytes": 5 * m * f + 4 * m * -(-f // BLOCK), "flops": 8 * m * f}
    return {"bytes": 10 * m * f, "flops": 14 * m * f}


def _round8(v, code):
    """The nearest value of the 8-bit type to a float64, ties to even."""
    digits, least = (3, -6) if code == "e4m3" else (2, -14)
    exponent = torch.frexp(v)[1] - 1
    step = torch.ldexp(torch.ones_like(v), exponent.clamp(min=least) - digits)
    return (torch.round(v / step) * step).clamp(-TOP[code], TOP[code])


def _blocks64(v, code):
    """float64 codes before their rounding, and the scales as [M, ceil(K / 128)]."""
    m, k = v.shape
    kb = -(-k // BLOCK)
    top = torch.stack([v[:, b * BLOCK : (b + 1) * BLOCK].abs().amax(1) for b in range(kb)], 1)
    scale = torch.clamp(top / TOP[code], min=1e-30)
    return v / torch.repeat_interleave(scale, BLOCK, dim=1)[:, :k], scale


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("linear", "mm", "dgrad"):
        n, k = case["N"], case["K"]
        if kind == "mm":
            codes, scale = s["q"].double(), s["s"].double().t()
        else:
            codes, scale = _blocks64(s["x"].double(), case["code"])
            codes = _round8(codes, case["code"])
        a = codes * torch.repeat_interleave(scale, BLOCK, dim=1)[:, : codes.shape[1]]
        row = torch.arange(n, device="cuda") // BLOCK
        col = torch.arange(k, device="cuda") // BLOCK
        w = s["w"].double() * s["ws"].double()[row][:, col]
        out = torch.mm(a, w if kind == "dgrad" else w.T)
        return out if s["bias"] is None else out + s["bias"].double()
    if kind == "norm":
        h = s["x"].double()
        if s["residual"] is not None:  # the stream is kept in the input's type, and the norm is of what is kept
            h = (h + s["residual"].double()).to(s["x"].dtype).double()
        rstd = 1 / torch.sqrt((h * h).sum(1) / h.shape[1] + EPS)
        codes, scale = _blocks64(h * rstd[:, None] * s["weight"].double(), case["code"])
        return codes, scale.t(), h, rstd
    if kind == "norm_grad":
        hat = s["x"].double() * s["rstd"].double()[:, None]
        g = s["grad"].double()
        wg = g * s["weight"].double()
        gx = s["rstd"].double()[:, None] * (wg - hat * (wg * hat).sum(1, keepdim=True) / hat.shape[1])
        return gx if s["residual"] is None else gx + s["residual"].double(), (g * hat).sum(0)
    f = case["F"]
    gate, up = s["gate_up"].double().split(f, 1)
    sig = torch.sigmoid(gate)
    if kind == "silu":
        codes, scale = _blocks64(gate * sig * up, case["code"])
        return codes, scale.t()
    g = s["grad"].double()
    return torch.cat([g * up * (sig + gate * sig * (1 - sig)), g * gate * sig], 1)
