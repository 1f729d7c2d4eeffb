"""64-bit definitions of the block-scaled fp8 operators, on the CPU, from their formulas (the reference has none of them).

`codes` come back before their rounding to 8 bits where a test has to say how far a code may be off: half a step of the
type at that value.
"""

import torch

BLOCK = 128
TOP = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}
# (half a step relative to the value, half a step of the smallest numbers)
HALF_STEP = {torch.float8_e4m3fn: (2.0**-4, 2.0**-10), torch.float8_e5m2: (2.0**-3, 2.0**-17)}


def half_step(value: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """How far the nearest 8-bit number may be from a float64 `value` within the type's range."""
    relative, least = HALF_STEP[dtype]
    return torch.clamp(value.abs() * relative, min=least)


def block_scales(y: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """`[ceil(K / 128), M]` float64 scales of a float64 `[M, K]`."""
    tops = [y[:, k : k + BLOCK].abs().amax(dim=1) for k in range(0, y.shape[1], BLOCK)]
    return torch.stack(tops).clamp(min=1e-30 * TOP[dtype]) / TOP[dtype]


def spread(scale: torch.Tensor, width: int) -> torch.Tensor:
    """The scale of every element, `[M, width]`."""
    return scale.t().repeat_interleave(BLOCK, 1)[:, :width]


def quantize(y: torch.Tensor, dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    """float64 codes before rounding, and scales."""
    scale = block_scales(y, dtype)
    return y / spread(scale, y.shape[1]), scale


def quantize_f32(x: torch.Tensor, dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    """The quantizer's own float32 steps: a reciprocal and two products per block, one product per element, one rounding."""
    m, k = x.shape
    kb = -(-k // BLOCK)
    padded = torch.zeros(m, kb * BLOCK)
    padded[:, :k] = x.float()
    top = padded.view(m, kb, BLOCK).abs().amax(2).clamp(min=1e-30 * TOP[dtype])
    inverse = top.reciprocal() * TOP[dtype]
    q = (padded.view(m, kb, BLOCK) * inverse[:, :, None]).view(m, kb * BLOCK)[:, :k].to(dtype)
    return q, (top * torch.tensor(1 / TOP[dtype])).t().contiguous()


def weight_values(w: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    n, k = w.shape
    return w.double() * scale.double().repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]


def product(a, a_scale, w, w_scale, bias=None, transposed_b=False) -> tuple[torch.Tensor, torch.Tensor]:
    """`A @ W^T + bias` (or `A @ W`) and the sum of the magnitudes that went into every output."""
    av = a.double() * spread(a_scale.double(), a.shape[1])
    wv = weight_values(w, w_scale)
    wv = wv if transposed_b else wv.t()
    out, size = av @ wv, av.abs() @ wv.abs()
    if bias is not None:
        out, size = out + bias.double(), size + bias.double().abs()
    return out, size


def rms_norm(h: torch.Tensor, weight: torch.Tensor, eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    """`(y, rstd)` of a `[M, K]` row matrix."""
    rstd = (h.double().square().mean(1) + eps).rsqrt()
    return h.double() * rstd[:, None] * weight.double(), rstd


def rms_norm_grad(grad, x, weight, rstd, grad_residual=None):
    """`(grad_x, grad_weight)` with `rstd` as given, and the magnitudes behind both."""
    n = x.double() * rstd.double()[:, None]
    u = grad.double() * weight.double()
    mean = (u * n).mean(1, keepdim=True)
    gx = rstd.double()[:, None] * (u - n * mean)
    size = rstd.double()[:, None] * (u.abs() + n.abs() * (u * n).abs().mean(1, keepdim=True))
    if grad_residual is not None:
        gx, size = gx + grad_residual.double(), size + grad_residual.double().abs()
    each = grad.double() * n
    return gx, each.sum(0), size, each.abs().sum(0)


def silu_mul(gate_up: torch.Tensor) -> torch.Tensor:
    gate, up = gate_up.double().chunk(2, 1)
    return gate * torch.sigmoid(gate) * up


def silu_mul_grad(grad: torch.Tensor, gate_up: torch.Tensor) -> torch.Tensor:
    gate, up = gate_up.double().chunk(2, 1)
    s = torch.sigmoid(gate)
    return torch.cat([grad.double() * up * s * (1 + gate * (1 - s)), grad.double() * gate * s], 1)
