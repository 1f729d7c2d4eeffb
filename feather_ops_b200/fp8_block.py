"""Block-scaled fp8 linear layers: fp8 x fp8 products with a float32 scale per 128 channels, and the operators around them
that write their outputs in that form. No counterpart in the reference, whose fp8 weights have one scale and whose 8-bit
activations are int8 with one scale per row (`feather_ops/scaled_mm.py`, `feather_ops/int8_convrot.py`).

An activation `[M, K]` in 8 bits is a pair `(q, scale)`: `q` `[M, K]` codes (`float8_e4m3fn`, or `float8_e5m2` where range
counts more than precision, as for gradients) and `scale` `[ceil(K / 128), M]` float32, one for every 128 consecutive
channels of a row. A weight `[N, K]` has `weight_scale` `[ceil(N / 128), ceil(K / 128)]`, one for every 128 x 128 block, so the
same codes serve both directions:

    forward   C[M, N] = A[M, K] @ W[N, K]^T + bias
    backward  C[M, K] = A[M, N] @ W[N, K]      (`transposed_b=True`)

A feed-forward block, one sequence step or a training step:

    q, s, stream, rstd = rms_norm_quantize_fp8(x, norm_weight, residual)
    gate_up = fp8_block_mm(q, s, w_gate_up, w_gate_up_scale)
    q2, s2 = silu_mul_quantize_fp8(gate_up)
    y = fp8_block_mm(q2, s2, w_down, w_down_scale)

    d_hidden = fp8_block_dgrad(d_y, w_down, w_down_scale)
    d_gate_up = silu_mul_dgrad(d_hidden, gate_up)
    d_normed = fp8_block_dgrad(d_gate_up, w_gate_up, w_gate_up_scale)
    d_stream, d_norm_weight = rms_norm_dgrad(d_normed, stream, norm_weight, rstd, grad_residual=d_stream_after)

The 8-bit weights are frozen, as in the int8 path: there is a gradient for activations and for the norm's weight. The
gradients are those of the formulas without the rounding to 8 bits. A block that holds an infinity or a NaN reads back as
NaN. All sizes along a row are multiples of 16; matrices are contiguous and 16-byte aligned.
"""

import torch

FP8_BLOCK = 128
_TOP = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}
_LEAST_SCALE = 1e-30  # blocks of zeros get this scale: its inverse is finite, and so is its product with a weight's scale


def _top(dtype: torch.dtype) -> float:
    if dtype not in _TOP:
        raise ValueError(f"the codes must be float8_e4m3fn or float8_e5m2, got {dtype}")
    return _TOP[dtype]


def _blocks(size: int) -> int:
    return -(-size // FP8_BLOCK)


def _norm_partials(rows: int, width: int) -> int:
    """Floats of scratch for the norm's weight gradient (the rule of `feather_rms_norm_dgrad_partial_floats`)."""
    return min(-(-rows // 4), 296) * width


def _empty_codes(rows: int, width: int, dtype: torch.dtype, device) -> tuple[torch.Tensor, torch.Tensor]:
    _top(dtype)
    q = torch.empty((rows, width), device=device, dtype=dtype)
    return q, torch.empty((_blocks(width), rows), device=device, dtype=torch.float32)


def quantize_fp8_weight(weight: torch.Tensor, dtype: torch.dtype = torch.float8_e4m3fn) -> tuple[torch.Tensor, torch.Tensor]:
    """Offline weight quantization: `[N, K]` -> codes `[N, K]` and scales `[ceil(N / 128), ceil(K / 128)]` (absmax of a
    128 x 128 block over the type's largest value). Plain torch, on any device."""
    if weight.ndim != 2:
        raise ValueError(f"weight must be [N, K], got {tuple(weight.shape)}")
    top = _top(dtype)
    n, k = weight.shape
    nb, kb = _blocks(n), _blocks(k)
    padded = torch.nn.functional.pad(weight.float(), (0, kb * FP8_BLOCK - k, 0, nb * FP8_BLOCK - n)).view(nb, FP8_BLOCK, kb, FP8_BLOCK)
    absmax = padded.abs().amax(dim=(1, 3)).clamp(min=_LEAST_SCALE * top)
    codes = (padded * (top / absmax)[:, None, :, None]).view(nb * FP8_BLOCK, kb * FP8_BLOCK)[:n, :k]
    return codes.to(dtype).contiguous(), absmax / top


def dequantize_fp8_weight(q: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """`code * scale`, float32."""
    n, k = q.shape
    if tuple(scale.shape) != (_blocks(n), _blocks(k)):
        raise ValueError(f"a {n} x {k} weight has {_blocks(n)} x {_blocks(k)} block scales, got {tuple(scale.shape)}")
    return q.float() * scale.repeat_interleave(FP8_BLOCK, 0)[:n].repeat_interleave(FP8_BLOCK, 1)[:, :k]


def quantize_fp8_activation(x: torch.Tensor, dtype: torch.dtype = torch.float8_e4m3fn) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes and block scales of a `[M, K]` fp16/bf16 activation, in one kernel: with `t` the largest magnitude of a block
    (at least `1e-30 * top`), `scale = t / top` and `q = fp8(x * (top / t))`. Returns `(q [M, K], scale [ceil(K / 128), M])`."""
    q, scale = _empty_codes(x.shape[0], x.shape[1], dtype, x.device)
    torch.ops.feather_ops.fp8_block_quantize.default(x, q, scale)
    return q, scale


def fp8_block_mm(a, a_scale, weight, weight_scale, bias=None, out_dtype=torch.bfloat16, transposed_b=False):
    """`A @ W^T + bias` (or `A @ W` with `transposed_b`) of fp8 codes with block scales, accumulated in float32 and rounded
    once. `a` `[M, K]` (`[M, N]`) with `a_scale` as `quantize_fp8_activation` gives them; `weight` `[N, K]` with
    `weight_scale`. Either side may be e4m3 or e5m2. `bias` (forward only) has `N` values of `out_dtype`."""
    n, k = weight.shape
    out = torch.empty((a.shape[0], k if transposed_b else n), device=a.device, dtype=out_dtype)
    torch.ops.feather_ops.fp8_block_mm.default(a, a_scale, weight, weight_scale, bias, out, transposed_b)
    return out


def fp8_block_linear(x, weight, weight_scale, bias=None, out_dtype=torch.bfloat16, dtype=torch.float8_e4m3fn):
    """Forward `x @ W^T + bias` of a 16-bit activation `[..., K]`: quantized to `dtype`, then the product."""
    n, k = weight.shape
    if x.shape[-1] != k:
        raise ValueError(f"activation has {x.shape[-1]} features, the weight {k}")
    q, scale = quantize_fp8_activation(x.reshape(-1, k), dtype)
    return fp8_block_mm(q, scale, weight, weight_scale, bias, out_dtype).reshape(*x.shape[:-1], n)


def fp8_block_dgrad(grad_out, weight, weight_scale, out_dtype=torch.bfloat16, dtype=torch.float8_e4m3fn):
    """Input gradient `g @ W` of a 16-bit `[..., N]` gradient, quantized to `dtype` along its own rows: the weight's codes and
    block scales are those of the forward product."""
    n, k = weight.shape
    if grad_out.shape[-1] != n:
        raise ValueError(f"gradient has {grad_out.shape[-1]} features, the weight {n}")
    q, scale = quantize_fp8_activation(grad_out.reshape(-1, n), dtype)
    return fp8_block_mm(q, scale, weight, weight_scale, None, out_dtype, True).reshape(*grad_out.shape[:-1], k)


def rms_norm_quantize_fp8(x, weight, residual=None, eps=1e-6, dtype=torch.float8_e4m3fn):
    """Residual addition, RMS norm and quantization in one kernel: `h = x + residual` (rounded to x's dtype; `h = x` without
    a residual), `y = h / sqrt(mean(h^2) + eps) * weight`, and y's codes and block scales. `x` `[..., K]` fp16/bf16, `weight`
    `[K]` in x's dtype or float32, `K <= 32768`.

    Returns `(q [rows, K], scale [ceil(K / 128), rows], h, rstd [rows])`: `h` has x's shape and is x itself without a residual;
    `rstd` is what the backward pass needs."""
    k = x.shape[-1]
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"residual is {tuple(residual.shape)}, x {tuple(x.shape)}")
    rows = x.reshape(-1, k)
    q, scale = _empty_codes(rows.shape[0], k, dtype, x.device)
    rstd = torch.empty(rows.shape[0], device=x.device, dtype=torch.float32)
    if residual is None:
        torch.ops.feather_ops.rms_norm_fp8.default(rows, None, weight, None, q, scale, rstd, eps)
        return q, scale, x, rstd
    stream = torch.empty_like(rows)
    torch.ops.feather_ops.rms_norm_fp8.default(rows, residual.reshape(-1, k), weight, stream, q, scale, rstd, eps)
    return q, scale, stream.view(x.shape), rstd


def rms_norm_dgrad(grad_out, x, weight, rstd, grad_residual=None):
    """Backward pass of the norm: `x` is what it was taken of (`h` of `rms_norm_quantize_fp8`), `grad_out` the gradient of
    its output. `grad_residual`, the gradient that reaches `h` along the residual stream, is added in the same pass; the result
    is the gradient of both `x` and the residual of the forward call. Returns `(grad_x, grad_weight float32 [K])`."""
    k = x.shape[-1]
    if grad_out.shape != x.shape or (grad_residual is not None and grad_residual.shape != x.shape):
        raise ValueError("grad_out and grad_residual must have x's shape")
    rows = x.reshape(-1, k)
    m = rows.shape[0]
    grad_x = torch.empty_like(rows)
    if m == 0:
        return grad_x.view(x.shape), torch.zeros(k, device=x.device, dtype=torch.float32)
    grad_weight = torch.empty(k, device=x.device, dtype=torch.float32)
    partials = torch.empty(_norm_partials(m, k), device=x.device, dtype=torch.float32)
    residual = None if grad_residual is None else grad_residual.reshape(-1, k)
    torch.ops.feather_ops.rms_norm_dgrad.default(grad_out.reshape(-1, k), rows, weight, rstd, residual, grad_x, grad_weight, partials)
    return grad_x.view(x.shape), grad_weight


def silu_mul_quantize_fp8(gate_up, dtype=torch.float8_e4m3fn):
    """Codes and block scales of `silu(gate) * up`, in one kernel. `gate_up` `[..., 2 F]` fp16/bf16 with the gate's columns
    first. Returns `(q [rows, F], scale [ceil(F / 128), rows])`."""
    rows = gate_up.reshape(-1, gate_up.shape[-1])
    q, scale = _empty_codes(rows.shape[0], rows.shape[1] // 2, dtype, gate_up.device)
    torch.ops.feather_ops.silu_mul_fp8.default(rows, q, scale)
    return q, scale


def silu_mul_dgrad(grad_out, gate_up):
    """Gradient of `gate_up` `[..., 2 F]` from `grad_out` `[..., F]`, the gradient of `silu(gate) * up`."""
    f = gate_up.shape[-1] // 2
    if grad_out.shape != (*gate_up.shape[:-1], f):
        raise ValueError(f"grad_out is {tuple(grad_out.shape)}, gate_up {tuple(gate_up.shape)}")
    rows = gate_up.reshape(-1, gate_up.shape[-1])
    out = torch.empty_like(rows)
    torch.ops.feather_ops.silu_mul_dgrad.default(grad_out.reshape(-1, f), rows, out)
    return out.view(gate_up.shape)


for _name in ("fp8_block_quantize", "fp8_block_mm", "rms_norm_fp8", "rms_norm_dgrad", "silu_mul_fp8", "silu_mul_dgrad"):
    # every operator writes into its arguments and returns nothing, which is all that a compiled caller has to know
    torch.library.register_fake(f"feather_ops::{_name}", lambda *args: None)
