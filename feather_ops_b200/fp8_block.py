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
_ops = torch.ops.feather_ops
_TOP = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}
_LEAST_SCALE = 1e-30  # blocks of zeros get this scale: its inverse is finite, and so is its product with a weight's scale


def _top(dtype: torch.dtype) -> float:
    if dtype not in _TOP:
        raise ValueError(f"the codes must be float8_e4m3fn or float8_e5m2, got {dtype}")
    return _TOP[dtype]


def _is_e5m2(dtype: torch.dtype) -> bool:
    if dtype is torch.float8_e4m3fn:
        return False
    _top(dtype)
    return True


def _is_fp16(dtype: torch.dtype) -> bool:
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise ValueError(f"the output must be float16 or bfloat16, got {dtype}")
    return dtype is torch.float16


def _rows(x: torch.Tensor) -> torch.Tensor:
    return x if x.ndim == 2 else x.reshape(-1, x.shape[-1])


def _blocks(size: int) -> int:
    return -(-size // FP8_BLOCK)


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
    (at least `1e-30 * top`), `scale = t * (1 / top)` and `q = fp8(x * (top * (1 / t)))`, each step rounded to float32. Returns `(q [M, K], scale [ceil(K / 128), M])`."""
    return _ops.fp8_block_quantize.default(x, _is_e5m2(dtype))


def fp8_block_mm(a, a_scale, weight, weight_scale, bias=None, out_dtype=torch.bfloat16, transposed_b=False):
    """`A @ W^T + bias` (or `A @ W` with `transposed_b`) of fp8 codes with block scales, accumulated in float32 and rounded
    once. `a` `[M, K]` (`[M, N]`) with `a_scale` as `quantize_fp8_activation` gives them; `weight` `[N, K]` with
    `weight_scale`. Either side may be e4m3 or e5m2. `bias` (forward only) has `N` values of `out_dtype`."""
    return _ops.fp8_block_mm.default(a, a_scale, weight, weight_scale, bias, _is_fp16(out_dtype), transposed_b)


def _quantized_product(x, weight, weight_scale, bias, out_dtype, dtype, transposed_b):
    """Quantizer and product of `x` `[..., depth]` in one operator call: one launch up to 8 rows, else two."""
    out = _ops.fp8_block_linear.default(_rows(x), weight, weight_scale, bias, _is_fp16(out_dtype), transposed_b, _is_e5m2(dtype))
    return out if x.ndim == 2 else out.view(*x.shape[:-1], out.shape[1])


def fp8_block_linear(x, weight, weight_scale, bias=None, out_dtype=torch.bfloat16, dtype=torch.float8_e4m3fn):
    """Forward `x @ W^T + bias` of a 16-bit activation `[..., K]`: quantized to `dtype`, then the product. The bits are those of
    `quantize_fp8_activation` and `fp8_block_mm`."""
    if x.shape[-1] != weight.shape[1]:
        raise ValueError(f"activation has {x.shape[-1]} features, the weight {weight.shape[1]}")
    return _quantized_product(x, weight, weight_scale, bias, out_dtype, dtype, False)


def fp8_block_dgrad(grad_out, weight, weight_scale, out_dtype=torch.bfloat16, dtype=torch.float8_e4m3fn):
    """Input gradient `g @ W` of a 16-bit `[..., N]` gradient, quantized to `dtype` along its own rows: the weight's codes and
    block scales are those of the forward product."""
    if grad_out.shape[-1] != weight.shape[0]:
        raise ValueError(f"gradient has {grad_out.shape[-1]} features, the weight {weight.shape[0]}")
    return _quantized_product(grad_out, weight, weight_scale, None, out_dtype, dtype, True)


def rms_norm_quantize_fp8(x, weight, residual=None, eps=1e-6, dtype=torch.float8_e4m3fn):
    """Residual addition, RMS norm and quantization in one kernel: `h = x + residual` (rounded to x's dtype; `h = x` without
    a residual), `y = h / sqrt(mean(h^2) + eps) * weight`, and y's codes and block scales. `x` `[..., K]` fp16/bf16, `weight`
    `[K]` in x's dtype or float32, `K <= 32768`.

    Returns `(q [rows, K], scale [ceil(K / 128), rows], h, rstd [rows])`: `h` has x's shape and is x itself without a residual;
    `rstd` is what the backward pass needs."""
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"residual is {tuple(residual.shape)}, x {tuple(x.shape)}")
    rows = _rows(x)
    if residual is None:
        q, scale, rstd = _ops.rms_norm_fp8.default(rows, weight, eps, _is_e5m2(dtype))
        return q, scale, x, rstd
    q, scale, rstd, stream = _ops.add_rms_norm_fp8.default(rows, _rows(residual), weight, eps, _is_e5m2(dtype))
    return q, scale, stream.view(x.shape) if x.ndim != 2 else stream, rstd


def rms_norm_dgrad(grad_out, x, weight, rstd, grad_residual=None):
    """Backward pass of the norm: `x` is what it was taken of (`h` of `rms_norm_quantize_fp8`), `grad_out` the gradient of
    its output. `grad_residual`, the gradient that reaches `h` along the residual stream, is added in the same pass; the result
    is the gradient of both `x` and the residual of the forward call. Returns `(grad_x, grad_weight float32 [K])`."""
    if grad_out.shape != x.shape or (grad_residual is not None and grad_residual.shape != x.shape):
        raise ValueError("grad_out and grad_residual must have x's shape")
    if x.numel() == 0:
        return torch.empty_like(x), torch.zeros(x.shape[-1], device=x.device, dtype=torch.float32)
    grad_x, grad_weight = _ops.rms_norm_dgrad.default(_rows(grad_out), _rows(x), weight, rstd, None if grad_residual is None else _rows(grad_residual))
    return grad_x if x.ndim == 2 else grad_x.view(x.shape), grad_weight


def silu_mul_quantize_fp8(gate_up, dtype=torch.float8_e4m3fn):
    """Codes and block scales of `silu(gate) * up`, in one kernel. `gate_up` `[..., 2 F]` fp16/bf16 with the gate's columns
    first. Returns `(q [rows, F], scale [ceil(F / 128), rows])`."""
    return _ops.silu_mul_fp8.default(_rows(gate_up), _is_e5m2(dtype))


def silu_mul_dgrad(grad_out, gate_up):
    """Gradient of `gate_up` `[..., 2 F]` from `grad_out` `[..., F]`, the gradient of `silu(gate) * up`."""
    f = gate_up.shape[-1] // 2
    if grad_out.shape != (*gate_up.shape[:-1], f):
        raise ValueError(f"grad_out is {tuple(grad_out.shape)}, gate_up {tuple(gate_up.shape)}")
    out = _ops.silu_mul_dgrad.default(_rows(grad_out), _rows(gate_up))
    return out if gate_up.ndim == 2 else out.view(gate_up.shape)


# What a compiled caller has to know of the operators: the shapes and types of what they return.
def _fake_codes(rows, width, like, e5m2):
    dtype = torch.float8_e5m2 if e5m2 else torch.float8_e4m3fn
    return like.new_empty((rows, width), dtype=dtype), like.new_empty((_blocks(width), rows), dtype=torch.float32)


def _fake_out(rows, weight, like, out_fp16, transposed_b):
    return like.new_empty((rows, weight.shape[1 if transposed_b else 0]), dtype=torch.float16 if out_fp16 else torch.bfloat16)


@torch.library.register_fake("feather_ops::fp8_block_quantize")
def _(x, e5m2):
    return _fake_codes(x.shape[0], x.shape[1], x, e5m2)


@torch.library.register_fake("feather_ops::fp8_block_mm")
def _(a, a_scale, weight, weight_scale, bias, out_fp16, transposed_b):
    return _fake_out(a.shape[0], weight, a, out_fp16, transposed_b)


@torch.library.register_fake("feather_ops::fp8_block_linear")
def _(x, weight, weight_scale, bias, out_fp16, transposed_b, e5m2):
    return _fake_out(x.shape[0], weight, x, out_fp16, transposed_b)


@torch.library.register_fake("feather_ops::rms_norm_fp8")
def _(x, weight, eps, e5m2):
    return *_fake_codes(x.shape[0], x.shape[1], x, e5m2), x.new_empty((x.shape[0],), dtype=torch.float32)


@torch.library.register_fake("feather_ops::add_rms_norm_fp8")
def _(x, residual, weight, eps, e5m2):
    return *_fake_codes(x.shape[0], x.shape[1], x, e5m2), x.new_empty((x.shape[0],), dtype=torch.float32), torch.empty_like(x)


@torch.library.register_fake("feather_ops::rms_norm_dgrad")
def _(grad, x, weight, rstd, grad_residual):
    return torch.empty_like(x), x.new_empty((x.shape[1],), dtype=torch.float32)


@torch.library.register_fake("feather_ops::silu_mul_fp8")
def _(gate_up, e5m2):
    return _fake_codes(gate_up.shape[0], gate_up.shape[1] // 2, gate_up, e5m2)


@torch.library.register_fake("feather_ops::silu_mul_dgrad")
def _(grad, gate_up):
    return torch.empty_like(gate_up)
