"""feather_ops for B200: the quantized matmul family of woct0rdho/feather-ops on sm_100a.

Same Python surface as the reference package (`feather_ops/__init__.py:18-31` there): `scaled_mm_hip`,
the int8 ConvRot functions and the 3x3 conv, all running hand-written tcgen05 kernels through
`torch.ops.feather_ops.*`. Beside them, without a counterpart in the reference: block-scaled fp8 linears with the RMS norm
and the gate that write their inputs (`fp8_block`). Importing the package loads the native extension and fails loudly when it has
not been built: there is no CPU or eager fallback for the kernels.
"""

import sys

import torch  # noqa: F401  the extension links against libtorch, so torch has to be loaded first

# `python -m feather_ops_b200._build` imports this package before it runs the build script: that one entry gets through without
# the extension (an older one may lack operators that the modules below register for), everything else fails loudly.
_BUILDING = "feather_ops_b200._build" in getattr(sys, "orig_argv", [])

if not _BUILDING:
    try:
        from . import _C  # noqa: F401  registers torch.ops.feather_ops.{scaled_mm,int8_scaled_mm,convrot_quantize,conv2d_3x3,...}
    except ImportError as exc:  # pragma: no cover - depends on the build state
        raise ImportError(
            "feather_ops_b200._C is not built (or failed to load): run `python -m feather_ops_b200._build` "
            "(needs nvcc and g++, no GPU). The kernels have no fallback path."
        ) from exc

    from .conv2d import conv3x3_prepacked, prepack_conv2d_weight_3x3
    from .conv2d_module import Conv2d
    from .fp8_block import (
        dequantize_fp8_weight,
        fp8_block_dgrad,
        fp8_block_linear,
        fp8_block_mm,
        quantize_fp8_activation,
        quantize_fp8_weight,
        rms_norm_dgrad,
        rms_norm_quantize_fp8,
        silu_mul_dgrad,
        silu_mul_quantize_fp8,
    )
    from .int8_convrot import (
        convrot_int8_dgrad,
        convrot_int8_linear,
        dequantize_convrot_weight,
        int8_scaled_mm,
        int8_scaled_mm_plain,
        prepack_int8_weight,
        quantize_convrot_activation,
        quantize_convrot_weight,
        unpack_int8_weight,
    )
    from .scaled_mm import prepack_b_for_scaled_mm, scaled_mm_hip

    __all__ = [
        "Conv2d",
        "conv3x3_prepacked",
        "convrot_int8_dgrad",
        "convrot_int8_linear",
        "dequantize_convrot_weight",
        "dequantize_fp8_weight",
        "fp8_block_dgrad",
        "fp8_block_linear",
        "fp8_block_mm",
        "int8_scaled_mm",
        "int8_scaled_mm_plain",
        "prepack_b_for_scaled_mm",
        "prepack_conv2d_weight_3x3",
        "prepack_int8_weight",
        "quantize_convrot_activation",
        "quantize_convrot_weight",
        "quantize_fp8_activation",
        "quantize_fp8_weight",
        "rms_norm_dgrad",
        "rms_norm_quantize_fp8",
        "scaled_mm_hip",
        "silu_mul_dgrad",
        "silu_mul_quantize_fp8",
        "unpack_int8_weight",
    ]
