"""Host side of the block-scaled fp8 operators: weight quantization, the oracle's gradients, argument checks without a device."""

import pytest
import torch

import feather_ops_b200 as fo
from oracle import fp8_block as ofb

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
@pytest.mark.parametrize("shape", [(16, 16), (128, 256), (272, 400), (1, 129)])
def test_weight_quantization(shape, dtype):
    w = 0.02 * torch.randn(*shape, generator=torch.Generator().manual_seed(1))
    w[: shape[0] // 2, : shape[1] // 2] *= 8
    q, s = fo.quantize_fp8_weight(w, dtype)
    assert q.shape == w.shape and q.is_contiguous() and s.shape == (-(-shape[0] // 128), -(-shape[1] // 128))
    for i in range(s.shape[0]):
        for j in range(s.shape[1]):
            block = w[128 * i : 128 * (i + 1), 128 * j : 128 * (j + 1)].double()
            scale = block.abs().max() / ofb.TOP[dtype]
            assert abs(s[i, j].double() - scale) <= 2**-23 * scale
            codes = q[128 * i : 128 * (i + 1), 128 * j : 128 * (j + 1)].double()
            assert ((codes - block / scale).abs() <= ofb.half_step(block / scale, dtype) * (1 + 2**-18)).all()
    assert torch.equal(fo.dequantize_fp8_weight(q, s).double(), ofb.weight_values(q, s).float().double())


def test_weight_of_zeros_and_refusals():
    q, s = fo.quantize_fp8_weight(torch.zeros(16, 32))
    assert torch.equal(fo.dequantize_fp8_weight(q, s), torch.zeros(16, 32))
    with pytest.raises(ValueError):
        fo.quantize_fp8_weight(torch.zeros(16))
    with pytest.raises(ValueError):
        fo.quantize_fp8_weight(torch.zeros(16, 16), torch.int8)
    with pytest.raises(ValueError):
        fo.dequantize_fp8_weight(q, torch.ones(2, 1))


def test_calls_that_are_refused_before_any_kernel():
    x, w = torch.zeros(4, 128, dtype=torch.bfloat16), torch.zeros(256, 128).to(E4M3)
    scale = torch.ones(2, 1)
    with pytest.raises(ValueError, match="features"):
        fo.fp8_block_linear(torch.zeros(4, 64, dtype=torch.bfloat16), w, scale)
    with pytest.raises(ValueError, match="features"):
        fo.fp8_block_dgrad(x, w, scale)
    with pytest.raises(ValueError, match="float8"):
        fo.quantize_fp8_activation(x, torch.int8)
    with pytest.raises(ValueError, match="output"):
        fo.fp8_block_mm(x.to(E4M3), torch.ones(1, 4), w, scale, None, torch.float32)
    with pytest.raises(ValueError, match="residual"):
        fo.rms_norm_quantize_fp8(x, torch.ones(128), x[:2])
    with pytest.raises(ValueError, match="shape"):
        fo.rms_norm_dgrad(x[:2], x, torch.ones(128), torch.ones(4))
    with pytest.raises(ValueError, match="grad_out"):
        fo.silu_mul_dgrad(x, x)
    with pytest.raises(NotImplementedError):   # no CPU path
        fo.quantize_fp8_activation(x)


def test_launchers_refuse_bad_arguments_without_a_device(lib):
    p = 1 << 20  # never dereferenced: every call below is refused
    assert not lib.launch_fp8_block_quantize(p, p, p, 4, 24, 0, 0, None)
    assert not lib.launch_fp8_block_quantize(p, p, p, -1, 32, 0, 0, None)
    assert not lib.launch_fp8_block_quantize(p + 2, p, p, 4, 32, 0, 0, None)
    assert not lib.launch_fp8_block_quantize(None, p, p, 4, 32, 0, 0, None)
    assert lib.launch_fp8_block_quantize(p, p, p, 0, 32, 0, 0, None)
    assert not lib.launch_fp8_block_mm(p, p, p, p, None, p, 4, 24, 32, False, 0, 0, 1, None)
    assert not lib.launch_fp8_block_mm(p, p, p, p, None, p, 4, 32, 24, False, 0, 0, 1, None)
    assert not lib.launch_fp8_block_mm(p, p, p, p, p, p, 4, 32, 32, True, 0, 0, 1, None)
    assert not lib.launch_fp8_block_mm(p, p, p, p, None, p, 4, 32, 32, False, 0, 0, 2, None)
    assert not lib.launch_fp8_block_mm(p, p, p + 8, p, None, p, 4, 32, 32, False, 0, 0, 1, None)
    assert not lib.launch_fp8_block_mm(p, None, p, p, None, p, 4, 32, 32, False, 0, 0, 1, None)
    assert not lib.launch_fp8_block_mm(p, p, p, p, None, p, 1 << 31, 32, 32, False, 0, 0, 1, None)
    assert lib.launch_fp8_block_mm(p, p, p, p, None, p, 0, 32, 32, False, 0, 0, 1, None)
    assert not lib.launch_rms_norm_fp8(p, p, p, None, p, p, p, 4, 32, 1e-6, 0, 0, 0, None)
    assert not lib.launch_rms_norm_fp8(p, None, p, None, p, p, p, 4, 32768 + 16, 1e-6, 0, 0, 0, None)
    assert not lib.launch_rms_norm_dgrad(p, p, p, p, None, p, p, p, 0, 32, 0, 0, None)
    assert not lib.launch_rms_norm_dgrad(p, p, p, p, p + 8, p, p, p, 4, 32, 0, 0, None)
    assert not lib.launch_silu_mul_fp8(p, p, p, 4, 8, 0, 0, None)
    assert not lib.launch_silu_mul_dgrad(p, p, None, 4, 16, 0, None)


def test_launchers_refuse_scales_off_their_alignment(lib):
    p = 1 << 20  # never dereferenced: every call below is refused
    assert not lib.launch_fp8_block_mm(p, p + 2, p, p, None, p, 4, 32, 32, False, 0, 0, 1, None)
    assert not lib.launch_fp8_block_mm(p, p, p, p + 1, None, p, 4, 32, 32, False, 0, 0, 1, None)
    assert not lib.launch_fp8_block_mm(p, p, p, p, p + 1, p, 4, 32, 32, False, 0, 0, 1, None)
    assert not lib.launch_fp8_block_linear(p, None, p, p + 2, None, p, 4, 32, 32, False, 0, 0, 0, 1, None)
    assert not lib.launch_fp8_block_linear(p, p + 8, p, p, None, p, 40, 32, 32, False, 0, 0, 0, 1, None)
    assert not lib.launch_fp8_block_linear(p, None, p, p, None, p, 40, 32, 32, False, 0, 0, 0, 1, None)
    assert not lib.launch_fp8_block_quantize(p, p, p + 2, 4, 32, 0, 0, None)
    assert not lib.launch_rms_norm_fp8(p, None, p, None, p, p + 2, p, 4, 32, 1e-6, 0, 0, 0, None)
    assert not lib.launch_rms_norm_fp8(p, None, p, None, p, p, p + 2, 4, 32, 1e-6, 0, 0, 0, None)
    assert not lib.launch_rms_norm_dgrad(p, p, p, p + 2, None, p, p, p, 4, 32, 0, 0, None)
    assert not lib.launch_rms_norm_dgrad(p, p, p, p, None, p, p + 4, p, 4, 32, 0, 0, None)


def test_scratch_of_the_norms_weight_gradient(lib):
    # few rows: none. Else a row of partials per CTA: two rows of the input each at least, and no more CTAs than the SMs hold
    for m, k, ctas in ((0, 272, 0), (1, 272, 0), (1024, 8192, 0), (512, 496, 0), (513, 496, 33), (1025, 4096, 296), (100, 16384, 50), (100000, 2048, 592), (100000, 4096, 296), (100000, 1296, 740), (100000, 5120, 444), (100000, 32768, 148), (100000, 8192, 148), (100000, 512, 592)):
        assert lib.feather_rms_norm_dgrad_partial_floats(m, k) == ctas * k


def test_norm_gradient_formula_against_differences():
    g = torch.Generator().manual_seed(2)
    x, w, grad = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((3, 32), (32,), (3, 32)))
    gx, gw, _, _ = ofb.rms_norm_grad(grad, x, w, ofb.rms_norm(x, w, 1e-6)[1])
    step = 1e-6

    def loss(x, w):
        return (ofb.rms_norm(x, w, 1e-6)[0] * grad).sum()

    for i in range(3):
        for j in (0, 7, 31):
            d = torch.zeros_like(x)
            d[i, j] = step
            # central differences: step^2 of curvature, 1e-16 / step of rounding
            assert abs((loss(x + d, w) - loss(x - d, w)) / (2 * step) - gx[i, j]) < 1e-7
    for j in (0, 7, 31):
        d = torch.zeros_like(w)
        d[j] = step
        assert abs((loss(x, w + d) - loss(x, w - d)) / (2 * step) - gw[j]) < 1e-7


def test_gate_gradient_formula_against_differences():
    g = torch.Generator().manual_seed(3)
    x, grad = torch.randn(2, 32, generator=g, dtype=torch.float64), torch.randn(2, 16, generator=g, dtype=torch.float64)
    ref = ofb.silu_mul_grad(grad, x)
    step = 1e-6
    for i in range(2):
        for j in (0, 5, 15, 16, 31):
            d = torch.zeros_like(x)
            d[i, j] = step
            assert abs(((ofb.silu_mul(x + d) - ofb.silu_mul(x - d)) * grad).sum() / (2 * step) - ref[i, j]) < 1e-7


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
def test_oracles_of_the_quantizer_agree(dtype):
    x = torch.randn(9, 272, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
    q, s = ofb.quantize_f32(x, dtype)
    codes, scale = ofb.quantize(x.double(), dtype)
    assert ((s.double() - scale).abs() <= 2**-23 * scale).all()
    assert ((q.double() - codes).abs() <= ofb.half_step(codes, dtype) * (1 + 2**-18)).all()


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
def test_the_documented_formula_gives_the_oracles_bits(dtype):
    """`quantize_f32` are the steps that the quantizer is tested against bit for bit on a device: what is documented has to be those."""
    import pathlib
    import re

    header = (pathlib.Path(__file__).resolve().parents[1] / "include" / "feather_ops_b200.h").read_text()
    x = torch.randn(64, 128, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16)
    q_ref, s_ref = ofb.quantize_f32(x, dtype)
    top = torch.tensor(ofb.TOP[dtype])
    names = {"t": x.float().abs().amax(1), "top": top, "fp8": lambda v: v.to(dtype)}
    for text in (fo.quantize_fp8_activation.__doc__, header[: header.index("launch_fp8_block_quantize(")]):
        scale = re.search(r"scale = ([^`,\n]*?)(?:`| and)", text)[1]
        code = re.search(r"\bq = (fp8\([^`,\n]*\))", text)[1].replace("x *", "x.float() *")
        assert torch.equal(eval(scale, dict(names)), s_ref[0])
        codes = [eval(code, names | {"x": x[i], "t": names["t"][i]}) for i in range(x.shape[0])]
        assert torch.equal(torch.stack([c.view(torch.uint8) for c in codes]), q_ref.view(torch.uint8))
