"""The fp8 product for many tokens where a CTA pair has several tiles: what goes on from one to the next (rings, parities, scales fetched
ahead, output images) with fewer k blocks than the scales are fetched ahead and with more, odd and even numbers of them, ragged in every axis.

Every output is compared, against a 64-bit product on the device. Tolerances as in test_fp8_block_gpu.py.
"""

import pytest
import torch

import feather_ops_b200 as fo
from feather_ops_b200 import _lib
from oracle import fp8_block as ofb

pytestmark = pytest.mark.gpu

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
HALF = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


@pytest.fixture(autouse=True)
def every_wait_completed(cuda_device):
    yield
    assert _lib.read_status("feather_fp8_block_mm_status") == (0, 0)


def operands(m, width, depth, transposed, w_type=E4M3):
    g = torch.Generator(device="cuda").manual_seed(m + width + depth)
    rand = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    x = rand(m, depth) * torch.exp(0.5 * rand(depth)) * torch.exp(rand(m, 1))
    w = 0.02 * rand(depth, width) if transposed else 0.02 * rand(width, depth)
    return *fo.quantize_fp8_activation(x.bfloat16()), *fo.quantize_fp8_weight(w * torch.exp(rand(w.shape[0], 1)), w_type)


def check(out, q, s, w, ws, bias, transposed):
    ref, size = ofb.product(q, s, w, ws, bias, transposed)
    tol = ref.abs() * HALF[out.dtype] + size * (2.0**-16 + (s.shape[0] + 16) * 2.0**-24)
    off = (out.double() - ref).abs()
    assert (off <= tol).all(), (off > tol).nonzero()[:8]


# 2600 rows and 4112 outputs are 11 x 17 tiles, two or three for each of 74 pairs
@pytest.mark.parametrize("transposed", [False, True], ids=["forward", "backward"])
@pytest.mark.parametrize("depth", [112, 256, 272, 400, 656, 768, 896, 1040, 1280])
def test_tiles_of_a_pair_one_after_the_other(cuda_device, depth, transposed):
    m, width = 2600, 4112
    q, s, w, ws = operands(m, width, depth, transposed)
    room = torch.full(((m + 4) * width,), 77.0, device=cuda_device, dtype=torch.bfloat16)
    out = room[2 * width : (m + 2) * width].view(m, width)
    n, k = (depth, width) if transposed else (width, depth)
    stream = torch.cuda.current_stream().cuda_stream
    assert _lib.load().launch_fp8_block_mm(q.data_ptr(), s.data_ptr(), w.data_ptr(), ws.data_ptr(), None, out.data_ptr(), m, n, k, transposed, 0, 0, 1, stream)
    check(out, q, s, w, ws, None, transposed)
    assert (room[: 2 * width] == 77).all() and (room[(m + 2) * width :] == 77).all()
    assert torch.equal(fo.fp8_block_mm(q, s, w, ws, None, torch.bfloat16, transposed), out)
    # scales that are NaN: a row's, one of each tile row, in the last block of the contraction; no other row knows
    rows = torch.arange(5, m, 256, device=cuda_device)
    bad = s.clone()
    bad[-1, rows] = float("nan")
    got = fo.fp8_block_mm(q, bad, w, ws, None, torch.bfloat16, transposed)
    assert got[rows].isnan().all()
    keep = torch.ones(m, device=cuda_device, dtype=torch.bool)
    keep[rows] = False
    assert torch.equal(got[keep], out[keep])


@pytest.mark.parametrize("out_type", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("depth", [400, 1040])
def test_bias_and_types_over_several_tiles(cuda_device, depth, out_type):
    q, s, w, ws = operands(2570, 4368, depth, False, E5M2)
    bias = torch.randn(4368 + 1, device=cuda_device).to(out_type)[1:]   # on a two-byte boundary
    check(fo.fp8_block_mm(q, s, w, ws, bias, out_type), q, s, w, ws, bias, False)


# 34 and 67 tile rows in bands of 32: a full band and a short one, and two full ones
@pytest.mark.parametrize("transposed", [False, True], ids=["forward", "backward"])
@pytest.mark.parametrize("m", [8500, 17000])
def test_walk_in_bands(cuda_device, m, transposed):
    q, s, w, ws = operands(m, 1552, 4096, transposed)
    check(fo.fp8_block_mm(q, s, w, ws, None, torch.bfloat16, transposed), q, s, w, ws, None, transposed)


def test_the_same_bits_over_several_tiles(cuda_device):
    q, s, w, ws = operands(4000, 4112, 1296, False)
    first = fo.fp8_block_mm(q, s, w, ws)
    for _ in range(20):
        assert torch.equal(fo.fp8_block_mm(q, s, w, ws), first)
