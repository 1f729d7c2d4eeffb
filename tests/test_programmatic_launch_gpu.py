"""Calls behind a kernel that lets them start at once and writes one of their inputs late.

The results are those of the same call on inputs that were there long before, bit for bit, however late the kernel ahead is: a wait inside
the call's kernels has a limit of two seconds, which must not begin before the kernel ahead has finished.
"""

import threading

import pytest
import torch

import feather_ops_b200 as fo
from feather_ops_b200 import _lib

pytestmark = pytest.mark.gpu

SHORT, LONG = 1_000_000, 5_000_000_000   # SM clocks: half a millisecond, and 2.5 s at the highest clock


@pytest.fixture(autouse=True)
def every_wait_completed(cuda_device):
    yield
    for symbol in ("feather_fp8_block_mm_status", "feather_int8_mm_status"):
        assert _lib.read_status(symbol) == (0, 0)


def rand(*shape, seed=0, dtype=torch.bfloat16, size=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * size).to(dtype).cuda()


def late(call, tensors, which, cycles):
    """`call(*tensors)` with tensor `which` written right before it by a kernel that takes `cycles` to begin."""
    expected = call(*tensors)
    inputs = [t.clone() if isinstance(t, torch.Tensor) else t for t in tensors]
    value, target = tensors[which], inputs[which]
    target.view(torch.uint8).fill_(0x11)
    torch.cuda.synchronize()
    stream = torch.cuda.current_stream().cuda_stream
    assert _lib.load().feather_selftest_late_writer(value.data_ptr(), target.data_ptr(), target.numel() * target.element_size(), cycles, stream) == 0
    got = call(*inputs)
    torch.cuda.synchronize()
    for a, b in zip(*((r,) if isinstance(r, torch.Tensor) else r for r in (got, expected))):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def product(m, transposed=False):
    n, k = 528, 656
    w = fo.quantize_fp8_weight(rand(n, k, seed=1, dtype=torch.float32, size=0.02))
    a = fo.quantize_fp8_activation(rand(m, n if transposed else k, seed=2))
    bias = None if transposed else rand(n, seed=3)
    return (lambda *t: fo.fp8_block_mm(*t, torch.bfloat16, transposed)), (*a, *w, bias)


@pytest.mark.parametrize("which", range(5), ids=["codes", "scales", "weight", "weight scales", "bias"])
@pytest.mark.parametrize("m", [3, 20, 100, 300, 2600])
def test_product(cuda_device, m, which):
    late(*product(m), which, SHORT)


@pytest.mark.parametrize("which", range(4), ids=["codes", "scales", "weight", "weight scales"])
@pytest.mark.parametrize("m", [3, 20, 100, 300, 2600])
def test_product_backward(cuda_device, m, which):
    late(*product(m, True), which, SHORT)


@pytest.mark.parametrize("which", range(4), ids=["x", "weight", "weight scales", "bias"])
@pytest.mark.parametrize("m", [1, 8, 9, 300])
def test_linear(cuda_device, m, which):
    w = fo.quantize_fp8_weight(rand(528, 656, seed=1, dtype=torch.float32, size=0.02))
    late(fo.fp8_block_linear, (rand(m, 656, seed=2), *w, rand(528, seed=3)), which, SHORT)


@pytest.mark.parametrize("which", range(3), ids=["x", "weight", "residual"])
@pytest.mark.parametrize("m,weight_type", [(1, torch.bfloat16), (300, torch.float32), (2100, torch.bfloat16)])
def test_norm(cuda_device, m, weight_type, which):
    late(fo.rms_norm_quantize_fp8, (rand(m, 2064, seed=1), rand(2064, seed=2, dtype=weight_type), rand(m, 2064, seed=3)), which, SHORT)


@pytest.mark.parametrize("which", range(5), ids=["grad", "x", "weight", "rstd", "grad of the residual"])
@pytest.mark.parametrize("m,weight_type", [(1, torch.bfloat16), (300, torch.float32), (2100, torch.bfloat16)])
def test_norm_gradient(cuda_device, m, weight_type, which):
    rstd = rand(m, seed=4, dtype=torch.float32).abs()
    late(fo.rms_norm_dgrad, (rand(m, 2064, seed=1), rand(m, 2064, seed=2), rand(2064, seed=3, dtype=weight_type), rstd, rand(m, 2064, seed=5)), which, SHORT)


@pytest.mark.parametrize("m", [1, 300, 9000])
def test_quantizer_and_gate(cuda_device, m):
    late(fo.quantize_fp8_activation, (rand(m, 656, seed=1),), 0, SHORT)
    late(fo.silu_mul_quantize_fp8, (rand(m, 1312, seed=2),), 0, SHORT)
    for which in (0, 1):
        late(fo.silu_mul_dgrad, (rand(m, 656, seed=3), rand(m, 1312, seed=4)), which, SHORT)


def int8_product(plain):
    n, k, m = 528, 1024, 2600
    g = torch.Generator().manual_seed(1)
    a, w = (torch.randint(-127, 128, s, generator=g, dtype=torch.int8).cuda() for s in ((m, k), (n, k)))
    scale, column = (torch.rand(s, generator=g).cuda() for s in (m, n))
    call = fo.int8_scaled_mm_plain if plain else fo.int8_scaled_mm
    return call, (a, w if plain else fo.prepack_int8_weight(w), scale, column, rand(n, seed=2))


@pytest.mark.parametrize("which", range(5), ids=["codes", "weight", "scales", "column scales", "bias"])
@pytest.mark.parametrize("plain", [False, True], ids=["prepack", "plain"])
def test_int8_product(cuda_device, plain, which):
    late(*int8_product(plain), which, SHORT)


@pytest.mark.parametrize("m", [3, 20, 100, 2600])
def test_product_behind_a_kernel_of_some_seconds(cuda_device, m):
    late(*product(m), 0, LONG)


def test_linear_behind_a_kernel_of_some_seconds(cuda_device):
    w = fo.quantize_fp8_weight(rand(528, 656, seed=1, dtype=torch.float32, size=0.02))
    late(fo.fp8_block_linear, (rand(3, 656, seed=2), *w), 0, LONG)


@pytest.mark.parametrize("plain", [False, True], ids=["prepack", "plain"])
def test_int8_product_behind_a_kernel_of_some_seconds(cuda_device, plain):
    late(*int8_product(plain), 0, LONG)


@pytest.mark.parametrize("which", range(3), ids=["codes", "weight", "scales"])
@pytest.mark.parametrize("plain", [False, True], ids=["prepack", "plain"])
def test_int8_product_backward(cuda_device, plain, which):
    n, k, m = 528, 1024, 2600
    g = torch.Generator().manual_seed(3)
    a, w = (torch.randint(-127, 128, s, generator=g, dtype=torch.int8).cuda() for s in ((m, n), (n, k)))
    call = fo.int8_scaled_mm_plain if plain else fo.int8_scaled_mm
    late(lambda *t: call(*t, transposed_b=True), (a, w if plain else fo.prepack_int8_weight(w), torch.rand(m, generator=g).cuda()), which, SHORT)


def chain():
    """A function of two matrices that runs every operator that starts early, each behind another one."""
    w1, w2 = (fo.quantize_fp8_weight(rand(*s, seed=i, dtype=torch.float32, size=0.05)) for i, s in enumerate(((1056, 400), (400, 528))))
    norm_weight = rand(400, seed=4)

    def run(x, r):
        q, s, h, rstd = fo.rms_norm_quantize_fp8(x, norm_weight, r)
        gate_up = fo.fp8_block_mm(q, s, *w1)
        y = fo.fp8_block_mm(*fo.silu_mul_quantize_fp8(gate_up), *w2)
        d_gate_up = fo.silu_mul_dgrad(fo.fp8_block_dgrad(y, *w2), gate_up)
        return h, gate_up, y, d_gate_up, *fo.rms_norm_dgrad(fo.fp8_block_linear(d_gate_up[:, :400].contiguous(), *w1)[:, :400].contiguous(), h, norm_weight, rstd)

    return run, w1


@pytest.mark.parametrize("m", [1, 30, 300, 1200])
def test_captured_among_copies_fills_forks_and_joins(cuda_device, m):
    run, w = chain()
    x, r = rand(m, 400, seed=5), rand(m, 400, seed=6)
    expected, swapped = run(x, r), run(r, x)
    linear = fo.fp8_block_linear(x, *w)
    xs, rs = torch.zeros_like(x), torch.zeros_like(r)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        xs.copy_(x)
        rs.copy_(r)
        here = run(xs, rs)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            there = run(rs, xs)
        apart = fo.fp8_block_linear(xs, *w)
        torch.cuda.current_stream().wait_stream(side)
        joined = fo.fp8_block_linear(xs, *w)   # behind two kernels
        xs.zero_()
        zeros = fo.quantize_fp8_activation(xs)[0]
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((*here, *there, apart, joined), (*expected, *swapped, linear, linear)))
        assert not zeros.view(torch.uint8).any()


def test_from_several_threads(cuda_device):
    run, _ = chain()
    x, r = rand(300, 400, seed=5), rand(300, 400, seed=6)
    expected = run(x, r), run(r, x)
    torch.cuda.synchronize()
    same = {}

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            got = [run(*((x, r), (r, x))[i % 2]) for _ in range(20)]
        stream.synchronize()
        same[i] = all(torch.equal(a, b) for results in got for a, b in zip(results, expected[i % 2]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert same == dict.fromkeys(range(6), True)
