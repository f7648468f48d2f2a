"""The microscaled 4-bit operators (dimo_amd/mx4.py) on the GPU against a float64 definition (tests/expert_cases.py has the
checks and derives the tolerances)."""
import pytest
import torch

from tests import expert_cases as cases

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops():
    from dimo_amd import experts, mx4
    return mx4, experts


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("R,K,kind,pad", [(1, 1, "normal", 0), (5, 32, "normal", 0), (700, 100, "normal", 4), (901, 77, "borders", 3),
                                          (4000, 64, "range", 0), (4, 96, "special", 0), (1001, 1000, "normal", 0),
                                          (300, 2048, "borders", 8)])
def test_quantize(ops, R, K, dtype, kind, pad):
    cases.check_quantize(ops[0], "cuda", R, K, dtype, kind, pad, seed=R + K)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("counts,K,N,act,bias,tail,grouped", [
    ([1], 1, 1, None, True, 0, False),
    ([70], 96, 65, "relu", True, 0, False),
    ([33, 0, 66], 64, 40, "silu", True, 3, True),
    ([0, 0], 32, 8, None, False, 4, True),
    ([5, 130], 200, 72, None, False, 0, True),
    ([1, 0, 2, 1, 0, 4], 2048, 512, None, True, 0, True),
    ([300, 513, 0, 129], 512, 257, None, True, 5, True),
    ([1000], 1024, 640, "silu", True, 0, False),
    ([3], 4096, 1000, None, True, 0, False),
    ([300, 0, 513, 128, 129, 256, 1, 700], 520, 7200, None, True, 300, True),  # 256 x 256 tiles, their halves
    ([7, 0, 9], 288, 72, "silu", True, 0, True), ([7, 1, 9], 288, 72, "silu", True, 0, True),  # at the kernel for few rows's border
])
def test_linear(ops, counts, K, N, dtype, act, bias, tail, grouped):
    cases.check_mx4_linear(*ops, "cuda", counts, K, N, dtype, act, bias, tail, grouped, seed=K)


@pytest.mark.parametrize("T,k,E,K,F", [(1, 2, 8, 512, 256), (300, 2, 4, 72, 40), (200, 4, 16, 256, 512)])
def test_layer(ops, T, k, E, K, F):
    cases.check_mx4_layer(*ops, "cuda", T, k, E, K, F)


def test_offsets_beyond_32_bits(ops):
    """Rows whose values lie more than 2^31 behind their matrix' first, and whose codes lie more than 2^32 bytes behind:
    the same as those rows alone."""
    mx4, _ = ops
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(2_100_000, 4096, generator=g, device="cuda", dtype=torch.bfloat16)
    q, alone = mx4.quantize_mx4(x), mx4.quantize_mx4(x[-90:])
    assert torch.equal(q.codes[-90:], alone.codes) and torch.equal(q.scales[-90:], alone.scales)
    del x
    w = mx4.quantize_mx4(torch.randn(40, 4096, generator=g, device="cuda"))
    X, W = alone.dequantize().double().cpu(), w.dequantize().double().cpu()
    cases.near(mx4.mx4_linear(q, w)[-90:], X @ W.T, BF16, cases.product_slack(4096, X.abs() @ W.abs().T), "y")
    tail = mx4.MX4(q.codes[-90:], q.scales[-90:], 4096).dequantize(torch.bfloat16)
    assert torch.equal(q.dequantize(torch.bfloat16)[-90:], tail)


def test_nan_block_makes_its_row_nan(ops):
    mx4, _ = ops
    x = torch.randn(300, 256, device="cuda")
    x[1, 40] = float("inf")
    y = mx4.mx4_linear(mx4.quantize_mx4(x), mx4.quantize_mx4(torch.randn(136, 256, device="cuda")), out_dtype=F32)
    assert torch.isnan(y[1]).all() and torch.isfinite(y[0]).all() and torch.isfinite(y[2:]).all()
