"""The microscaled 4-bit kernels (dimo_amd/csrc/mx4.hip) on the CPU SIMT emulation, through dimo_amd/mx4.py, against a
float64 definition (tests/expert_cases.py); and what the entry points refuse."""
import pytest
import torch

from dimo_amd import experts as ex
from dimo_amd import mx4
from tests import expert_cases as cases
from tests import expert_emulation

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture
def emulated(monkeypatch):
    expert_emulation.use(monkeypatch, ex, mx4)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("R,K,kind,pad", [(1, 1, "normal", 0), (5, 32, "normal", 0), (7, 100, "normal", 4), (9, 77, "borders", 3),
                                          (40, 64, "range", 0), (4, 96, "special", 0)])
def test_quantize(emulated, R, K, dtype, kind, pad):
    cases.check_quantize(mx4, "cpu", R, K, dtype, kind, pad, seed=R + K)


@pytest.mark.parametrize("counts,K,N,dtype,act,bias,tail,grouped", [
    ([1], 1, 1, F32, None, True, 0, False),
    ([70], 96, 65, BF16, "relu", True, 0, False),
    ([33, 0, 66], 64, 40, F32, "silu", True, 3, True),
    ([0, 0], 32, 8, F16, None, False, 4, True),
    ([5, 130], 200, 72, BF16, None, False, 0, True),
])
def test_linear(emulated, counts, K, N, dtype, act, bias, tail, grouped):
    cases.check_mx4_linear(mx4, ex, "cpu", counts, K, N, dtype, act, bias, tail, grouped, seed=K)


def test_layer(emulated):
    cases.check_mx4_layer(mx4, ex, "cpu", 30, 2, 4, 72, 40)


def test_nan_block_makes_its_row_nan(emulated):
    x = torch.randn(3, 64)
    x[1, 40] = float("inf")
    y = mx4.mx4_linear(mx4.quantize_mx4(x), mx4.quantize_mx4(torch.randn(8, 64)), out_dtype=F32)
    assert torch.isnan(y[1]).all() and torch.isfinite(y[0]).all() and torch.isfinite(y[2]).all()


def test_no_rows(emulated):
    x = mx4.quantize_mx4(torch.zeros(0, 64))
    assert tuple(x.shape) == (0, 64)
    assert tuple(mx4.mx4_linear(x, mx4.quantize_mx4(torch.ones(8, 64))).shape) == (0, 8)


def test_no_cpu_path():
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        mx4.quantize_mx4(torch.zeros(4, 64))


def _m(*shape):
    return mx4.quantize_mx4(torch.zeros(*shape))


@pytest.mark.parametrize("call", [
    lambda: mx4.quantize_mx4(torch.zeros(4, 64, dtype=torch.float64)),
    lambda: mx4.quantize_mx4(torch.zeros(4, 0)),
    lambda: mx4.quantize_mx4(torch.zeros(5, 64), ex.group_rows(torch.zeros(4, 2, dtype=torch.int32), 3)),
    lambda: mx4.quantize_mx4(torch.zeros(4, 64), ex.RowGroups(torch.zeros(4, dtype=torch.int32))),
    lambda: mx4.MX4(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8), 64),
    lambda: mx4.MX4(torch.zeros(4, 32), torch.zeros(4, 2, dtype=torch.uint8), 64),
    lambda: mx4.MX4(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(3, 2, dtype=torch.uint8), 64),
    lambda: mx4.mx4_linear(_m(4, 64), _m(8, 32)),
    lambda: mx4.mx4_linear(_m(4, 64), _m(2, 8, 64)),
    lambda: mx4.mx4_linear(_m(4, 64), _m(2, 8, 64), groups=ex.RowGroups(torch.zeros(4, dtype=torch.int32))),
    lambda: mx4.mx4_linear(_m(4, 64), _m(8, 64), bias=torch.zeros(8)),
    lambda: mx4.mx4_linear(_m(4, 64), _m(8, 64), bias=torch.zeros(7, dtype=BF16)),
    lambda: mx4.mx4_linear(_m(4, 64), _m(8, 64), activation="tanh"),
    lambda: mx4.mx4_linear(_m(4, 64), _m(8, 64), out_dtype=torch.float64),
])
def test_bad_arguments(emulated, call):
    with pytest.raises(ValueError):
        call()


def test_c_entry_points_refuse_sizes():
    L, many = expert_emulation.emulated_library(), (1 << 30) + 1
    assert L.dimo_mx4_quantize(0, 4, many, 16, many, None, 16, 16, None) == -1
    assert L.dimo_mx4_dequantize(0, 4, many, 16, 16, 16, None) == -1
    for sizes in ((many, 1, 8, 8), (4, 1, many, 8), (4, 1, 8, many)):
        assert L.dimo_mx4_linear(0, *sizes, 16, 16, None, 16, 16, None, 0, 16, None) == -1


def test_c_entry_points_refuse():
    L = expert_emulation.emulated_library()
    assert L.dimo_mx4_quantize(0, 4, 0, 1, 8, None, 4, 1, None) == -1
    assert L.dimo_mx4_quantize(0, 4, 8, 1, 7, None, 4, 1, None) == -1
    assert L.dimo_mx4_quantize(0, 4, 8, 1, 8, None, 2, 1, None) == -1
    assert L.dimo_mx4_quantize(3, 4, 8, 1, 8, None, 4, 1, None) == -1
    assert L.dimo_mx4_dequantize(0, 4, 8, 4, 1, None, None) == -1
    assert L.dimo_mx4_linear(0, 4, 2, 32, 8, 16, 1, None, 16, 1, None, 0, 16, None) == -1
    assert L.dimo_mx4_linear(0, 4, 1, 32, 8, 8, 1, None, 16, 1, None, 0, 16, None) == -1
    assert L.dimo_mx4_linear(0, 4, 1, 32, 8, 16, 1, None, 16, 1, None, 3, 16, None) == -1
