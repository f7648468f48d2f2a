"""Bounds that the documentation of the expert operators states, on the CPU SIMT emulation."""
import pytest
import torch

from dimo_amd import experts as ex
from dimo_amd import mx4
from tests import expert_bounds_cases as cases
from tests import expert_emulation


@pytest.fixture
def emulated(monkeypatch):
    expert_emulation.use(monkeypatch, ex, mx4)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_4bit_error(emulated, dtype):
    cases.check_4bit_error(mx4, "cpu", dtype)


@pytest.mark.parametrize("rows", [30, 300])  # (the kernel for few rows, the tiles)
@pytest.mark.parametrize("scale", [2.0 ** -120, 2.0 ** -110, 2.0 ** -40, 1.0, 2.0 ** 120])
@pytest.mark.parametrize("seed", [0, 1])
def test_fp32_products(emulated, rows, scale, seed):
    cases.check_fp32_products(ex, "cpu", rows, scale, seed)


@pytest.mark.parametrize("rows", [30, 300])
def test_infinite_operands(emulated, rows):
    cases.check_infinite_operands(ex, "cpu", rows)
