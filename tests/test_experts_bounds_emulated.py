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
