"""The slope on the way out of a gradient of x is multiplied before the rounding, on the CPU SIMT emulation."""
import pytest
import torch

from dimo_amd import experts as ex
from tests import expert_emulation
from tests.expert_slope_cases import check_slope_rounds_once


@pytest.mark.parametrize("counts,K,N,dtype,act,tail", [
    ([70, 0, 5, 64], 40, 72, torch.bfloat16, "silu", 3), ([70, 0, 5, 64], 37, 65, torch.float16, "silu", 0),
    ([70, 0, 5, 64], 37, 65, torch.float16, "relu", 0), ([33, 20], 24, 40, torch.float32, "silu", 1),
    ([48 + i % 7 for i in range(128)], 104, 40, torch.bfloat16, "silu", 3)])
def test_slope_rounds_once(monkeypatch, counts, K, N, dtype, act, tail):
    expert_emulation.use(monkeypatch, ex)
    check_slope_rounds_once(ex, "cpu", counts, K, N, dtype, act, tail, seed=K)
