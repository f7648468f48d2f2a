"""The expert block's weights over the chosen and over all experts, on the CPU SIMT emulation."""
import pytest
import torch

from dimo_amd import experts as ex
from dimo_amd import mx4
from tests import expert_emulation
from tests import expert_weights_cases as cases


@pytest.fixture
def emulated(monkeypatch):
    expert_emulation.use(monkeypatch, ex, mx4)


def test_block_with_one_choice(emulated):
    cases.check_block_with_one_choice(ex, "cpu", T=30)


@pytest.mark.parametrize("T,K,F,E,k,dtype", [(0, 8, 8, 3, 2, torch.float32), (50, 24, 40, 4, 1, torch.float32),
                                             (50, 24, 40, 4, 2, torch.bfloat16), (33, 17, 9, 5, 5, torch.float16)])
def test_weights_over_all(emulated, T, K, F, E, k, dtype):
    cases.check_weights_over_all(ex, "cpu", T, K, F, E, k, dtype)


def test_quantized_block_with_one_choice(emulated):
    cases.check_quantized_block_with_one_choice(ex, mx4, "cpu", T=20)
