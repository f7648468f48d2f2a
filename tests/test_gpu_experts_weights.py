"""The expert block's weights over the chosen and over all experts, on the GPU."""
import pytest
import torch

from dimo_amd import experts as ex
from dimo_amd import mx4
from tests import expert_weights_cases as cases

pytestmark = pytest.mark.gpu


def test_block_with_one_choice():
    cases.check_block_with_one_choice(ex, "cuda")


@pytest.mark.parametrize("T,K,F,E,k,dtype", [(0, 8, 8, 3, 2, torch.float32), (50, 24, 40, 4, 1, torch.float32),
                                             (700, 264, 136, 4, 2, torch.bfloat16), (33, 17, 9, 5, 5, torch.float16)])
def test_weights_over_all(T, K, F, E, k, dtype):
    cases.check_weights_over_all(ex, "cuda", T, K, F, E, k, dtype)


def test_quantized_block_with_one_choice():
    cases.check_quantized_block_with_one_choice(ex, mx4, "cuda")
