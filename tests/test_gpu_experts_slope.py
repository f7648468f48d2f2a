"""The slope on the way out of a gradient of x is multiplied before the rounding, on the GPU, every tile size."""
import pytest
import torch

from dimo_amd import experts as ex
from tests.expert_slope_cases import check_slope_rounds_once

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["relu", "silu"])
@pytest.mark.parametrize("counts,K,N,tail", [
    ([70, 0, 5, 64], 40, 72, 3), ([70, 0, 5, 64], 37, 65, 0), ([48 + i % 7 for i in range(128)], 104, 40, 3),
    ([48 + i % 7 for i in range(128)], 101, 40, 3), ([300, 0, 513, 128, 129, 256, 1, 700], 7200, 72, 130),
    ([1024] * 8, 1800, 136, 0)])
def test_slope_rounds_once(counts, K, N, dtype, act, tail):
    check_slope_rounds_once(ex, "cuda", counts, K, N, dtype, act, tail, seed=K)
