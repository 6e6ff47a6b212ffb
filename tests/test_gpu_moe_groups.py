"""GPU tests of the group-limited choice where f32 sums cannot decide it: the
definition's order in 64-bit arithmetic holds whatever the biases."""
import pytest
import torch

import gemm_sm100 as gs
from test_gpu_moe import SIGMOID, SOFTMAX, check_route, run_route

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("score", [SIGMOID, SOFTMAX])
@pytest.mark.parametrize("size,big", [(2, 100.0), (2, 30000.0), (5, 100.0), (32, 1000.0)])
def test_biases_that_cancel_within_a_group(handle, score, size, big):
    """A group's two best c are near big and -big: their sum is small, but each is rounded in steps of its own size."""
    gen = torch.Generator().manual_seed(size + int(big))
    t, groups = 3000, 2
    logits = torch.randn(t, size, generator=gen).repeat(1, groups)
    logits[:, size:] += torch.randn(t, size, generator=gen) * 4e-6   # nearly tied groups
    bias = torch.full((size,), -4 * big)
    bias[0], bias[-1] = big, -big
    bias = bias.repeat(groups)
    got = run_route(handle, logits, 2, score, bias, groups, 1, True)
    check_route(got, logits, 2, score, bias, groups, 1, True, 1.0, None, 1)
