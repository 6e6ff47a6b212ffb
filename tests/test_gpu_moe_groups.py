"""GPU tests of the group-limited choice where f32 sums cannot decide it: the
definition's order in 64-bit arithmetic holds whatever the biases."""
import math

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


@pytest.mark.parametrize("score", [SIGMOID, SOFTMAX])
@pytest.mark.parametrize("pairs", [
    [(3e38, 1e38), (3e38, 2e38)],                          # both sums pass f32's range
    [(-3e38, -2e38), (-3e38, -1e38)],                      # and below it
    [(-3e38, -2e38), (-3e38, -1e38), (-3e38, -3e38)],
    [(1.0, 0.0), (3e38, 1e38), (3e38, 3e38), (2.0, 2.0)],
    [(math.inf, 0.0), (math.inf, 1e38), (math.inf, math.inf)],  # ties: the lowest
    [(-math.inf, -3e38), (-3e38, -3e38), (-math.inf, -math.inf)],
])
@pytest.mark.parametrize("t", [9, 200])
def test_sums_beyond_f32(handle, score, pairs, t):
    """Finite biases whose sum overflows f32 decide by the sum; infinite ones tie."""
    gen = torch.Generator().manual_seed(len(pairs) + t)
    bias = torch.tensor([b for p in pairs for b in p])
    logits = torch.randn(t, len(bias), generator=gen)
    for top_groups in range(1, len(pairs)):
        got = run_route(handle, logits, 2, score, bias, len(pairs), top_groups, True)
        check_route(got, logits, 2, score, bias, len(pairs), top_groups, True, 1.0, None, 1)
