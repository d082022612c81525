"""Routing with biases at the ends of 32 bits: experts switched off by the type's lowest number, runs whose two best keys have no
sum in 32 bits."""
import math

import pytest
import torch

from alsparse_b200 import capi, spblas
from rows_util import choice64, gen, normal, ok

pytestmark = pytest.mark.gpu
LOWEST = torch.finfo(torch.float32).min
# experts, runs: runs that lanes hold whole, runs that go over lanes, more than 256 experts
SHAPES = [(256, 8), (64, 4), (96, 32), (60, 4), (250, 10), (220, 4), (512, 8), (300, 4), (1024, 32)]


def _check(score, logits, bias, groups, top_groups, k):
    index = torch.full((logits.shape[0], k), 77, dtype=torch.int32, device="cuda")
    weight = torch.empty(logits.shape[0], k, device="cuda")
    ok(spblas.route(score, logits, bias, groups, top_groups, False, 1.0, index, weight))
    assert torch.equal(index, choice64(logits, bias, score, groups, top_groups, k))
    return index


@pytest.mark.parametrize("score", [capi.SCORE_SIGMOID, capi.SCORE_SOFTMAX])
@pytest.mark.parametrize("experts,groups", SHAPES)
def test_a_run_switched_off_by_the_lowest_bias_comes_before_a_masked_one(score, experts, groups):
    each = experts // groups
    logits, bias = normal(gen(experts), 20, experts), torch.zeros(experts, device="cuda")
    logits[:, 1:each] = -math.inf              # the first run has one expert, the second nothing to choose
    logits[:, each:2 * each] = -math.inf
    bias[2 * each:] = LOWEST                   # all behind it are switched off, which leaves them behind the first
    bias[2 * each:] *= 1 - torch.arange(experts - 2 * each, device="cuda") % each * 2e-5  # ... one behind the other
    index = _check(score, logits, bias, groups, 2, min(each + 1, 4))
    assert bool((index >= 0).all()) and bool((index[:, 0] == 0).all()) and bool((index[:, 1:] >= 2 * each).all())


@pytest.mark.parametrize("score", [capi.SCORE_SIGMOID, capi.SCORE_SOFTMAX])
@pytest.mark.parametrize("experts,groups", SHAPES)
@pytest.mark.parametrize("sign", [1, -1])
def test_runs_whose_sums_pass_32_bits(score, experts, groups, sign):
    each = experts // groups
    logits, bias = normal(gen(experts), 20, experts), torch.zeros(experts, device="cuda")
    for i in range(groups):                    # of the same sign: each run's sum is beyond 32 bits, and the last is the best
        bias[i * each:(i + 1) * each] = sign * 3.4e38 * (0.6 + 0.4 * (i if sign > 0 else groups - 1 - i) / groups)
    bias *= 1 - torch.arange(experts, device="cuda") % each * 2e-5   # no two keys of a run alike
    index = _check(score, logits, bias, groups, 1, min(each, 4))
    assert bool((index >= (groups - 1) * each).all())
    bias[::3] = LOWEST
    _check(score, logits, bias, groups, max(1, groups // 2), min(each, 4))
    bias[1::3] = math.inf
    bias[2::5] = -math.inf
    _check(score, logits, bias, groups, max(1, groups // 2), min(each, 4))


@pytest.mark.parametrize("experts,groups", SHAPES)
def test_mixed_biases(experts, groups):
    g = gen(experts)
    for top in {1, 2, groups // 2, groups - 1}:
        logits = normal(g, 200, experts, by=2.0)
        logits[torch.rand(200, experts, generator=g, device="cuda") < 0.3] = -math.inf
        pick = torch.randint(0, 5, (experts,), generator=g, device="cuda")
        bias = torch.tensor([0.0, LOWEST, LOWEST / 2, 1e-3, LOWEST / 1.5], device="cuda")[pick]
        for score in (capi.SCORE_SIGMOID, capi.SCORE_SOFTMAX):
            _check(score, logits, bias, groups, top, min(6, top * (experts // groups)))
