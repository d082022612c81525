"""Routing against its definition in 64 bits: the choice exactly, weights and gradients within the roundings of 32 bits."""
import math

import pytest
import torch

from alsparse_b200 import capi, spblas
from rows_util import TYPES, U, assert_within, choice64, floor_of, gen, half_step, normal, ok, strided, untouched, weights64

pytestmark = pytest.mark.gpu
SIGMOID, SOFTMAX = capi.SCORE_SIGMOID, capi.SCORE_SOFTMAX


def _route(score, logits, bias, groups, top_groups, renorm, scale, k):
    index = torch.full((logits.shape[0], k), 77, dtype=torch.int32, device="cuda")
    weight = torch.full((logits.shape[0], k), 77.0, device="cuda")
    ok(spblas.route(score, logits, bias, groups, top_groups, renorm, scale, index, weight))
    return index, weight


def _bound(logits, k):
    """Relative error of a weight: the argument of exp rounds once (by the distance of the logit from the largest), exp itself is
    within two steps, the sum of positive terms adds one rounding per term of a lane and per step of the tree, the two
    quotients and the scale one each; numerator and denominator both."""
    x = logits.float()
    finite = torch.where(x.isfinite(), x, 0.0)
    spread = 2 * finite.abs().amax(1, keepdim=True).double().clamp(max=104)
    return U * (2 * spread + 16 + logits.shape[1] / 32 + 5 + k)


def _check(score, logits, bias, groups, top_groups, renorm, scale, k):
    index, weight = _route(score, logits, bias, groups, top_groups, renorm, scale, k)
    assert torch.equal(index, choice64(logits, bias, score, groups, top_groups, k))
    exact = weights64(logits, index, score, renorm, scale)
    assert_within(weight, exact, _bound(logits, k) * exact.abs() + 2.0 ** -126, "weight")
    return index, weight


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("score", [SIGMOID, SOFTMAX])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("tokens,experts,groups,top_groups,k", [(1, 1, 1, 1, 1), (1, 256, 8, 4, 8), (33, 60, 1, 1, 4), (500, 256, 8, 4, 8), (100, 64, 4, 1, 6), (77, 1024, 32, 5, 32),
                                                                (200, 96, 32, 3, 5), (50, 8, 8, 3, 3), (130, 130, 1, 1, 32), (64, 512, 1, 1, 10), (9, 30, 3, 3, 30)])
def test_route(dtype, score, biased, tokens, experts, groups, top_groups, k):
    g = gen(tokens + experts + k)
    logits = normal(g, tokens, experts, by=2.0)
    logits[torch.rand(tokens, experts, generator=g, device="cuda") < 0.05] = -math.inf
    if tokens > 3:
        logits[1], logits[2, 1:] = -math.inf, -math.inf
    logits = logits.to(dtype)
    bias = normal(g, experts, by=0.2) if biased else None
    for renorm in (False, True):
        _check(score, logits, bias, groups, top_groups, renorm, 2.5, k)


@pytest.mark.parametrize("experts,groups,top_groups", [(24, 1, 1), (40, 2, 1), (128, 4, 2), (160, 8, 4), (160, 5, 2), (192, 6, 2), (192, 32, 9), (220, 4, 1), (224, 7, 3), (250, 10, 4),
                                                       (256, 32, 8), (256, 2, 1), (300, 4, 2), (384, 8, 4), (768, 12, 5), (1000, 8, 3), (1024, 4, 2)])
def test_every_number_of_experts_a_lane(experts, groups, top_groups):
    g = gen(experts)
    for dtype in (torch.float32, torch.bfloat16):
        logits = normal(g, 300, experts, by=1.5)
        logits[torch.rand(300, experts, generator=g, device="cuda") < 0.1] = -math.inf
        logits[7, : experts // 2] = 0.25
        logits = logits.to(dtype)
        # rows that begin on 16-byte boundaries, and rows that do not
        for x in (logits, strided(logits, experts + 3, 1)[0]):
            for score in (SIGMOID, SOFTMAX):
                for bias in (None, normal(g, experts, by=0.2)):
                    _check(score, x, bias, groups, top_groups, True, 1.0, 6)
                    _check(score, x, bias, 1, 1, False, 1.0, 6)


@pytest.mark.parametrize("score", [SIGMOID, SOFTMAX])
@pytest.mark.parametrize("biased", [False, True])
def test_ties_go_to_the_lowest_index(score, biased):
    logits = torch.zeros(40, 96, device="cuda")
    logits[1:, 50] = 1.0
    logits[2:, 51] = 1.0
    logits[3:] = (logits[3:] + torch.arange(96, device="cuda") // 7).bfloat16().float()
    bias = torch.zeros(96, device="cuda") if biased else None
    index, _ = _check(score, logits, bias, 1, 1, True, 1.0, 8)
    assert index[0].tolist() == list(range(8)) and index[2].tolist() == [50, 51, 0, 1, 2, 3, 4, 5]
    _check(score, logits, bias, 8, 2, True, 1.0, 8)
    zeros = torch.zeros(1, 64, device="cuda")
    zeros[0, ::2] = -0.0
    index, _ = _route(score, zeros, None if bias is None else bias[:64], 1, 1, False, 1.0, 4)
    assert index[0].tolist() == [0, 1, 2, 3]


@pytest.mark.parametrize("score", [SIGMOID, SOFTMAX])
def test_keys_that_32_bits_cannot_tell_apart(score):
    """Logits and biases made so that neighbouring keys differ by far less than a step of 32 bits."""
    g = gen(3)
    tokens, experts = 300, 64
    logits = normal(g, tokens, experts)
    target = 1.0
    # the bias that lifts every score of token 0 to nearly the same key; the other tokens stay ordinary
    s = torch.sigmoid(logits.double()) if score == SIGMOID else torch.softmax(logits.double(), 1)
    bias = (target - s[0]).float()
    key = s[0] + bias.double()
    assert float(key.max() - key.min()) < 3e-7
    logits[100:200] = logits[0]
    logits[100:200, 5] += torch.linspace(-1e-6, 1e-6, 100, device="cuda")
    _check(score, logits, bias, 1, 1, True, 1.0, 8)
    _check(score, logits, bias, 8, 3, False, 1.0, 6)


@pytest.mark.parametrize("score", [SIGMOID, SOFTMAX])
@pytest.mark.parametrize("dtype", TYPES)
def test_extreme_logits(score, dtype):
    big = torch.finfo(dtype).max
    rows = [[-big] * 8, [big, -big, 0.0, 1.0, -1.0, 0.5, -math.inf, 2.0], [-math.inf] * 8, [-math.inf, -big] + [-math.inf] * 6,
            [-200.0, -201.0, -202.0, -150.0, -300.0, -250.0, -220.0, -210.0], [200.0, 201.0, 199.0, 150.0, 180.0, 90.0, 100.0, 120.0]]
    logits = torch.tensor(rows, device="cuda").to(dtype)
    # a bias lifts experts whose scores are far below: renormalised weights are shares of the chosen all the same
    bias = torch.tensor([0.0, 0.0, 5.0, 0.0, 5.0, 0.0, 0.0, 0.0], device="cuda")
    for b in (None, bias):
        for renorm in (True, False):
            index, weight = _check(score, logits, b, 1, 1, renorm, 1.0, 2)
            assert index[2].tolist() == [-1, -1] and weight[2].tolist() == [0.0, 0.0]
            assert index[3].tolist() == [1, -1] and weight[3, 1] == 0
            assert bool(weight.isfinite().all())
            if renorm:
                assert bool(((weight.sum(1) - 1).abs() < 1e-6)[[0, 1, 3, 4, 5]].all())


def test_nan_and_infinite_logits():
    logits = torch.zeros(4, 16, device="cuda")
    logits[0, 9], logits[1, 3], logits[2, 4], logits[2, 2] = math.nan, math.inf, math.inf, -math.inf
    logits[3, 5] = -math.nan
    index, weight = _route(SIGMOID, logits, None, 1, 1, False, 1.0, 3)
    assert index.tolist() == [[9, 0, 1], [3, 0, 1], [4, 0, 1], [5, 0, 1]]
    assert weight[0].isnan().tolist() == [True, False, False] and weight[1].tolist() == [1.0, 0.5, 0.5]
    index, weight = _route(SOFTMAX, logits, None, 1, 1, True, 1.0, 3)
    assert index.tolist() == [[9, 0, 1], [3, 0, 1], [4, 0, 1], [5, 0, 1]] and bool(weight[:3].isnan().all())
    index, weight = _route(SIGMOID, logits, torch.zeros(16, device="cuda"), 4, 2, False, 1.0, 3)
    assert index.tolist() == [[9, 0, 1], [3, 0, 1], [4, 0, 1], [5, 0, 1]]
    # a bias of minus infinity switches an expert off
    bias = torch.zeros(16, device="cuda")
    bias[:14] = -math.inf
    index, weight = _route(SIGMOID, torch.zeros(2, 16, device="cuda"), bias, 1, 1, True, 1.0, 4)
    assert index.tolist() == [[14, 15, -1, -1]] * 2 and weight.tolist() == [[0.5, 0.5, 0.0, 0.0]] * 2


def test_strided_operands():
    g = gen(5)
    plain = normal(g, 37, 100)
    logits, _ = strided(plain, 111, 3)
    index, si = strided(torch.zeros(37, 5, dtype=torch.int32, device="cuda"), 9, 1)
    weight, sw = strided(torch.zeros(37, 5, device="cuda"), 6, 1)
    bi, bw = si.clone(), sw.clone()
    ok(spblas.route(SOFTMAX, logits, None, 5, 2, False, 1.0, index, weight))
    i2, w2 = _route(SOFTMAX, plain, None, 5, 2, False, 1.0, 5)
    assert torch.equal(index, i2) and torch.equal(weight, w2)
    assert untouched(index, si, bi) and untouched(weight, sw, bw)
    dweight, _ = strided(normal(g, 37, 5), 8, 1)
    d, sd = strided(torch.zeros(37, 100, device="cuda"), 101, 1)
    bd = sd.clone()
    ok(spblas.route_grad(SOFTMAX, logits, index, False, 1.0, dweight, d))
    d2 = torch.empty(37, 100, device="cuda")
    ok(spblas.route_grad(SOFTMAX, plain, i2, False, 1.0, dweight.contiguous(), d2))
    assert torch.equal(d, d2) and untouched(d, sd, bd)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("score", [SIGMOID, SOFTMAX])
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("tokens,experts,k", [(1, 1, 1), (1, 256, 8), (33, 60, 4), (200, 256, 8), (40, 1000, 32)])
def test_gradient(dtype, score, renorm, tokens, experts, k):
    g = gen(tokens + experts)
    logits = normal(g, tokens, experts, by=2.0)
    logits[torch.rand(tokens, experts, generator=g, device="cuda") < 0.05] = -math.inf
    if tokens > 3:
        logits[1], logits[2, 1:] = -math.inf, -math.inf
    logits = logits.to(dtype)
    index, _ = _route(score, logits, None, 1, 1, renorm, 2.5, k)
    dweight = normal(g, tokens, k)
    dweight[index < 0] = math.nan  # never read into a result
    d = torch.full((tokens, experts), math.nan, dtype=dtype, device="cuda")
    ok(spblas.route_grad(score, logits, index, renorm, 2.5, dweight, d))
    x = torch.where(logits == -math.inf, -1e30, logits.double()).requires_grad_()
    clean = torch.where(index < 0, 0.0, dweight).double()
    # masked logits far below all others have the same gradient, none
    w = weights64(x, index, score, renorm, 2.5)
    exact = torch.autograd.grad((w * clean).sum(), x)[0]
    exact = torch.where(logits == -math.inf, 0.0, exact)
    # a difference of two sums, each off by the relative error of the weights, over the sizes of its terms
    size = 2.5 * clean.abs().sum(1, keepdim=True)
    bound = 4 * _bound(logits, k) * size + half_step(dtype) * exact.abs() + floor_of(dtype)
    assert_within(d, exact, bound, "gradient")


def test_gradient_against_differences():
    g = gen(21)
    for score in (SIGMOID, SOFTMAX):
        for renorm in (False, True):
            logits, direction, dweight = normal(g, 20, 40), normal(g, 20, 40), normal(g, 20, 6)
            index, _ = _route(score, logits, None, 1, 1, renorm, 1.0, 6)
            d = torch.empty_like(logits)
            ok(spblas.route_grad(score, logits, index, renorm, 1.0, dweight, d))
            h = 2.0 ** -6
            sides = []
            for s in (h, -h):
                # the choice is kept by a bias that lifts the chosen experts alone, token by token
                for t in range(20):
                    bias = torch.zeros(40, device="cuda")
                    bias[index[t].long()] = 100.0 - torch.arange(6, device="cuda", dtype=torch.float32) * 10
                    i, w = _route(score, (logits + s * direction)[t:t + 1].contiguous(), bias, 1, 1, renorm, 1.0, 6)
                    assert torch.equal(i[0], index[t])
                    sides.append((w[0].double() * dweight[t].double()).sum())
            up, down = torch.stack(sides[:20]), torch.stack(sides[20:])
            slope = (up - down) / (2 * h)
            # third derivatives of weights of at most 1 along the direction (softmax: below 8 |d|^3): h^2 / 6 of that, and the
            # rounding of weights over 2 h
            size = dweight.double().abs().sum(1)
            reach = direction.double().abs().amax(1)
            bound = size * (h * h / 6 * 8 * reach ** 3 + 40 * U / h) + 1e-6 * size
            assert_within((d.double() * direction.double()).sum(1), slope, bound, "directional derivative")


def test_gradient_of_bad_and_repeated_indices():
    logits = torch.tensor([[0.0, 1.0, 2.0, 3.0]], device="cuda")
    index = torch.tensor([[2, 2, 7, -5]], dtype=torch.int32, device="cuda")
    d = torch.empty_like(logits)
    ok(spblas.route_grad(SIGMOID, logits, index, False, 1.0, torch.tensor([[1.0, 2.0, math.nan, 4.0]], device="cuda"), d))
    s = 1 / (1 + math.exp(-2.0))
    assert d[0, [0, 1, 3]].tolist() == [0.0] * 3 and float(d[0, 2]) == pytest.approx(3 * s * (1 - s), rel=1e-6)


def test_refusals_on_the_device():
    x, i, w = torch.zeros(4, 8, device="cuda"), torch.zeros(4, 2, dtype=torch.int32, device="cuda"), torch.zeros(4, 2, device="cuda")
    assert spblas.route(SIGMOID, x.cpu(), None, 1, 1, True, 1.0, i, w) == capi.INVALID_POINTER
    assert spblas.route(SIGMOID, x, torch.zeros(8), 1, 1, True, 1.0, i, w) == capi.INVALID_POINTER
    assert spblas.route(SIGMOID, x, None, 1, 1, True, 1.0, i, x[:, :2]) == capi.INVALID_VALUE
    assert spblas.route(SIGMOID, x, None, 3, 1, True, 1.0, i, w) == capi.INVALID_VALUE
    assert spblas.route_grad(SIGMOID, x, i, True, 1.0, w, x) == capi.INVALID_VALUE
    ok(spblas.route(SIGMOID, x[:0], None, 1, 1, True, 1.0, i[:0], w[:0]))
