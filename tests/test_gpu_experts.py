"""Rows of tokens to their experts and back: the plan exactly, dispatch bit for bit, combine and its gradients in 64 bits."""
import math

import pytest
import torch

from alsparse_b200 import capi, spblas
from rows_util import TYPES, U, assert_within, buffer_of, floor_of, gen, half_step, normal, ok, plan64, strided, untouched

pytestmark = pytest.mark.gpu


def _index(g, tokens, k, experts, kind="mixed"):
    index = torch.randint(0, experts, (tokens, k), generator=g, device="cuda", dtype=torch.int32)
    if kind == "mixed" and tokens:
        index[torch.rand(tokens, k, generator=g, device="cuda") < 0.3] = experts // 3
        index[torch.rand(tokens, k, generator=g, device="cuda") < 0.1] = -1
        index[torch.rand(tokens, k, generator=g, device="cuda") < 0.02] = experts
    elif kind == "empty":
        index[:] = -1
    elif kind == "one":
        index[:] = experts - 1
    return index


def _plan(index, experts):
    offsets = torch.full((experts + 1,), -9, dtype=torch.int32, device="cuda")
    slot = torch.full_like(index, -9)
    ok(spblas.expert_plan(index, offsets, slot, buffer_of(spblas.expert_plan_buffer_size(index.shape[0], index.shape[1], experts))))
    return offsets, slot


@pytest.mark.parametrize("kind", ["mixed", "even", "empty", "one"])
@pytest.mark.parametrize("tokens,k,experts", [(0, 2, 5), (1, 1, 1), (1, 8, 256), (32, 8, 256), (513, 1, 7), (700, 6, 1024), (4096, 1, 64), (4097, 1, 64), (5000, 8, 60), (16384, 8, 256), (300_000, 1, 33)])
def test_plan(kind, tokens, k, experts):
    index = _index(gen(tokens + k), tokens, k, experts, kind)
    offsets, slot = _plan(index, experts)
    want_offsets, want_slot = plan64(index.cpu(), experts)
    assert torch.equal(offsets.cpu(), want_offsets) and torch.equal(slot.cpu(), want_slot)


def test_plan_of_strided_choices():
    index, _ = strided(_index(gen(1), 900, 5, 40), 7, 1)
    slot, space = strided(torch.zeros(900, 5, dtype=torch.int32, device="cuda"), 6, 3)
    before = space.clone()
    offsets = torch.empty(41, dtype=torch.int32, device="cuda")
    ok(spblas.expert_plan(index, offsets, slot, buffer_of(spblas.expert_plan_buffer_size(900, 5, 40))))
    want = plan64(index.cpu(), 40)
    assert torch.equal(offsets.cpu(), want[0]) and torch.equal(slot.cpu(), want[1]) and untouched(slot, space, before)


SHAPES = [(1, 1, 1, 1), (1, 8, 64, 2048), (32, 8, 256, 96), (200, 6, 60, 1001), (300, 2, 5, 5000), (1000, 9, 33, 130), (64, 5, 16, 30)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,k,experts,width", SHAPES)
def test_dispatch(dtype, tokens, k, experts, width):
    g = gen(tokens + width)
    index, x = _index(g, tokens, k, experts), normal(g, tokens, width, dtype=dtype)
    offsets, slot = _plan(index, experts)
    xs = torch.full((tokens * k + 3, width), 7.0, dtype=dtype, device="cuda")
    ok(spblas.expert_dispatch(x, slot, xs))
    want = torch.full_like(xs, 7.0)
    some = slot.reshape(-1) >= 0
    want[slot.reshape(-1)[some].long()] = x.repeat_interleave(k, 0)[some]
    assert torch.equal(xs, want)  # the rows behind the last among them


def _combine_exact(y, slot, weight):
    some = slot >= 0
    w = torch.where(some, 1.0 if weight is None else weight.double(), 0.0)
    rows = torch.where(some[:, :, None], y.double()[slot.clamp(min=0).long()], 0.0)
    return (rows * w[:, :, None]).sum(1), (rows.abs() * w.abs()[:, :, None]).sum(1), rows, w


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,k,experts,width", SHAPES)
def test_combine_and_its_gradients(dtype, tokens, k, experts, width):
    g = gen(tokens + width)
    _, slot = _plan(_index(g, tokens, k, experts), experts)
    y, weight = normal(g, tokens * k, width, dtype=dtype), normal(g, tokens, k)
    used = torch.zeros(tokens * k, dtype=torch.bool, device="cuda")
    used[slot[slot >= 0].long()] = True
    y[~used] = math.nan              # rows behind the last are not read
    weight[slot < 0] = math.nan      # nor the weights of empty choices
    for w, beta in ((weight, 0.0), (None, 0.0), (weight, 1.0), (weight, -0.5)):
        old = normal(g, tokens, width, dtype=dtype) if beta else torch.full((tokens, width), math.nan, dtype=dtype, device="cuda")
        out = old.clone()
        ok(spblas.expert_combine(y, slot, w, beta, out))
        exact, size, _, _ = _combine_exact(torch.where(used[:, None], y, 0.0), slot, w)
        if beta:
            exact, size = exact + beta * old.double(), size + abs(beta) * old.double().abs()
        bound = U * (k + 1) * size
        assert_within(out, exact, bound + half_step(dtype) * (exact.abs() + bound) + floor_of(dtype), "combine")
    dout = normal(g, tokens, width, dtype=dtype)
    for w in (weight, None):
        dy, dweight = torch.full_like(y, 3.0), torch.full((tokens, k), math.nan, device="cuda")
        ok(spblas.expert_combine_grad(dout, y, slot, w, dy, dweight))
        _, _, rows, w64 = _combine_exact(torch.where(used[:, None], y, 0.0), slot, w)
        want = torch.full((tokens * k, width), 3.0, dtype=torch.float64, device="cuda")
        some = (slot >= 0).reshape(-1)
        want[slot.reshape(-1)[some].long()] = (w64[:, :, None] * dout.double()[:, None, :]).reshape(-1, width)[some]
        assert_within(dy, want, (half_step(dtype) + 2 * U) * want.abs() + floor_of(dtype), "dy")
        exact = (rows * dout.double()[:, None, :]).sum(2)
        # one product and sum per element of the row
        assert_within(dweight, exact, U * (width + 8) * (rows.abs() * dout.double().abs()[:, None, :]).sum(2), "dweight")


def test_gradient_of_dispatch_is_combine_with_ones():
    """<dispatch(x), d> = <x, combine(d)>, the second one without weights."""
    g = gen(31)
    _, slot = _plan(_index(g, 70, 4, 9), 9)
    x, d = normal(g, 70, 33), normal(g, 280, 33)
    xs, dx = torch.zeros(280, 33, device="cuda"), torch.empty(70, 33, device="cuda")
    ok(spblas.expert_dispatch(x, slot, xs))
    ok(spblas.expert_combine(d, slot, None, 0.0, dx))
    left, right = (xs.double() * d.double()).sum(), (x.double() * dx.double()).sum()
    assert abs(left - right) <= 5 * U * (xs.double() * d.double()).abs().sum()


def test_gradients_of_combine_against_differences():
    g = gen(32)
    _, slot = _plan(_index(g, 20, 3, 5), 5)
    y, weight, dout = normal(g, 60, 17), normal(g, 20, 3), normal(g, 20, 17)
    dy, dweight = torch.zeros_like(y), torch.empty_like(weight)
    ok(spblas.expert_combine_grad(dout, y, slot, weight, dy, dweight))

    def value(y, weight):
        out = torch.empty(20, 17, device="cuda")
        ok(spblas.expert_combine(y, slot, weight, 0.0, out))
        return (out.double() * dout.double()).sum()

    h = 0.25
    for a, d in ((y, dy), (weight, dweight)):
        direction = normal(g, *a.shape)
        plus, minus = a + h * direction, a - h * direction
        args = (lambda v: (v, weight)) if a is y else (lambda v: (y, v))
        slope = (value(*args(plus)) - value(*args(minus))) / (2 * h)
        # the product is linear in each: what is left is roundings, of the moved operand and of the sums, over 2 h
        size = 4 * 20 * 3 * 17 * 16
        assert abs(slope - (d.double() * direction.double()).sum()) <= 8 * U / h * size


def test_strided_rows():
    g = gen(6)
    for dtype in TYPES:
        _, slot0 = _plan(_index(g, 50, 3, 6), 6)
        slot, _ = strided(slot0, 5, 1)
        x, _ = strided(normal(g, 50, 72, dtype=dtype), 81, 1)
        xs, space = strided(torch.zeros(150, 72, dtype=dtype, device="cuda"), 77, 2)
        before = space.clone()
        ok(spblas.expert_dispatch(x, slot, xs))
        plain = torch.zeros(150, 72, dtype=dtype, device="cuda")
        ok(spblas.expert_dispatch(x.contiguous(), slot0, plain))
        assert torch.equal(xs, plain) and untouched(xs, space, before)
        weight, _ = strided(normal(g, 50, 3), 4, 1)
        out, so = strided(torch.zeros(50, 72, dtype=dtype, device="cuda"), 75, 5)
        before = so.clone()
        ok(spblas.expert_combine(xs, slot, weight, 0.0, out))
        plain_out = torch.empty(50, 72, dtype=dtype, device="cuda")
        ok(spblas.expert_combine(plain, slot0, weight.contiguous(), 0.0, plain_out))
        assert torch.equal(out, plain_out) and untouched(out, so, before)
        dy, sy = strided(torch.zeros(150, 72, dtype=dtype, device="cuda"), 90, 3)
        dw, sw = strided(torch.zeros(50, 3, device="cuda"), 7, 1)
        by, bw = sy.clone(), sw.clone()
        ok(spblas.expert_combine_grad(x, xs, slot, weight, dy, dw))
        assert untouched(dy, sy, by) and untouched(dw, sw, bw)
        plain_dy, plain_dw = torch.zeros(150, 72, dtype=dtype, device="cuda"), torch.empty(50, 3, device="cuda")
        ok(spblas.expert_combine_grad(x.contiguous(), plain, slot0, weight.contiguous(), plain_dy, plain_dw))
        assert torch.equal(dy, plain_dy)
        # narrower loads take the elements of a row in another order
        size = (x.double().abs().amax() * plain.double().abs().amax()) * 72
        assert_within(dw, plain_dw, 2 * U * 80 * size)


def test_slots_outside_the_rows_are_empty():
    slot = torch.tensor([[0, 5], [-3, 1], [2, 1000]], dtype=torch.int32, device="cuda")
    x, xs, out = torch.arange(12.0, device="cuda").view(3, 4), torch.zeros(4, 4, device="cuda"), torch.empty(3, 4, device="cuda")
    ok(spblas.expert_dispatch(x, slot, xs))
    assert torch.equal(xs[[0, 1, 2]], x) and not xs[3].any()
    ok(spblas.expert_combine(xs, slot, None, 0.0, out))
    assert torch.equal(out, x)
    dy, dw = torch.zeros(4, 4, device="cuda"), torch.empty(3, 2, device="cuda")
    ok(spblas.expert_combine_grad(x, xs, slot, None, dy, dw))
    assert torch.equal(dy, xs) and dw[:, 0].tolist()[1] == 0 and dw[:, 1].tolist()[0] == 0 and dw[2, 1] == 0
    # no rows at all
    ok(spblas.expert_combine(xs[:0], slot, None, 0.0, out))
    assert not out.any()


def test_refusals_on_the_device():
    x, slot, xs = torch.zeros(4, 8, device="cuda"), torch.zeros(4, 2, dtype=torch.int32, device="cuda"), torch.zeros(8, 8, device="cuda")
    assert spblas.expert_dispatch(x, slot, xs.cpu()) == capi.INVALID_POINTER
    assert spblas.expert_dispatch(x, slot.cpu(), xs) == capi.INVALID_POINTER
    assert spblas.expert_dispatch(xs[:4], slot, xs) == capi.INVALID_VALUE
    assert spblas.expert_dispatch(x, slot.long(), xs) == capi.INVALID_VALUE
    assert spblas.expert_combine(xs, slot, None, 0.0, xs[2:6]) == capi.INVALID_VALUE
    offsets = torch.zeros(65, dtype=torch.int32, device="cuda")
    index = torch.zeros(9000, 1, dtype=torch.int32, device="cuda")
    assert spblas.expert_plan(index, offsets, torch.zeros_like(index), None) == capi.NOT_INITIALIZED    # needs a workspace
    assert spblas.expert_plan(index, offsets, index, buffer_of(spblas.expert_plan_buffer_size(9000, 1, 64))) == capi.INVALID_VALUE
