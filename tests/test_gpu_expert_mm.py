"""The experts' products and the gradient of their weights against products in 64 bits."""
import math

import pytest
import torch

from alsparse_b200 import capi, spblas
from rows_util import TYPES, U, assert_within, floor_of, gen, half_step, normal, ok, strided, untouched

pytestmark = pytest.mark.gpu
N, T = capi.NON_TRANSPOSE, capi.TRANSPOSE


def _offsets(counts, first=0):
    o = [first]
    for c in counts:
        o.append(o[-1] + c)
    return torch.tensor(o, dtype=torch.int32, device="cuda")


def _finished():
    assert spblas.expert_mm_status() == (capi.SUCCESS, 0)


def _check_mm(op, offsets, x, w, y, what=""):
    """y is filled with 7 before the call: rows of no expert have to keep it."""
    before = y.clone()
    ok(spblas.expert_mm(op, offsets, x, w, y))
    _finished()
    o = offsets.tolist()
    seen = torch.zeros(x.shape[0], dtype=torch.bool, device="cuda")
    for e in range(w.shape[0]):
        r = slice(o[e], o[e + 1])
        seen[r] = True
        m = w[e].double().t() if op == T else w[e].double()
        exact, size = x[r].double() @ m, x[r].double().abs() @ m.abs()
        # products of 16-bit elements are exact in 32 bits; a sum of n terms in any order, cut off instead of rounded
        bound = 2 * U * (x.shape[1] + 8) * size
        assert_within(y[r], exact, bound + half_step(y.dtype) * (exact.abs() + bound) + floor_of(y.dtype), f"{what} expert {e}")
    assert torch.equal(y[~seen], before[~seen])


def _check_grad(offsets, dy, x, beta, dw, what=""):
    old = dw.clone()
    ok(spblas.expert_mm_grad(offsets, dy, x, beta, dw))
    _finished()
    o = offsets.tolist()
    for e in range(dw.shape[0]):
        r = slice(o[e], o[e + 1])
        a, b = dy[r].double(), x[r].double()
        exact, size = a.t() @ b, a.abs().t() @ b.abs()
        if beta:
            exact, size = exact + beta * old[e].double(), size + abs(beta) * old[e].double().abs()
        bound = 2 * U * (o[e + 1] - o[e] + 8) * size
        assert_within(dw[e], exact, bound + half_step(dw.dtype) * (exact.abs() + bound) + floor_of(dw.dtype), f"{what} expert {e}")


COUNTS = [([1], 1), ([5, 0, 33, 1], 39), ([0, 0, 0], 4), ([300, 0, 129, 128, 127], 690), ([64] * 7 + [65], 513), ([17, 2, 40, 0, 8, 31], 98), ([700], 700)]
SIZES = [(16, 16), (64, 128), (8, 24), (240, 200), (136, 520), (1408, 256), (96, 1000)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("op", [T, N])
@pytest.mark.parametrize("out,inner", SIZES)
@pytest.mark.parametrize("counts,rows", COUNTS)
def test_product(dtype, op, out, inner, counts, rows):
    g = gen(out + rows)
    w = normal(g, len(counts), out, inner, dtype=dtype)
    wide, thin = (inner, out) if op == T else (out, inner)
    x, y = normal(g, rows, wide, dtype=dtype), torch.full((rows, thin), 7.0, dtype=dtype, device="cuda")
    _check_mm(op, _offsets(counts), x, w, y)


@pytest.mark.parametrize("dtype,out_type", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.bfloat16, torch.float32), (torch.float16, torch.float32)])
@pytest.mark.parametrize("out,inner", SIZES)
@pytest.mark.parametrize("counts,rows", COUNTS)
def test_gradient(dtype, out_type, out, inner, counts, rows):
    g = gen(out + rows)
    dy, x = normal(g, rows, out, dtype=dtype), normal(g, rows, inner, dtype=dtype)
    for beta in (0.0, 0.5):
        dw = normal(g, len(counts), out, inner, dtype=out_type) if beta else torch.full((len(counts), out, inner), math.nan, dtype=out_type, device="cuda")
        _check_grad(_offsets(counts), dy, x, beta, dw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("op", [T, N])
@pytest.mark.parametrize("out,inner", [(1, 1), (7, 33), (65, 130), (100, 63), (301, 1155)])
def test_odd_sizes_and_32_bits(dtype, op, out, inner):
    """Rows that begin on no 16-byte boundary, and 32-bit elements."""
    g = gen(out)
    counts = [70, 0, 3, 1, 130]
    w = normal(g, 5, out, inner, dtype=dtype)
    wide, thin = (inner, out) if op == T else (out, inner)
    x, y = normal(g, 210, wide, dtype=dtype), torch.full((210, thin), 7.0, dtype=dtype, device="cuda")
    _check_mm(op, _offsets(counts), x, w, y)
    dy, x = normal(g, 210, out, dtype=dtype), normal(g, 210, inner, dtype=dtype)
    for beta, t in ((0.0, dtype), (1.0, torch.float32)):
        dw = normal(g, 5, out, inner, dtype=t) if beta else torch.full((5, out, inner), math.nan, dtype=t, device="cuda")
        _check_grad(_offsets(counts), dy, x, beta, dw)


@pytest.mark.parametrize("mean", [3, 100])
def test_nothing_comes_over_from_other_experts(mean):
    """Each product reads the rows, the weights and the columns of its own expert: NaN everywhere else."""
    g = gen(mean)
    counts = [mean, mean + 1, mean * 2, mean - 1]
    offsets = _offsets(counts, first=5)
    rows = sum(counts) + 11
    x0, w0 = normal(g, rows, 200, dtype=torch.bfloat16), normal(g, 4, 72, 200, dtype=torch.bfloat16)
    o = offsets.tolist()
    for e in range(4):
        x, w = torch.full_like(x0, math.nan), torch.full_like(w0, math.nan)
        r = slice(o[e], o[e + 1])
        x[r], w[e] = x0[r], w0[e]
        y = torch.zeros(rows, 72, dtype=torch.bfloat16, device="cuda")
        ok(spblas.expert_mm(T, offsets, x, w, y))
        assert bool(y[r].isfinite().all()) and not y[: o[0]].any() and not y[o[4]:].any()
        dy, dx = torch.full((rows, 72), math.nan, dtype=torch.bfloat16, device="cuda"), torch.zeros(rows, 200, dtype=torch.bfloat16, device="cuda")
        dy[r] = 1.0
        ok(spblas.expert_mm(N, offsets, dy, w, dx))
        assert bool(dx[r].isfinite().all()) and not dx[: o[0]].any() and not dx[o[4]:].any()
        dw = torch.full((4, 72, 200), 2.0, dtype=torch.bfloat16, device="cuda")
        ok(spblas.expert_mm_grad(offsets, dy, x, 0.0, dw))
        assert bool(dw[e].isfinite().all())
        exact = dy[r].double().t() @ x[r].double()
        size = dy[r].double().abs().t() @ x[r].double().abs()
        assert_within(dw[e], exact, 2 * U * 210 * size + half_step(torch.bfloat16) * (exact.abs() + 2 * U * 210 * size))
    _finished()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strided_operands(dtype):
    g = gen(8)
    counts = [30, 0, 150, 7]
    offsets, rows = _offsets(counts), 190
    for ldx, shift in ((136, 8), (131, 1)):  # on 16-byte boundaries for 16-bit elements, and not
        x, _ = strided(normal(g, rows, 120, dtype=dtype), ldx, shift)
        space = normal(g, 4 * 100 * 128 + 8, dtype=dtype)
        w = torch.as_strided(space, (4, 96, 120), (100 * 128, 128, 1), 8)
        y, sy = strided(torch.full((rows, 96), 7.0, dtype=dtype, device="cuda"), 104, shift)
        before = sy.clone()
        _check_mm(T, offsets, x, w, y)
        assert untouched(y, sy, before)
        d, sd = strided(torch.full((rows, 120), 7.0, dtype=dtype, device="cuda"), 123, shift)
        before = sd.clone()
        _check_mm(N, offsets, y, w, d)
        assert untouched(d, sd, before)
        grad = torch.zeros(4 * 100 * 128 + 8, dtype=dtype, device="cuda")
        dw = torch.as_strided(grad, (4, 96, 120), (100 * 128, 128, 1), 8)
        _check_grad(offsets, y, x, 0.0, dw)
        rest = grad.clone()
        torch.as_strided(rest, (4, 96, 120), (100 * 128, 128, 1), 8).zero_()
        assert not rest.any()


def test_many_experts_few_rows_and_long_sums():
    g = gen(14)
    counts = torch.randint(0, 3, (1000,), generator=g, device="cuda").tolist()
    offsets, rows = _offsets(counts), sum(counts)
    x, w = normal(g, rows, 64, dtype=torch.bfloat16), normal(g, 1000, 40, 64, dtype=torch.bfloat16)
    y = torch.full((rows, 40), 7.0, dtype=torch.bfloat16, device="cuda")
    ok(spblas.expert_mm(T, offsets, x, w, y))
    at = torch.repeat_interleave(torch.arange(1000, device="cuda"), torch.tensor(counts, device="cuda"))
    exact = torch.einsum("rk,rnk->rn", x.double(), w[at].double())
    size = torch.einsum("rk,rnk->rn", x.double().abs(), w[at].double().abs())
    assert_within(y, exact, 2 * U * 72 * size + half_step(torch.bfloat16) * 1.01 * exact.abs() + floor_of(torch.bfloat16))
    x, w = normal(g, 9, 16384, dtype=torch.bfloat16), normal(g, 2, 128, 16384, dtype=torch.bfloat16)
    _check_mm(T, _offsets([4, 5]), x, w, torch.full((9, 128), 7.0, dtype=torch.bfloat16, device="cuda"))
    dy, x = normal(g, 20_000, 64, dtype=torch.bfloat16), normal(g, 20_000, 72, dtype=torch.bfloat16)
    _check_grad(_offsets([1, 19_990]), dy, x, 0.0, torch.zeros(2, 64, 72, dtype=torch.float32, device="cuda"))
    _finished()


def test_offsets_that_do_not_ascend_write_only_inside():
    """A plan that is not one is not multiplied by, and nothing outside the rows is touched."""
    x, w = torch.ones(300, 64, dtype=torch.bfloat16, device="cuda"), torch.ones(4, 64, 64, dtype=torch.bfloat16, device="cuda")
    y, space = strided(torch.zeros(300, 64, dtype=torch.bfloat16, device="cuda"), 64, 64)
    before = space.clone()
    for bad in ([0, 300, 0, 300, 300], [-50, 10, 400, 2_000_000_000, 5], [300, 200, 100, 50, 0]):
        offsets = torch.tensor(bad, dtype=torch.int32, device="cuda")
        ok(spblas.expert_mm(T, offsets, x, w, y))
        assert untouched(y, space, before) and bool(((y == 0) | (y == 64)).all())
        dw = torch.zeros(4, 64, 64, device="cuda")
        ok(spblas.expert_mm_grad(offsets, x, x, 0.0, dw))
        assert bool(dw.isfinite().all())
    _finished()


def test_lengths_of_zero():
    x, w = torch.zeros(6, 0, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, 8, 0, dtype=torch.bfloat16, device="cuda")
    y = torch.full((6, 8), 7.0, dtype=torch.bfloat16, device="cuda")
    ok(spblas.expert_mm(T, _offsets([2, 3]), x, w, y))
    assert not y[:5].any() and bool((y[5] == 7).all())
    ok(spblas.expert_mm(N, _offsets([2, 3]), y, w, x))
    none = torch.zeros(0, 8, dtype=torch.bfloat16, device="cuda")
    dw = torch.full((2, 8, 8), 4.0, dtype=torch.bfloat16, device="cuda")
    ok(spblas.expert_mm(T, _offsets([0, 0]), none, dw, none))
    ok(spblas.expert_mm_grad(_offsets([0, 0]), none, none, 0.25, dw))
    assert bool((dw == 1).all())


def test_gradient_against_differences():
    """The product is linear in x and in w: a step of 1/4 along a direction gives the gradients' inner products."""
    g = gen(19)
    offsets = _offsets([40, 0, 3, 90])
    bf = torch.bfloat16
    x, w, dy = normal(g, 133, 64, dtype=bf), normal(g, 4, 72, 64, dtype=bf), normal(g, 133, 72, dtype=bf)
    dx, dw = torch.zeros(133, 64, dtype=bf, device="cuda"), torch.zeros(4, 72, 64, device="cuda")
    ok(spblas.expert_mm(N, offsets, dy, w, dx))
    ok(spblas.expert_mm_grad(offsets, dy, x, 0.0, dw))

    def value(x, w):
        y = torch.zeros(133, 72, dtype=bf, device="cuda")
        ok(spblas.expert_mm(T, offsets, x, w, y))
        return y.double()

    for which, grad in ((0, dx), (1, dw)):
        a = (x, w)[which]
        moved = (a + 0.25 * normal(g, *a.shape, dtype=bf)).to(bf)
        step = moved.double() - a.double()
        up, at = value(*((moved, w) if which == 0 else (x, moved))), value(x, w)
        # what rounding to 16 bits leaves in the two values, and in the gradient
        bound = ((up.abs() + at.abs()) * dy.double().abs()).sum() * half_step(bf) * 1.01 + (grad.double().abs() * step.abs()).sum() * (half_step(bf) if which == 0 else 1e-4)
        assert abs(((up - at) * dy.double()).sum() - (grad.double() * step).sum()) <= bound


def test_refusals_on_the_device():
    x, w, y = torch.zeros(4, 8, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, 8, 8, dtype=torch.bfloat16, device="cuda"), torch.zeros(4, 8, dtype=torch.bfloat16, device="cuda")
    o = _offsets([2, 2])
    assert spblas.expert_mm(T, o.cpu(), x, w, y) == capi.INVALID_POINTER
    assert spblas.expert_mm(T, o, x, w.cpu(), y) == capi.INVALID_POINTER
    assert spblas.expert_mm(T, o, x, w, x) == capi.INVALID_VALUE
    assert spblas.expert_mm(T, o, x, w, w[0, :4]) == capi.INVALID_VALUE
    assert spblas.expert_mm(T, o.long(), x, w, y) == capi.INVALID_VALUE
    assert spblas.expert_mm(T, o, x, w, y.float()) == capi.INVALID_VALUE
    assert spblas.expert_mm(T, o, x, w[:1].expand(2, 8, 8), y) == capi.INVALID_VALUE      # matrices in one place
    assert spblas.expert_mm(capi.CONJUGATE_TRANSPOSE, o, x, w, y) == capi.INVALID_VALUE
    assert spblas.expert_mm_grad(o, y, x, 0.0, w.half()) == capi.NOT_SUPPORTED
