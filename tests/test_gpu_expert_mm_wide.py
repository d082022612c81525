"""Gradients of the experts' weights at the widest sizes that the calls take, on the ordinary units and on the tensor cores."""
import pytest
import torch

from alsparse_b200 import spblas
from rows_util import U, assert_within, floor_of, gen, half_step, normal, ok

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("out,inner", [(1 << 24, 1), (4_194_241, 3), (1, 1 << 24), (3, 4_194_241), (70_000, 130)])
def test_gradient(dtype, out, inner):
    g = gen(out)
    offsets = torch.tensor([1, 4, 4], dtype=torch.int32, device="cuda")
    dy, x = normal(g, 5, out, dtype=dtype), normal(g, 5, inner, dtype=dtype)
    dw = torch.full((2, out, inner), 7.0, dtype=dtype, device="cuda")
    ok(spblas.expert_mm_grad(offsets, dy, x, 0.0, dw))
    a, b = dy[1:4].double(), x[1:4].double()
    bound = 2 * U * 11 * (a.abs().t() @ b.abs())
    exact = a.t() @ b
    assert_within(dw[0], exact, bound + half_step(dtype) * (exact.abs() + bound) + floor_of(dtype))
    assert not dw[1].any()
    assert spblas.expert_mm_status() == (0, 0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradient_without_rows(dtype):
    dw = torch.full((1, 4_194_241, 2), 8.0, dtype=dtype, device="cuda")
    none = torch.zeros(0, 4_194_241, dtype=dtype, device="cuda")
    ok(spblas.expert_mm_grad(torch.zeros(2, dtype=torch.int32, device="cuda"), none, none[:, :2], 0.25, dw))
    assert bool((dw == 2).all())
