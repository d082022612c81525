"""The operators on rows of experts where elements lie more than 2^31 behind the first, and where a shifted load reaches over the
columns of another operand that is being written."""
import pytest
import torch

from alsparse_b200 import capi, spblas
from rows_util import TYPES, U, assert_within, floor_of, gen, half_step, normal, ok

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("width", [4096, 4095])
def test_rows_beyond_32_bits(width):
    g, rows, tokens, k = gen(width), 560_000, 3, 2   # 2.3e9 elements
    xs = torch.zeros(rows, width, dtype=BF, device="cuda")
    slot = torch.tensor([[rows - 1, 0], [530_000, -1], [rows, 540_001]], dtype=torch.int32, device="cuda")
    x = normal(g, tokens, width, dtype=BF)
    ok(spblas.expert_dispatch(x, slot, xs))
    assert torch.equal(xs[[rows - 1, 0, 530_000, 540_001]], x[[0, 0, 1, 2]]) and not xs[[1, rows - 2, 529_999, 530_001, 540_000, 540_002]].any()
    weight, out = normal(g, tokens, k), torch.empty(tokens, width, dtype=BF, device="cuda")
    ok(spblas.expert_combine(xs, slot, weight, 0.0, out))
    w = torch.where((slot >= 0) & (slot < rows), weight, 0.0).double()
    exact, size = w.sum(1)[:, None] * x.double(), w.abs().sum(1)[:, None] * x.double().abs()
    assert_within(out, exact, 3 * U * size + half_step(BF) * (exact.abs() + 3 * U * size) + floor_of(BF))
    dout, dweight, dy = normal(g, tokens, width, dtype=BF), torch.empty(tokens, k, device="cuda"), torch.zeros(rows, width, dtype=BF, device="cuda")
    ok(spblas.expert_combine_grad(dout, xs, slot, weight, dy, dweight))
    for t, j in ((0, 0), (0, 1), (1, 0), (2, 1)):
        exact = weight[t, j].double() * dout[t].double()
        assert_within(dy[int(slot[t, j])], exact, (half_step(BF) + 2 * U) * exact.abs() + floor_of(BF))
        parts = dout[t].double() * x[t].double()
        assert_within(dweight[t, j], parts.sum(), U * (width + 8) * parts.abs().sum())
    assert dweight[1, 1] == 0 and dweight[2, 0] == 0 and not dy[[1, rows - 2, 529_999, 540_000]].any()
    del xs, dy
    torch.cuda.empty_cache()


def _some_rows(rows, x, m, y):
    """Rows of y against x times m of their expert, in 64 bits."""
    for r in rows:
        a = x[r].double()
        exact, size = a @ m, a.abs() @ m.abs()
        bound = 2 * U * (x.shape[1] + 8) * size
        assert_within(y[r], exact, bound + half_step(BF) * (exact.abs() + bound) + floor_of(BF), f"row {r}")


@pytest.mark.parametrize("inner", [64, 63])
def test_products_of_rows_beyond_32_bits(inner):
    g, rows, out = gen(inner), 2_200_000, 1024   # y and dy: 2.25e9 elements
    offsets = torch.tensor([7, 1_000_001, rows - 3], dtype=torch.int32, device="cuda")
    x, w = normal(g, rows, inner, dtype=BF), normal(g, 2, out, inner, dtype=BF)
    y = torch.full((rows, out), 7.0, dtype=BF, device="cuda")
    ok(spblas.expert_mm(capi.TRANSPOSE, offsets, x, w, y))
    _some_rows((7, 999_999, 1_000_000), x, w[0].double().t(), y)
    _some_rows((1_000_001, 2_097_151, 2_097_152, 2_150_000, rows - 4), x, w[1].double().t(), y)
    assert bool((y[:7] == 7).all()) and bool((y[rows - 3:] == 7).all())
    dx = torch.full((rows, inner), 7.0, dtype=BF, device="cuda")
    ok(spblas.expert_mm(capi.NON_TRANSPOSE, offsets, y, w, dx))
    _some_rows((7, 1_000_000), y, w[0].double(), dx)
    _some_rows((1_000_001, 2_097_152, rows - 4), y, w[1].double(), dx)
    y.zero_()   # dy: a few rows at the far end
    at = torch.tensor([1_000_000, 2_097_153, rows - 4], device="cuda")
    y[at] = normal(g, 3, out, dtype=BF)
    dw = torch.empty(2, out, inner, device="cuda")
    ok(spblas.expert_mm_grad(offsets, y, x, 0.0, dw))
    for e, r in ((0, at[:1]), (1, at[1:])):
        a, b = y[r].double(), x[r].double()
        assert_within(dw[e], a.t() @ b, 2 * U * 16 * (a.abs().t() @ b.abs()))
    assert spblas.expert_mm_status() == (capi.SUCCESS, 0)
    del y
    torch.cuda.empty_cache()


@pytest.mark.parametrize("inner", [8192, 8190])
def test_products_with_weights_beyond_32_bits(inner):
    g, experts, out = gen(inner), 36, 8192       # 2.4e9 elements
    w = torch.zeros(experts, out, inner, dtype=BF, device="cuda")
    counts = [2] * experts
    offsets = torch.arange(experts + 1, dtype=torch.int32, device="cuda") * 2
    for e in (0, 31, 32, 35):
        w[e] = normal(g, out, inner, dtype=BF)
    x, y = normal(g, sum(counts), inner, dtype=BF), torch.full((sum(counts), out), 7.0, dtype=BF, device="cuda")
    ok(spblas.expert_mm(capi.TRANSPOSE, offsets, x, w, y))
    for e in (0, 31, 32, 35):
        _some_rows((2 * e, 2 * e + 1), x, w[e].double().t(), y)
    assert not y[4].any() and not y[68].any()
    dw = torch.full_like(w, 7.0)
    ok(spblas.expert_mm_grad(offsets, y, x, 0.0, dw))
    for e in (0, 32, 35, 34):
        a, b = y[2 * e:2 * e + 2].double(), x[2 * e:2 * e + 2].double()
        exact, size = a.t() @ b, a.abs().t() @ b.abs()
        assert_within(dw[e], exact, 2 * U * 10 * size + half_step(BF) * (exact.abs() + 2 * U * 10 * size) + floor_of(BF))
    assert spblas.expert_mm_status() == (capi.SUCCESS, 0)
    del w, dw
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [5, 33, 259, 2047])
def test_operands_in_columns_of_one_block(dtype, width):
    """Source and result side by side in rows of 3 * width + 2 elements, on every alignment as the rows go down."""
    g, tokens, k = gen(width), 301, 3
    ld, n = 3 * width + 2, tokens * 3
    for first, second in ((0, width), (width + 1, 1), (1, 2 * width + 1)):
        block = normal(g, n, ld, dtype=dtype)
        slot = torch.randperm(n, generator=g, device="cuda").to(torch.int32).reshape(tokens, k)
        weight = normal(g, tokens, k)
        before = block.clone()
        a, b = block[:, first:first + width], block[:, second:second + width]

        def rest():
            mask = torch.ones(ld, dtype=torch.bool, device="cuda")
            mask[second:second + width] = False
            return torch.equal(block[:, mask], before[:, mask])

        ok(spblas.expert_dispatch(a[:tokens], slot, b))
        assert torch.equal(b[slot.long()], a[:tokens, None].expand(-1, k, -1)) and rest()
        old = b[:tokens].double().clone()
        ok(spblas.expert_combine(a, slot, weight, 0.5, b[:tokens]))
        parts = a[slot.long()].double() * weight.double()[:, :, None]
        exact, size = parts.sum(1) + 0.5 * old, parts.abs().sum(1) + 0.5 * old.abs()
        bound = U * (k + 2) * size
        assert_within(b[:tokens], exact, bound + half_step(dtype) * (exact.abs() + bound) + floor_of(dtype))
        assert rest()
        tokens_of = torch.randint(-1, n, (n,), generator=g, device="cuda")
        ok(spblas.embedding(tokens_of, a, 1.0, b))
        assert torch.equal(b, torch.where((tokens_of >= 0)[:, None], a[tokens_of.clamp(min=0)], 0.0)) and rest()
        dout, dweight = normal(g, tokens, width, dtype=dtype), torch.empty(tokens, k, device="cuda")
        ok(spblas.expert_combine_grad(dout, a, slot, weight, b, dweight))
        exact = weight.double()[:, :, None] * dout.double()[:, None, :]
        assert_within(b[slot.long()], exact, (half_step(dtype) + 2 * U) * exact.abs() + floor_of(dtype))
        parts = a[slot.long()].double() * dout.double()[:, None, :]
        assert_within(dweight, parts.sum(2), U * (width + 8) * parts.abs().sum(2))
        assert rest()
