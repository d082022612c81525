"""Rows on no 16-byte boundary through the operators on rows: pieces at the ends of rows and of operands, widths that leave a
group of threads nearly empty, few rows and many."""
import pytest
import torch

from alsparse_b200 import spblas
from rows_util import TYPES, U, assert_within, buffer_of, floor_of, gen, half_step, normal, ok, strided, untouched

pytestmark = pytest.mark.gpu


def _rows(many, width, dtype):
    """Enough rows for the shapes that keep many vectors in flight, or a handful."""
    return 310_000 // (width * torch.finfo(dtype).bits // 128 + 2) + 1 if many else 5


CASES = [(w, m) for w in (1, 3, 7, 8, 9, 15, 17, 255, 259, 531, 2047, 2176) for m in (False, True) if not (m and w < 15)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width,many", CASES)
@pytest.mark.parametrize("shifts", [(0, 0), (1, 0), (0, 3), (5, 2)])
def test_lookup(dtype, width, many, shifts):
    g, count = gen(width), _rows(many, width, dtype)
    table, _ = strided(normal(g, 37, width, dtype=dtype), width + shifts[0], shifts[0])
    y, space = strided(torch.zeros(count, width, dtype=dtype, device="cuda"), width + shifts[1], shifts[1])
    before = space.clone()
    tokens = torch.randint(-1, 38, (count,), generator=g, device="cuda")
    tokens[0], tokens[-1] = 0, 36  # the rows whose vectors could reach out of the table
    inside = (tokens >= 0) & (tokens < 37)
    picked = torch.where(inside[:, None], table[tokens.clamp(0, 36)], 0.0)
    ok(spblas.embedding(tokens, table, 1.0, y))
    assert torch.equal(y, picked.to(dtype)) and untouched(y, space, before)
    ok(spblas.embedding(tokens, table, -1.75, y))
    exact = picked.double() * -1.75
    assert_within(y, exact, (half_step(dtype) + 2 * U) * exact.abs() + floor_of(dtype))
    assert untouched(y, space, before)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width,many", CASES)
@pytest.mark.parametrize("shifts", [(0, 0, 0), (1, 0, 3), (5, 2, 0), (0, 3, 1)])
def test_rows_of_experts(dtype, width, many, shifts):
    g, tokens, k = gen(width + 1), _rows(many, width, dtype), 3
    place = lambda t, s: strided(t, width + s, s)  # noqa: E731
    slot = torch.randperm(tokens * k, generator=g, device="cuda").to(torch.int32).reshape(tokens, k)
    some = torch.rand(tokens, k, generator=g, device="cuda") < 0.9
    some[0], some[-1] = True, False
    slot = torch.where(some, slot, -1).contiguous()
    at, there = slot[some].long(), some[:, :, None]
    used = torch.zeros(tokens * k, 1, dtype=torch.bool, device="cuda")
    used[at] = True

    x, _ = place(normal(g, tokens, width, dtype=dtype), shifts[0])
    xs, space = place(torch.full((tokens * k, width), float("nan"), dtype=dtype, device="cuda"), shifts[1])
    before = space.clone()
    ok(spblas.expert_dispatch(x, slot, xs))
    assert torch.equal(xs[at], x[:, None].expand(-1, k, -1)[some])
    assert bool(xs[~used[:, 0]].isnan().all()) and untouched(xs, space, before)

    weight = normal(g, tokens, k)
    rows = torch.where(there, xs[slot.clamp(min=0).long()].double(), 0.0)
    w = torch.where(some, weight.double(), 0.0)
    for beta in (0.0, 0.5):
        out, space = place(normal(g, tokens, width, dtype=dtype), shifts[2])
        old, before = out.double().clone(), space.clone()
        ok(spblas.expert_combine(xs, slot, weight, beta, out))
        parts = rows * w[:, :, None]
        exact, size = parts.sum(1) + beta * old, parts.abs().sum(1) + beta * old.abs()
        bound = U * (k + 2) * size  # a product and a sum each, and those of beta
        assert_within(out, exact, bound + half_step(dtype) * (exact.abs() + bound) + floor_of(dtype))
        assert untouched(out, space, before)

    dout, _ = place(normal(g, tokens, width, dtype=dtype), shifts[2])
    dy, space = place(torch.full((tokens * k, width), 7.0, dtype=dtype, device="cuda"), shifts[0])
    before, dweight = space.clone(), torch.full((tokens, k), float("nan"), device="cuda")
    ok(spblas.expert_combine_grad(dout, xs, slot, weight, dy, dweight))
    exact = (w[:, :, None] * dout.double()[:, None, :])[some]
    assert_within(dy[at], exact, (half_step(dtype) + 2 * U) * exact.abs() + floor_of(dtype))
    assert bool((dy[~used[:, 0]] == 7.0).all()) and untouched(dy, space, before)
    parts = rows * dout.double()[:, None, :]
    assert_within(dweight, parts.sum(2), U * (width + 8) * parts.abs().sum(2))


@pytest.mark.parametrize("width", [2**24, 2**24 - 4, 2**24 - 3])
def test_the_widest_rows(width):
    g = gen(width)
    x = normal(g, 1, width)
    slot, weight = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.full((1, 1), 0.5, device="cuda")
    y = torch.empty_like(x)
    ok(spblas.embedding(torch.zeros(1, dtype=torch.int64, device="cuda"), x, 1.0, y))
    assert torch.equal(x, y)
    y.zero_()
    ok(spblas.expert_dispatch(x, slot, y))
    assert torch.equal(x, y)
    ok(spblas.expert_combine(x, slot, weight, 0.0, y))
    assert torch.equal(x * 0.5, y)
    dweight = torch.empty(1, 1, device="cuda")
    ok(spblas.expert_combine_grad(x, x, slot, weight, y, dweight))
    assert torch.equal(x * 0.5, y)
    assert_within(dweight, (x.double() ** 2).sum()[None, None], U * (width / 256 + 32) * (x.double() ** 2).sum())  # 256 threads' sums


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("count,vocab", [(16_385, 90_000), (20_000, 700), (100_003, 151), (100_003, 160_000), (4_300_001, 700)])
def test_gradient_of_many_tokens(index, count, vocab):
    g = gen(count)
    tokens = torch.randint(-vocab // 10, vocab + vocab // 10, (2 * count,), generator=g, device="cuda")
    tokens[: count // 2] = tokens[: count // 2] % 7 * (vocab // 8)  # a few rows of many tokens
    tokens[-4:] = torch.tensor([vocab, -1, 2**31 - 1, -2**31], device="cuda")
    if index is torch.int64:
        tokens[:8] = torch.tensor([2**32, -2**32, 2**32 + 5, -2**63, 2**63 - 1, 2**40, vocab - 1, 0], device="cuda")
    tokens = tokens.to(index)[::2]
    inside = (tokens >= 0) & (tokens < vocab)
    dy, dtable = normal(g, count, 3), torch.full((vocab, 3), float("nan"), device="cuda")
    buffer = buffer_of(spblas.embedding_grad_buffer_size(count, vocab, 3))
    ok(spblas.embedding_grad(tokens, dy, 1.0, 0.0, dtable, buffer))
    exact, size, terms = (torch.zeros(vocab, 3, dtype=torch.float64, device="cuda") for _ in range(3))
    at = tokens[inside].long()
    exact.index_add_(0, at, dy[inside].double())
    size.index_add_(0, at, dy[inside].double().abs())
    terms.index_add_(0, at, torch.ones_like(dy[inside], dtype=torch.float64))
    assert_within(dtable, exact, U * (terms + 2) * size)  # any order of a row's terms
