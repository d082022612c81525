"""Embedding lookup and the gradient of its table against the same sums in 64 bits."""
import math

import pytest
import torch

from alsparse_b200 import capi, spblas
from rows_util import TYPES, U, assert_within, buffer_of, floor_of, gen, half_step, normal, ok, strided, untouched

pytestmark = pytest.mark.gpu


def _tokens(g, count, vocab, dtype=torch.int64, kind="mixed"):
    t = torch.randint(0, max(vocab, 1), (count,), generator=g, device="cuda")
    if kind == "mixed" and count:
        t[torch.rand(count, generator=g, device="cuda") < 0.4] = vocab // 2    # one word makes up much of the text
        t[torch.rand(count, generator=g, device="cuda") < 0.1] = -1
        t[torch.rand(count, generator=g, device="cuda") < 0.05] = vocab         # of another part of the table
        if dtype is torch.int64:
            t[torch.rand(count, generator=g, device="cuda") < 0.05] = (1 << 32) + 1
    elif kind == "one":
        t[:] = vocab - 1
    return t.to(dtype)


def _exact(tokens, table, scale):
    inside = (tokens >= 0) & (tokens < table.shape[0])
    y = table.double()[tokens.long().clamp(0, table.shape[0] - 1)] * scale
    return torch.where(inside[:, None], y, 0.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("count,vocab,width", [(1, 1, 1), (1, 777, 2048), (24, 1000, 96), (33, 5, 7), (2000, 513, 130), (700, 4000, 1001), (40, 300, 5000)])
def test_lookup(dtype, index, count, vocab, width):
    g = gen(count + width)
    tokens, table = _tokens(g, count, vocab, index), normal(g, vocab, width, dtype=dtype)
    for scale in (1.0, 2.75):
        y = torch.full((count, width), math.nan, dtype=dtype, device="cuda")
        ok(spblas.embedding(tokens, table, scale, y))
        exact = _exact(tokens, table, scale)
        if scale == 1.0:
            assert torch.equal(y.double(), exact)
        # the product is rounded to 32 bits and then to the type
        assert_within(y, exact, (half_step(dtype) + 2 * U) * exact.abs() + floor_of(dtype), "lookup")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width,ld,shift", [(64, 72, 0), (64, 64, 1), (30, 33, 3), (128, 200, 2), (256, 1024, 4)])
def test_lookup_of_strided_rows_and_tokens(dtype, width, ld, shift):
    g = gen(7)
    table, _ = strided(normal(g, 50, width, dtype=dtype), ld, shift)
    tokens = _tokens(g, 3 * 41, 50)[::3]
    y, space = strided(torch.zeros(41, width, dtype=dtype, device="cuda"), ld + 3, shift)
    before = space.clone()
    ok(spblas.embedding(tokens, table, 1.0, y))
    assert torch.equal(y.double(), _exact(tokens, table, 1.0))
    assert untouched(y, space, before)


def test_lookup_copies_special_values_and_does_not_read_unselected_rows():
    table = torch.tensor([[math.inf, -0.0], [math.nan, 1.0], [-math.inf, 3.0e38]], device="cuda")
    y = torch.empty(4, 2, device="cuda")
    ok(spblas.embedding(torch.tensor([0, 2, -1, 3], device="cuda"), table, 1.0, y))
    assert y.tolist() == [[math.inf, -0.0], [-math.inf, pytest.approx(3.0e38)], [0.0, 0.0], [0.0, 0.0]]
    ok(spblas.embedding(torch.tensor([-1, -1, -1, 9], device="cuda"), table, math.inf, y))
    assert y.tolist() == [[0.0, 0.0]] * 4


def _grad_exact(tokens, dy, alpha, beta, old, vocab):
    inside = (tokens >= 0) & (tokens < vocab)
    total = torch.zeros(vocab, dy.shape[1], dtype=torch.float64, device="cuda")
    size, count = torch.zeros_like(total), torch.zeros(vocab, 1, dtype=torch.float64, device="cuda")
    at, rows = tokens[inside].long(), dy[inside].double()
    total.index_add_(0, at, rows)
    size.index_add_(0, at, rows.abs())
    count.index_add_(0, at, torch.ones(len(at), 1, dtype=torch.float64, device="cuda"))
    exact = alpha * total + (beta * old.double() if beta else 0.0)
    # n terms are added one after the other at worst; the product with alpha, the one with beta and their sum round once each
    bound = U * ((count + 2) * abs(alpha) * size + 3 * abs(beta) * (old.double().abs() if beta else 0.0))
    return exact, bound


@pytest.mark.parametrize("dtype,out", [(torch.float32, torch.float32), (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16),
                                       (torch.bfloat16, torch.float32), (torch.float16, torch.float32)])
@pytest.mark.parametrize("count,vocab,width,kind", [(1, 1, 1, "one"), (24, 1000, 96, "mixed"), (0, 100, 64, "mixed"), (33, 5, 7, "mixed"), (2000, 1300, 130, "mixed"),
                                                    (3000, 600, 1001, "mixed"), (4097, 512, 64, "one"), (1500, 2000, 2048, "mixed"), (32, 513, 40, "one"), (65, 513, 40, "one")])
def test_gradient(dtype, out, count, vocab, width, kind):
    g = gen(count + width)
    for index, alpha, beta in ((torch.int64, 1.0, 0.0), (torch.int32, 0.125, 1.0), (torch.int64, -2.0, 0.5)):
        tokens, dy = _tokens(g, count, vocab, index, kind), normal(g, count, width, dtype=dtype)
        old = normal(g, vocab, width, dtype=out) if beta else torch.full((vocab, width), math.nan, dtype=out, device="cuda")
        d = old.clone()
        buffer = buffer_of(spblas.embedding_grad_buffer_size(count, vocab, width))
        ok(spblas.embedding_grad(tokens, dy, alpha, beta, d, buffer))
        exact, bound = _grad_exact(tokens, dy, alpha, beta, old, vocab)
        assert_within(d, exact, bound + half_step(out) * (exact.abs() + bound) + floor_of(out), "gradient")
        if beta == 1.0:  # rows that no token names stay, bit for bit
            idle = torch.ones(vocab, dtype=torch.bool, device="cuda")
            idle[tokens[(tokens >= 0) & (tokens < vocab)].long()] = False
            assert torch.equal(d[idle], old[idle])
        again = old.clone()
        ok(spblas.embedding_grad(tokens, dy, alpha, beta, again, buffer))
        assert torch.equal(d, again)


@pytest.mark.parametrize("width,ld,shift", [(64, 72, 0), (64, 64, 1), (30, 34, 2), (129, 200, 3)])
def test_gradient_of_strided_rows(width, ld, shift):
    g = gen(9)
    dy, _ = strided(normal(g, 300, width, dtype=torch.bfloat16), ld, shift)
    tokens = _tokens(g, 2 * 300, 70)[::2]
    for out in (torch.bfloat16, torch.float32):
        d, space = strided(torch.zeros(70, width, dtype=out, device="cuda"), ld + 1, shift)
        before = space.clone()
        buffer = buffer_of(spblas.embedding_grad_buffer_size(300, 70, width))
        ok(spblas.embedding_grad(tokens, dy, 1.0, 0.0, d, buffer))
        exact, bound = _grad_exact(tokens, dy, 1.0, 0.0, d, 70)
        assert_within(d, exact, bound + half_step(out) * (exact.abs() + bound) + floor_of(out))
        assert untouched(d, space, before)


def test_gradient_keeps_special_values_in_their_rows():
    dy = torch.ones(4, 3, device="cuda")
    dy[1, 1], dy[2, 2], dy[3] = math.nan, math.inf, math.nan
    d = torch.full((5, 3), math.nan, device="cuda")
    tokens = torch.tensor([1, 1, 3, -1], device="cuda")
    ok(spblas.embedding_grad(tokens, dy, 1.0, 0.0, d, buffer_of(spblas.embedding_grad_buffer_size(4, 5, 3))))
    assert torch.equal(d.isnan(), torch.tensor([[0, 0, 0], [0, 1, 0], [0, 0, 0], [0, 0, 0], [0, 0, 0]], device="cuda").bool())
    assert d[1, 0] == 2 and d[3].tolist() == [1.0, 1.0, math.inf] and not d[[0, 2, 4]].any()


def test_gradient_is_the_transpose_of_the_lookup():
    """<lookup(table), dy> = <table, gradient(dy)>, and the lookup is linear: differences of it give the same number."""
    g = gen(11)
    tokens, table, dy = _tokens(g, 500, 90), normal(g, 90, 48), normal(g, 500, 48)
    y, d = torch.empty(500, 48, device="cuda"), torch.empty(90, 48, device="cuda")
    ok(spblas.embedding(tokens, table, 1.5, y))
    ok(spblas.embedding_grad(tokens, dy, 1.5, 0.0, d, buffer_of(spblas.embedding_grad_buffer_size(500, 90, 48))))
    left, right = (y.double() * dy.double()).sum(), (table.double() * d.double()).sum()
    size = (y.double() * dy.double()).abs().sum()
    assert abs(left - right) <= U * (500 + 4) * size
    at, column, h = int(tokens[tokens >= 0][0]) % 90, 5, 0.25
    table[at, column] += h
    y2 = torch.empty_like(y)
    ok(spblas.embedding(tokens, table, 1.5, y2))
    slope = ((y2.double() - y.double()) * dy.double()).sum() / h
    # each changed element of y is rounded in both lookups
    assert abs(slope - d[at, column]) <= (4 / h) * U * float((y[:, column].abs() * dy[:, column].abs()).double().sum() + 500) + 500 * U * float(dy[:, column].abs().sum())


def test_more_tokens_than_a_block_of_the_sort_reads_at_once():
    g = gen(12)
    tokens, dy = _tokens(g, 300_000, 70_001, torch.int32), normal(g, 300_000, 8)
    d = torch.empty(70_001, 8, device="cuda")
    ok(spblas.embedding_grad(tokens, dy, 1.0, 0.0, d, buffer_of(spblas.embedding_grad_buffer_size(300_000, 70_001, 8))))
    exact, _ = _grad_exact(tokens, dy, 1.0, 0.0, d, 70_001)
    size, _ = _grad_exact(tokens, dy.abs(), 1.0, 0.0, d, 70_001)
    # 32 terms of a piece, then the pieces in eight shares and the eight sums: 32 + 300000 / 256 + 8 additions at most
    assert_within(d, exact, U * (32 + 300_000 / 256 + 10) * size)


def test_offsets_beyond_32_bits():
    """Rows that begin more than 2^32 bytes (and 2^31 elements) into the table."""
    width, vocab = 4096, 600_000
    table = torch.zeros(vocab, width, dtype=torch.bfloat16, device="cuda")
    table[vocab - 1] = 3.0
    table[550_000] = 5.0
    tokens = torch.tensor([vocab - 1, 0, 550_000], device="cuda")
    y = torch.empty(3, width, dtype=torch.bfloat16, device="cuda")
    ok(spblas.embedding(tokens, table, 1.0, y))
    assert y[:, 0].tolist() == [3.0, 0.0, 5.0] and y[:, -1].tolist() == [3.0, 0.0, 5.0]
    ok(spblas.embedding_grad(tokens, y, 2.0, 1.0, table, buffer_of(spblas.embedding_grad_buffer_size(3, vocab, width))))
    assert float(table[vocab - 1, 7]) == 9.0 and float(table[550_000, 9]) == 15.0 and not table[0].any() and not table[549_999].any()
    del table
    torch.cuda.empty_cache()


def test_table_and_result_in_columns_of_one_block():
    block = normal(gen(2), 9, 64)
    want = block[[7, 0, 3], :32].clone()
    ok(spblas.embedding(torch.tensor([7, 0, 3], device="cuda"), block[:, :32], 1.0, block[:3, 32:]))
    assert torch.equal(block[:3, 32:], want)


def test_refusals_on_the_device():
    t, table, y = torch.zeros(4, dtype=torch.int64, device="cuda"), torch.zeros(9, 8, device="cuda"), torch.zeros(4, 8, device="cuda")
    assert spblas.embedding(t, table, 1.0, table[:4]) == capi.INVALID_VALUE           # the output in the place of the table
    assert spblas.embedding(t.cpu(), table, 1.0, y) == capi.INVALID_POINTER
    assert spblas.embedding(t, table.cpu(), 1.0, y) == capi.INVALID_POINTER
    assert spblas.embedding(t.float(), table, 1.0, y) == capi.INVALID_VALUE
    assert spblas.embedding(t, table.double(), 1.0, y.double()) == capi.INVALID_VALUE
    assert spblas.embedding(t, table, 1.0, y.half()) == capi.INVALID_VALUE
    buffer = buffer_of(spblas.embedding_grad_buffer_size(4, 9, 8))
    small = buffer[: spblas.embedding_grad_buffer_size(4, 9, 8)[1] - 1]
    assert spblas.embedding_grad(t, y, 1.0, 0.0, table, small) == capi.INVALID_VALUE
    assert spblas.embedding_grad(t, y, 1.0, 0.0, table, None) == capi.NOT_INITIALIZED
    assert spblas.embedding_grad(t, y, 1.0, 0.0, table.half(), buffer) == capi.NOT_SUPPORTED
    assert spblas.embedding_grad(t, y, 1.0, 0.0, table, buffer[1:]) == capi.INVALID_VALUE
    ok(spblas.embedding_grad(t, y, 1.0, 0.0, table, buffer))
    empty = torch.empty(0, dtype=torch.int64, device="cuda")
    ok(spblas.embedding(empty, table, 1.0, y[:0]))
    if torch.cuda.device_count() > 1:
        assert spblas.embedding(t, table.to("cuda:1"), 1.0, y) == capi.INVALID_POINTER
