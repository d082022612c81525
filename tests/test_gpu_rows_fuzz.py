"""Seeded random shapes, types, strides and alignments through the operators on rows, against the same sums in 64 bits; what
lies around the outputs is compared too."""
import random

import pytest
import torch

from alsparse_b200 import capi, spblas
from rows_util import TYPES, U, assert_within, buffer_of, choice64, floor_of, gen, half_step, normal, ok, plan64, strided, untouched, weights64

pytestmark = pytest.mark.gpu


def _size(rng, lo, hi):
    return max(lo, min(hi, int(lo * (hi / lo) ** rng.random())))


def _place(rng, t):
    """t in rows of a random length and at a random place; half of the time aligned to 16 bytes."""
    if rng.random() < 0.5:
        unit = 16 // t.element_size()
        ld = -(-t.shape[1] // unit) * unit + unit * rng.randint(0, 2)
        return strided(t, ld, unit * rng.randint(0, 3))
    return strided(t, t.shape[1] + rng.randint(0, 9), rng.randint(0, 9))


@pytest.mark.parametrize("seed", range(40))
def test_embedding_and_gradient(seed):
    rng, g = random.Random(seed), gen(seed)
    dtype, index = rng.choice(TYPES), rng.choice([torch.int32, torch.int64])
    vocab, width, count = _size(rng, 1, 5000), _size(rng, 1, 3000), _size(rng, 1, 3000)
    tokens = torch.randint(-1, vocab + 1, (count * 2,), generator=g, device="cuda")
    tokens[torch.rand(count * 2, generator=g, device="cuda") < rng.choice([0.0, 0.5, 0.95])] = vocab // 2
    tokens = tokens.to(index)[::2]
    inside = (tokens >= 0) & (tokens < vocab)
    table, _ = _place(rng, normal(g, vocab, width, dtype=dtype))
    y, space = _place(rng, torch.zeros(count, width, dtype=dtype, device="cuda"))
    before, scale = space.clone(), rng.choice([1.0, -1.75])
    ok(spblas.embedding(tokens, table, scale, y))
    exact = torch.where(inside[:, None], table.double()[tokens.long().clamp(0, vocab - 1)] * scale, 0.0)
    assert_within(y, exact, (half_step(dtype) + 2 * U) * exact.abs() + floor_of(dtype))
    assert untouched(y, space, before)
    out, alpha, beta = rng.choice([dtype, torch.float32]), rng.choice([1.0, 0.5]), rng.choice([0.0, 1.0, -0.5])
    dy, _ = _place(rng, normal(g, count, width, dtype=dtype))
    d, space = _place(rng, normal(g, vocab, width, dtype=out))
    old, before = d.double().clone(), space.clone()
    ok(spblas.embedding_grad(tokens, dy, alpha, beta, d, buffer_of(spblas.embedding_grad_buffer_size(count, vocab, width))))
    total, size = torch.zeros_like(old), torch.zeros_like(old)
    total.index_add_(0, tokens[inside].long(), dy[inside].double())
    size.index_add_(0, tokens[inside].long(), dy[inside].double().abs())
    exact = alpha * total + beta * old
    # 32 terms of a piece, the pieces in eight shares or one after the other, and the two products
    terms = min(count, 32 + count / 32 + 10)
    bound = U * (terms * alpha * size + 3 * abs(beta) * old.abs())
    assert_within(d, exact, bound + half_step(out) * (exact.abs() + bound) + floor_of(out))
    assert untouched(d, space, before)


@pytest.mark.parametrize("seed", range(40))
def test_routing(seed):
    rng, g = random.Random(1000 + seed), gen(seed)
    dtype, score = rng.choice(TYPES), rng.choice([capi.SCORE_SOFTMAX, capi.SCORE_SIGMOID])
    groups = rng.choice([1, 1, 2, 3, 5, 8, 16, 32])
    each = _size(rng, 1, 1024 // groups)
    experts, top = groups * each, rng.randint(1, groups)
    tokens, k = _size(rng, 1, 600), rng.randint(1, min(32, top * each))
    x = normal(g, tokens, experts, by=rng.choice([0.1, 2.0, 20.0]))
    x[torch.rand(tokens, experts, generator=g, device="cuda") < rng.choice([0.0, 0.2, 0.9])] = -float("inf")
    logits, _ = _place(rng, x.to(dtype))
    bias = normal(g, experts, by=rng.choice([0.0, 0.01, 0.5])) if rng.random() < 0.6 else None
    renorm, scale = rng.random() < 0.5, rng.choice([1.0, 2.5])
    index, si = _place(rng, torch.zeros(tokens, k, dtype=torch.int32, device="cuda"))
    weight, sw = _place(rng, torch.zeros(tokens, k, device="cuda"))
    bi, bw = si.clone(), sw.clone()
    ok(spblas.route(score, logits, bias, groups, top, renorm, scale, index, weight))
    assert torch.equal(index, choice64(logits, bias, score, groups, top, k))
    exact = weights64(logits, index, score, renorm, scale)
    spread = 2 * torch.where(logits.isfinite(), logits.float().abs(), 0.0).amax(1, keepdim=True).double().clamp(max=104)
    relative = U * (2 * spread + 16 + experts / 32 + 5 + k)
    assert_within(weight, exact, relative * exact + 2.0 ** -126)
    assert untouched(index, si, bi) and untouched(weight, sw, bw)
    dweight, _ = _place(rng, normal(g, tokens, k))
    d, sd = _place(rng, torch.zeros(tokens, experts, dtype=dtype, device="cuda"))
    bd = sd.clone()
    ok(spblas.route_grad(score, logits, index, renorm, scale, dweight, d))
    leaf = torch.where(logits == -float("inf"), -1e30, logits.double()).requires_grad_()
    clean = torch.where(index < 0, 0.0, dweight).double()
    grad = torch.autograd.grad((weights64(leaf, index, score, renorm, scale) * clean).sum(), leaf)[0]
    grad = torch.where(logits == -float("inf"), 0.0, grad)
    assert_within(d, grad, 4 * relative * scale * clean.abs().sum(1, keepdim=True) + half_step(dtype) * grad.abs() + floor_of(dtype))
    assert untouched(d, sd, bd)


@pytest.mark.parametrize("seed", range(40))
def test_rows_of_experts(seed):
    rng, g = random.Random(2000 + seed), gen(seed)
    dtype = rng.choice(TYPES)
    tokens, k, experts, width = _size(rng, 1, 2000), rng.randint(1, 12), _size(rng, 1, 1024), _size(rng, 1, 2500)
    index, _ = _place(rng, torch.randint(-1, experts + 1, (tokens, k), generator=g, device="cuda", dtype=torch.int32))
    offsets = torch.empty(experts + 1, dtype=torch.int32, device="cuda")
    slot, ss = _place(rng, torch.zeros(tokens, k, dtype=torch.int32, device="cuda"))
    before = ss.clone()
    ok(spblas.expert_plan(index, offsets, slot, buffer_of(spblas.expert_plan_buffer_size(tokens, k, experts))))
    want = plan64(index.cpu(), experts)
    assert torch.equal(offsets.cpu(), want[0]) and torch.equal(slot.cpu(), want[1]) and untouched(slot, ss, before)
    x, _ = _place(rng, normal(g, tokens, width, dtype=dtype))
    xs, space = _place(rng, torch.full((tokens * k, width), 7.0, dtype=dtype, device="cuda"))
    before = space.clone()
    ok(spblas.expert_dispatch(x, slot, xs))
    some = slot.reshape(-1) >= 0
    full = torch.full((tokens * k, width), 7.0, dtype=dtype, device="cuda")
    full[slot.reshape(-1)[some].long()] = x.repeat_interleave(k, 0)[some]
    assert torch.equal(xs, full) and untouched(xs, space, before)
    weight = normal(g, tokens, k) if rng.random() < 0.7 else None
    out, space = _place(rng, normal(g, tokens, width, dtype=dtype))
    old, before, beta = out.double().clone(), space.clone(), rng.choice([0.0, 1.0, 0.5])
    ok(spblas.expert_combine(xs, slot, weight, beta, out))
    w = torch.where(slot >= 0, 1.0 if weight is None else weight.double(), 0.0)
    rows = xs.double()[slot.clamp(min=0).long()]
    exact, size = (rows * w[:, :, None]).sum(1) + beta * old, (rows * w[:, :, None]).abs().sum(1) + beta * old.abs()
    bound = U * (k + 2) * size
    assert_within(out, exact, bound + half_step(dtype) * (exact.abs() + bound) + floor_of(dtype))
    assert untouched(out, space, before)
    dout, _ = _place(rng, normal(g, tokens, width, dtype=dtype))
    dy, space = _place(rng, torch.full((tokens * k, width), 7.0, dtype=dtype, device="cuda"))
    before = space.clone()
    dweight = torch.full((tokens, k), float("nan"), device="cuda")
    ok(spblas.expert_combine_grad(dout, xs, slot, weight, dy, dweight))
    exact = torch.full((tokens * k, width), 7.0, dtype=torch.float64, device="cuda")
    exact[slot.reshape(-1)[some].long()] = (w[:, :, None] * dout.double()[:, None, :]).reshape(-1, width)[some]
    assert_within(dy, exact, (half_step(dtype) + 2 * U) * exact.abs() + floor_of(dtype))
    assert untouched(dy, space, before)
    there = (slot >= 0)[:, :, None]
    exact = torch.where(there, rows * dout.double()[:, None, :], 0.0)
    assert_within(dweight, exact.sum(2), U * (width + 8) * exact.abs().sum(2))


@pytest.mark.parametrize("seed", range(40))
def test_experts_products(seed):
    rng, g = random.Random(3000 + seed), gen(seed)
    dtype = rng.choice([torch.bfloat16, torch.float16, torch.bfloat16, torch.float16, torch.float32])
    experts, out, inner = _size(rng, 1, 40), _size(rng, 1, 700), _size(rng, 1, 700)
    counts = [0 if rng.random() < 0.2 else _size(rng, 1, rng.choice([4, 40, 400])) for _ in range(experts)]
    first, rows = rng.randint(0, 5), 0
    o = [first]
    for c in counts:
        o.append(o[-1] + c)
    rows = o[-1] + rng.randint(0, 5)
    if rows == 0:
        rows = 1
    offsets = torch.tensor(o, dtype=torch.int32, device="cuda")
    w, _ = _place(rng, normal(g, experts * out, inner, dtype=dtype))
    w = torch.as_strided(w, (experts, out, inner), (out * w.stride(0), w.stride(0), 1), w.storage_offset())
    for op in (capi.TRANSPOSE, capi.NON_TRANSPOSE):
        x, _ = _place(rng, normal(g, rows, inner if op == capi.TRANSPOSE else out, dtype=dtype))
        y, space = _place(rng, torch.full((rows, out if op == capi.TRANSPOSE else inner), 7.0, dtype=dtype, device="cuda"))
        before = space.clone()
        ok(spblas.expert_mm(op, offsets, x, w, y))
        exact = torch.full(y.shape, 7.0, dtype=torch.float64, device="cuda")
        bound = torch.zeros_like(exact)
        for e in range(experts):
            m = w[e].double().t() if op == capi.TRANSPOSE else w[e].double()
            r = slice(o[e], o[e + 1])
            exact[r] = x[r].double() @ m
            bound[r] = 2 * U * (x.shape[1] + 8) * (x[r].double().abs() @ m.abs())
        assert_within(y, exact, bound + half_step(dtype) * (exact.abs() + bound) + floor_of(dtype))
        assert untouched(y, space, before)
    dy, _ = _place(rng, normal(g, rows, out, dtype=dtype))
    x, _ = _place(rng, normal(g, rows, inner, dtype=dtype))
    kind, beta = rng.choice([dtype, torch.float32]), rng.choice([0.0, 0.0, 0.5])
    d, space = _place(rng, normal(g, experts * out, inner, dtype=kind))
    before = space.clone()
    dw = torch.as_strided(d, (experts, out, inner), (out * d.stride(0), d.stride(0), 1), d.storage_offset())
    old = dw.double().clone()
    ok(spblas.expert_mm_grad(offsets, dy, x, beta, dw))
    for e in range(experts):
        r = slice(o[e], o[e + 1])
        a, b = dy[r].double().t(), x[r].double()
        exact, size = a @ b + beta * old[e], a.abs() @ b.abs() + beta * old[e].abs()
        bound = 2 * U * (counts[e] + 8) * size
        assert_within(dw[e], exact, bound + half_step(kind) * (exact.abs() + bound) + floor_of(kind), f"dw {e}")
    assert untouched(d, space, before)
    assert spblas.expert_mm_status() == (capi.SUCCESS, 0)
