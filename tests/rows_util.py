"""Helpers for the tests of the operators on rows (embedding, routing, experts): inputs, bounds, plain results in 64 bits."""
import math

import torch

from alsparse_b200 import capi, spblas

TYPES = [torch.float32, torch.float16, torch.bfloat16]
U = 2.0 ** -24  # half a step of a 32-bit sum


def ok(status):
    assert status == capi.SUCCESS, (capi.STATUS_NAMES[status], spblas.last_error())


def half_step(t):
    """The rounding to type t is off by at most this, relative to the value."""
    return torch.finfo(t).eps / 2


def floor_of(t):
    """... or by this, where the value is below the type's normal numbers."""
    return torch.finfo(t).tiny * torch.finfo(t).eps


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(g, *shape, dtype=torch.float32, by=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * by).to(dtype)


def strided(t, ld, shift=0):
    """The rows of t, ld elements apart, `shift` elements behind the start of an allocation whose other elements are NaN."""
    rows, width = t.shape
    assert ld >= width
    space = torch.full((rows * ld + shift + 8,), math.nan, dtype=t.dtype, device="cuda") if t.is_floating_point() else \
        torch.full((rows * ld + shift + 8,), -7, dtype=t.dtype, device="cuda")
    view = torch.as_strided(space, (rows, width), (ld, 1), shift)
    view.copy_(t)
    return view, space


def untouched(view, space, before):
    """Elements of `space` outside `view` are as they were."""
    mask = torch.ones_like(space, dtype=torch.bool)
    torch.as_strided(mask, view.shape, view.stride(), view.storage_offset()).fill_(False)
    a, b = space[mask], before[mask]
    return bool(((a == b) | ((a != a) & (b != b))).all())


def assert_within(got, exact, bound, what=""):
    """|got - exact| <= bound, element by element; NaN where exact is NaN, infinities equal."""
    got, exact = got.double(), exact.double()
    bound = torch.as_tensor(bound, dtype=torch.float64, device=got.device).expand_as(exact)
    nan = exact.isnan()
    assert torch.equal(got.isnan(), nan), f"{what}: NaN in other places"
    inf = exact.isinf()
    assert torch.equal(got[inf], exact[inf]), f"{what}: infinities differ"
    fine = ~nan & ~inf
    off = (got - exact).abs()[fine]
    over = off > bound[fine]
    assert not bool(over.any()), f"{what}: {int(over.sum())} of {off.numel()} beyond the bound, worst {float((off / bound[fine].clamp(min=1e-300)).max()):.3g} times"


def buffer_of(size):
    ok(size[0])
    return torch.full((size[1] + 64,), 0xA5, dtype=torch.uint8, device="cuda")


def choice64(logits, bias, score, groups, top_groups, k):
    """The experts of each row, by keys in 64 bits."""
    x = logits.double()
    masked = x == -math.inf
    key = x.clone()
    if bias is not None:
        top = x.amax(1, keepdim=True)
        e = torch.where(masked, 0.0, torch.exp(x - torch.where(top == -math.inf, 0.0, top)))
        s = torch.sigmoid(x) if score == capi.SCORE_SIGMOID else e / e.sum(1, keepdim=True)
        key = torch.where(masked, -math.inf, s + bias.double())
    if top_groups < groups:
        part = key.view(key.shape[0], groups, -1)
        best = part.sort(dim=2, descending=True).values
        worth = best[:, :, 0]
        if bias is not None and best.shape[2] > 1:
            worth = worth + torch.where(best[:, :, 1] == -math.inf, 0.0, best[:, :, 1])
        kept = torch.zeros_like(worth, dtype=torch.bool)
        kept.scatter_(1, worth.sort(dim=1, descending=True, stable=True).indices[:, :top_groups], True)
        key = torch.where(kept[:, :, None], part, -math.inf).reshape(key.shape)
    best = key.sort(dim=1, descending=True, stable=True)
    return torch.where(best.values[:, :k] == -math.inf, -1, best.indices[:, :k]).int()


def weights64(logits, index, score, renorm, scale):
    """Weights of the chosen experts; differentiable where logits are."""
    x = logits.double()
    some = index >= 0
    v = x.gather(1, index.clamp(min=0).long())
    if renorm:
        # as shares of the chosen: by the logarithms of the scores
        log_s = torch.nn.functional.logsigmoid(v) if score == capi.SCORE_SIGMOID else v
        log_s = torch.where(some, log_s, -math.inf)
        top = log_s.amax(1, keepdim=True).detach()
        e = torch.where(some, torch.exp(log_s - torch.where(top == -math.inf, 0.0, top)), 0.0)
        total = e.sum(1, keepdim=True)
        w = torch.where(some, e / torch.where(total == 0, 1.0, total), 0.0)
    elif score == capi.SCORE_SIGMOID:
        w = torch.where(some, torch.sigmoid(v), 0.0)
    else:
        dead = (x == -math.inf).all(1, keepdim=True)
        w = torch.where(some, torch.softmax(torch.where(dead, 0.0, x), 1).gather(1, index.clamp(min=0).long()), 0.0)
    return w * scale


def plan64(index, experts):
    """(offsets, slot) by a walk over the pairs on the host."""
    rows = [[] for _ in range(experts)]
    flat = index.reshape(-1).tolist()
    for i, e in enumerate(flat):
        if 0 <= e < experts:
            rows[e].append(i)
    offsets, slot = [0], [-1] * len(flat)
    for r in rows:
        for i, at in enumerate(r):
            slot[at] = offsets[-1] + i
        offsets.append(offsets[-1] + len(r))
    return torch.tensor(offsets, dtype=torch.int32), torch.tensor(slot, dtype=torch.int32).view(index.shape)
