"""The operators on rows as a model uses them together: embedding, routing, the experts' rows and products and back, with
all gradients; recorded in CUDA graphs, on streams of their own and from several threads."""
import math
import subprocess
import sys
import threading

import pytest
import torch

from alsparse_b200 import capi, spblas
from rows_util import choice64, gen, normal, ok, weights64

pytestmark = pytest.mark.gpu
TOKENS, VOCAB, WIDTH, HIDDEN, EXPERTS, TOP = 300, 500, 64, 96, 16, 4


class Layer:
    """One embedding and one layer of experts, with what a program keeps for them."""

    def __init__(self, dtype, seed, tokens=TOKENS):
        g = gen(seed)
        f32, i32 = torch.float32, torch.int32
        self.dtype, self.n = dtype, tokens
        self.tokens = torch.randint(0, VOCAB, (tokens,), generator=g, device="cuda")
        self.tokens[::17] = -1
        self.table = normal(g, VOCAB, WIDTH, dtype=dtype)
        self.gate = normal(g, WIDTH, EXPERTS, by=0.3)
        self.up, self.down = normal(g, EXPERTS, HIDDEN, WIDTH, dtype=dtype, by=0.2), normal(g, EXPERTS, WIDTH, HIDDEN, dtype=dtype, by=0.2)
        self.bias = normal(g, EXPERTS, by=0.1)
        self.dout = normal(g, tokens, WIDTH, dtype=dtype)
        new = lambda *shape, dtype=dtype: torch.zeros(*shape, dtype=dtype, device="cuda")  # noqa: E731
        rows = tokens * TOP
        self.x, self.logits = new(tokens, WIDTH), new(tokens, EXPERTS, dtype=f32)
        self.index, self.weight = new(tokens, TOP, dtype=i32), new(tokens, TOP, dtype=f32)
        self.offsets, self.slot = new(EXPERTS + 1, dtype=i32), new(tokens, TOP, dtype=i32)
        self.xs, self.h, self.y, self.out = new(rows, WIDTH), new(rows, HIDDEN), new(rows, WIDTH), new(tokens, WIDTH)
        self.act = new(rows, HIDDEN)
        self.dy, self.dweight, self.dact, self.dh, self.dxs = new(rows, WIDTH), new(tokens, TOP, dtype=f32), new(rows, HIDDEN), new(rows, HIDDEN), new(rows, WIDTH)
        self.dup, self.ddown = new(EXPERTS, HIDDEN, WIDTH, dtype=f32), new(EXPERTS, WIDTH, HIDDEN, dtype=f32)
        self.dlogits, self.dx, self.dtable = new(tokens, EXPERTS, dtype=f32), new(tokens, WIDTH), new(VOCAB, WIDTH, dtype=f32)
        sizes = spblas.expert_plan_buffer_size(tokens, TOP, EXPERTS), spblas.embedding_grad_buffer_size(tokens, VOCAB, WIDTH)
        self.buffers = [torch.empty(max(n, 16), dtype=torch.uint8, device="cuda") for _, n in sizes]

    def forward(self):
        ok(spblas.embedding(self.tokens, self.table, 1.5, self.x))
        torch.mm(self.x.float(), self.gate, out=self.logits)
        ok(spblas.route(capi.SCORE_SIGMOID, self.logits, self.bias, 4, 2, True, 2.0, self.index, self.weight))
        ok(spblas.expert_plan(self.index, self.offsets, self.slot, self.buffers[0]))
        ok(spblas.expert_dispatch(self.x, self.slot, self.xs))
        ok(spblas.expert_mm(capi.TRANSPOSE, self.offsets, self.xs, self.up, self.h))
        torch.clamp(self.h, min=0, out=self.act)
        ok(spblas.expert_mm(capi.TRANSPOSE, self.offsets, self.act, self.down, self.y))
        ok(spblas.expert_combine(self.y, self.slot, self.weight, 0.0, self.out))

    def backward(self):
        ok(spblas.expert_combine_grad(self.dout, self.y, self.slot, self.weight, self.dy, self.dweight))
        ok(spblas.expert_mm_grad(self.offsets, self.dy, self.act, 0.0, self.ddown))
        ok(spblas.expert_mm(capi.NON_TRANSPOSE, self.offsets, self.dy, self.down, self.dact))
        torch.mul(self.dact, self.h > 0, out=self.dh)
        ok(spblas.expert_mm_grad(self.offsets, self.dh, self.xs, 0.0, self.dup))
        ok(spblas.expert_mm(capi.NON_TRANSPOSE, self.offsets, self.dh, self.up, self.dxs))
        ok(spblas.route_grad(capi.SCORE_SIGMOID, self.logits, self.index, True, 2.0, self.dweight, self.dlogits))
        # the rows' way back to the tokens, on top of the router's part
        self.dx.copy_(self.dlogits @ self.gate.t())
        ok(spblas.expert_combine(self.dxs, self.slot, None, 1.0, self.dx))
        ok(spblas.embedding_grad(self.tokens, self.dx, 1.5, 0.0, self.dtable, self.buffers[1]))

    RESULTS = ("x", "logits", "index", "weight", "offsets", "slot", "out", "dweight", "ddown", "dup", "dlogits", "dx", "dtable")

    def results(self):
        return [getattr(self, n).clone() for n in self.RESULTS]


def _reference(s):
    """The same layer in 64 bits, rounded to the layer's type where it stores its tensors."""
    r = lambda t: t.to(s.dtype).double()  # noqa: E731
    inside = (s.tokens >= 0)[:, None]
    x = r(torch.where(inside, s.table.double()[s.tokens.clamp(min=0)] * 1.5, 0.0))
    logits = (x @ s.gate.double()).requires_grad_()
    index = choice64(s.logits, s.bias, capi.SCORE_SIGMOID, 4, 2, TOP)
    w = weights64(logits, index, capi.SCORE_SIGMOID, True, 2.0)
    at = index.long()
    h = r(torch.einsum("td,tkhd->tkh", x, s.up.double()[at]))
    act = h.clamp(min=0)
    y = r(torch.einsum("tkh,tkdh->tkd", act, s.down.double()[at]))
    dout = s.dout.double()
    out = torch.einsum("tk,tkd->td", w.detach(), y)
    dw = torch.einsum("td,tkd->tk", dout, y)
    dy = r(w.detach()[:, :, None] * dout[:, None, :])
    one = torch.nn.functional.one_hot(at, EXPERTS).double()
    ddown = torch.einsum("tke,tkd,tkh->edh", one, dy, act)
    dh = r(torch.einsum("tkd,tkdh->tkh", dy, s.down.double()[at])) * (h > 0)
    dup = torch.einsum("tke,tkh,td->ehd", one, dh, x)
    dxs = r(torch.einsum("tkh,tkhd->tkd", dh, s.up.double()[at]))
    dlogits = torch.autograd.grad((w * dw).sum(), logits)[0]
    dx = r(r(dlogits @ s.gate.double().t()) + dxs.sum(1))
    dtable = torch.zeros(VOCAB, WIDTH, dtype=torch.float64, device="cuda")
    dtable.index_add_(0, s.tokens.clamp(min=0), torch.where(inside, 1.5 * dx, 0.0))
    return {"x": x, "logits": logits.detach(), "index": index, "weight": w.detach(), "out": out, "dweight": dw, "ddown": ddown, "dup": dup, "dlogits": dlogits,
            "dx": dx, "dtable": dtable}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_forward_and_backward(dtype):
    s = Layer(dtype, 1)
    s.forward()
    s.backward()
    want = _reference(s)
    assert torch.equal(s.index, want["index"])
    # Both sides round to the type at the same places, so what differs is the order of sums of at most 300 terms in 32 bits (2e-5)
    # and, where a value lies next to a border, one step of the type: at most one step in the norm, in each of the up to
    # four roundings that a gradient has behind it.
    step = max(4 * torch.finfo(dtype).eps, 1e-4)
    for name, exact in want.items():
        got = getattr(s, name).double()
        if name != "index":
            assert float((got - exact).norm()) <= step * float(exact.norm()), name
    assert spblas.expert_mm_status() == (capi.SUCCESS, 0)


def _on_stream(stream):
    spblas.set_stream(stream.cuda_stream)
    return torch.cuda.stream(stream)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_recorded_and_replayed_with_new_inputs(dtype):
    s, other = Layer(dtype, 2), Layer(dtype, 3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    try:
        with _on_stream(side):
            s.forward()
            s.backward()
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                s.forward()
                s.backward()
            for name in ("tokens", "table", "bias", "dout", "up", "gate"):   # another batch, through the same graph
                getattr(s, name).copy_(getattr(other, name))
            s.down.copy_(other.down)
            graph.replay()
            graph.replay()
            replayed = s.results()
            side.synchronize()
            other.forward()
            other.backward()
            direct = other.results()
            side.synchronize()
    finally:
        spblas.set_stream(None)
    for name, a, b in zip(Layer.RESULTS, replayed, direct):
        assert torch.equal(a, b), name


def test_two_graphs_at_the_same_time():
    """Each with its own workspaces: nothing is shared between calls."""
    layers = [Layer(torch.bfloat16, 4, tokens=1500), Layer(torch.bfloat16, 5, tokens=1500)]
    streams, graphs, want = [torch.cuda.Stream(), torch.cuda.Stream()], [], []
    torch.cuda.synchronize()
    try:
        for s, stream in zip(layers, streams):
            with _on_stream(stream):
                s.forward()
                s.backward()
                want.append(s.results())
                stream.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=stream):
                    s.forward()
                    s.backward()
                graphs.append(graph)
    finally:
        spblas.set_stream(None)
    for s in layers:
        for name in Layer.RESULTS:
            getattr(s, name).zero_()
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for s, results in zip(layers, want):
        for name, a, b in zip(Layer.RESULTS, s.results(), results):
            assert torch.equal(a, b), name


def test_calls_from_several_threads():
    """The library stream belongs to the process; calls of several threads on it are complete calls."""
    layers = [Layer(torch.bfloat16, 10 + i) for i in range(4)]
    want = []
    for s in layers:
        s.forward()
        s.backward()
        want.append(s.results())
    torch.cuda.synchronize()
    errors = []

    def work(s):
        try:
            for _ in range(5):
                s.forward()
                s.backward()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(s,)) for s in layers]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors
    for s, results in zip(layers, want):
        for name, a, b in zip(Layer.RESULTS, s.results(), results):
            assert torch.equal(a, b), name


def test_recorded_before_any_other_call():
    """The first calls of a process may be the recorded ones."""
    code = """
import sys, torch
sys.path[:0] = ["tests", "."]
from alsparse_b200 import spblas
import test_gpu_operators_chain as t
s = t.Layer(torch.bfloat16, 6)
torch.mm(s.x.float(), s.gate); s.dlogits @ s.gate.t()
side = torch.cuda.Stream()
torch.cuda.synchronize()
spblas.set_stream(side.cuda_stream)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=side):
    s.forward(); s.backward()
graph.replay(); torch.cuda.synchronize()
got = s.results()
with torch.cuda.stream(side):
    s.forward(); s.backward()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, s.results()))
print("as recorded")
"""
    p = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert p.returncode == 0 and "as recorded" in p.stdout, p.stdout + p.stderr


def test_a_decoding_step_of_one_token():
    s = Layer(torch.bfloat16, 8, tokens=1)
    s.tokens[0] = 3
    s.forward()
    s.backward()
    want = _reference(s)
    assert torch.equal(s.index, want["index"])
    for name in ("out", "dup", "ddown", "dx"):
        assert float((getattr(s, name).double() - want[name]).norm()) <= 4 * torch.finfo(torch.bfloat16).eps * float(want[name].norm()), name


def test_tokens_without_an_expert():
    """Rows whose logits are all masked go nowhere: their outputs and gradients are zero, the others are as without them."""
    s = Layer(torch.bfloat16, 9)
    ok(spblas.embedding(s.tokens, s.table, 1.0, s.x))
    s.logits.copy_(s.x.float() @ s.gate)
    s.logits[100:] = -math.inf
    ok(spblas.route(capi.SCORE_SIGMOID, s.logits, s.bias, 4, 2, True, 2.0, s.index, s.weight))
    ok(spblas.expert_plan(s.index, s.offsets, s.slot, s.buffers[0]))
    s.xs.fill_(math.nan)
    ok(spblas.expert_dispatch(s.x, s.slot, s.xs))
    s.h.fill_(math.nan)
    ok(spblas.expert_mm(capi.TRANSPOSE, s.offsets, s.xs, s.up, s.h))
    assert int(s.offsets[-1]) == 100 * TOP and bool(s.h[: 100 * TOP].isfinite().all()) and bool(s.h[100 * TOP:].isnan().all())
    torch.clamp(s.h, min=0, out=s.act)
    ok(spblas.expert_mm(capi.TRANSPOSE, s.offsets, s.act, s.down, s.y))
    s.y[100 * TOP:] = math.nan
    s.out.fill_(math.nan)
    ok(spblas.expert_combine(s.y, s.slot, s.weight, 0.0, s.out))
    assert bool(s.out.isfinite().all()) and not s.out[100:].any()
    s.dy[100 * TOP:] = math.nan
    ok(spblas.expert_combine_grad(s.dout, s.y, s.slot, s.weight, s.dy, s.dweight))
    assert not s.dweight[100:].any()
    ok(spblas.expert_mm_grad(s.offsets, s.dy, s.act, 0.0, s.ddown))
    assert bool(s.ddown.isfinite().all())
