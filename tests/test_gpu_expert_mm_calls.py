"""Calls of the experts' products beside other calls: several threads with different sizes, the status word, recorded calls."""
import threading

import pytest
import torch

from alsparse_b200 import capi, spblas
from rows_util import gen, normal, ok

pytestmark = pytest.mark.gpu


def _product(g, rows, experts=4, out=64, inner=64):
    x, w = normal(g, rows, inner, dtype=torch.bfloat16), normal(g, experts, out, inner, dtype=torch.bfloat16)
    offsets = torch.arange(experts + 1, dtype=torch.int32, device="cuda") * (rows // experts)
    return offsets, x, w, torch.zeros(rows, out, dtype=torch.bfloat16, device="cuda")


def test_status_is_refused_while_recording_and_the_recording_goes_on():
    offsets, x, w, y = _product(gen(1), 64)
    ok(spblas.expert_mm(capi.TRANSPOSE, offsets, x, w, y))
    want = y.clone()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    spblas.set_stream(side.cuda_stream)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            ok(spblas.expert_mm(capi.TRANSPOSE, offsets, x, w, y))
            assert [spblas.expert_mm_status(clear)[0] for clear in (False, True)] == [capi.EXECUTION_FAILED] * 2
            assert "captured" in spblas.last_error()
        y.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
        assert spblas.expert_mm_status(True) == (capi.SUCCESS, 0) == spblas.expert_mm_status()
    finally:
        spblas.set_stream(None)


def test_status_from_several_threads():
    seen = []

    def ask():
        for i in range(200):
            seen.append(spblas.expert_mm_status(i % 2 == 0))

    threads = [threading.Thread(target=ask) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert seen == [(capi.SUCCESS, 0)] * 800


@pytest.mark.parametrize("which", ["product", "gradient", "status"])
def test_first_call_of_a_thread(which):
    """Nothing else of CUDA has been called in it."""
    offsets, x, w, y = _product(gen(2), 64)
    dw = torch.zeros(4, 64, 64, device="cuda")
    call = {"product": lambda: spblas.expert_mm(capi.TRANSPOSE, offsets, x, w, y), "gradient": lambda: spblas.expert_mm_grad(offsets, y, x, 0.0, dw),
            "status": lambda: spblas.expert_mm_status()[0]}[which]
    torch.cuda.synchronize()
    seen = []
    thread = threading.Thread(target=lambda: seen.append((call(), spblas.last_error())))
    thread.start()
    thread.join()
    assert seen[0][0] == capi.SUCCESS, seen
    torch.cuda.synchronize()
    if which == "product":
        here = torch.zeros_like(y)
        ok(spblas.expert_mm(capi.TRANSPOSE, offsets, x, w, here))
        assert torch.equal(here, y)


@pytest.mark.parametrize("op", [capi.TRANSPOSE, capi.NON_TRANSPOSE])
def test_threads_with_different_sizes(op):
    """Few rows an expert and more of them take tiles, and shared memory, of different sizes."""
    calls = [_product(gen(rows), rows) for rows in (32, 128, 240, 32)]
    want = []
    for c in calls:
        ok(spblas.expert_mm(op, *c))
        want.append(c[3].clone())
        c[3].zero_()
    torch.cuda.synchronize()
    refused = []

    def work(c):
        for _ in range(4000):
            status = spblas.expert_mm(op, *c)
            if status != capi.SUCCESS:
                refused.append((status, spblas.last_error()))

    threads = [threading.Thread(target=work, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not refused, (len(refused), refused[0])
    for c, y in zip(calls, want):
        assert torch.equal(c[3], y)


@pytest.mark.parametrize("out_type", [torch.bfloat16, torch.float32])
def test_threads_with_different_gradients(out_type):
    """Narrow and wide columns of dy: stages of different sizes."""
    calls = []
    for out in (32, 96, 256):
        g = gen(out)
        offsets = torch.tensor([0, 20, 20, 70], dtype=torch.int32, device="cuda")
        calls.append((offsets, normal(g, 70, out, dtype=torch.bfloat16), normal(g, 70, 64, dtype=torch.bfloat16), 0.0,
                      torch.zeros(3, out, 64, dtype=out_type, device="cuda")))
    want = []
    for c in calls:
        ok(spblas.expert_mm_grad(*c))
        want.append(c[4].clone())
        c[4].zero_()
    torch.cuda.synchronize()
    refused = []

    def work(c):
        for _ in range(4000):
            status = spblas.expert_mm_grad(*c)
            if status != capi.SUCCESS:
                refused.append((status, spblas.last_error()))

    threads = [threading.Thread(target=work, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not refused, (len(refused), refused[0])
    for c, d in zip(calls, want):
        assert torch.equal(c[4], d)
