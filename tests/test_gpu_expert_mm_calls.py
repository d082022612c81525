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
