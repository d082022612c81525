"""Refusals of the operators on rows that need no device: sizes, enums, missing operands, shapes of the Python calls."""
import ctypes as C

import numpy as np
import pytest

from alsparse_b200 import capi, spblas

A = 1 << 20  # an address that no check looks behind


def call(name, *args):
    return getattr(capi.load(), "alphasparse_cuda_" + name)(*args)


@pytest.mark.parametrize("change,want", [({0: 5}, capi.INVALID_VALUE), ({1: 7}, capi.INVALID_VALUE), ({2: -1}, capi.INVALID_VALUE), ({2: 1 << 31}, capi.INVALID_VALUE),
                                         ({4: 0}, capi.INVALID_VALUE), ({5: -1}, capi.INVALID_VALUE), ({6: -1}, capi.INVALID_VALUE), ({6: 1 << 25}, capi.INVALID_VALUE),
                                         ({3: None}, capi.NOT_INITIALIZED), ({8: None}, capi.NOT_INITIALIZED), ({10: None}, capi.NOT_INITIALIZED),
                                         ({9: 7}, capi.INVALID_VALUE), ({11: 7}, capi.INVALID_VALUE), ({9: 1 << 31}, capi.INVALID_VALUE), ({8: A + 2}, capi.INVALID_VALUE),
                                         ({10: A + 16}, capi.INVALID_VALUE), ({2: 0, 3: None, 10: None}, capi.SUCCESS), ({6: 0}, capi.SUCCESS)])
def test_embedding(change, want):
    args = [capi.INDEX_I64, capi.TYPE_F32, 4, 3 * A, 1, 9, 8, 1.0, A, 8, 2 * A, 8]
    for at, v in change.items():
        args[at] = v
    assert call("embedding", *args) == want


@pytest.mark.parametrize("change,want", [({2: capi.TYPE_F16}, capi.NOT_SUPPORTED), ({2: 9}, capi.INVALID_VALUE), ({5: 0}, capi.INVALID_VALUE), ({4: None}, capi.NOT_INITIALIZED),
                                         ({9: None}, capi.NOT_INITIALIZED), ({12: None}, capi.NOT_INITIALIZED), ({14: None}, capi.NOT_INITIALIZED), ({15: 16}, capi.INVALID_VALUE),
                                         ({14: 5 * A + 8}, capi.INVALID_VALUE), ({12: 2 * A}, capi.INVALID_VALUE), ({6: 0, 12: None}, capi.SUCCESS), ({7: 0}, capi.SUCCESS)])
def test_embedding_grad(change, want):
    args = [capi.INDEX_I64, capi.TYPE_F32, capi.TYPE_F32, 4, 3 * A, 1, 9, 8, 1.0, 2 * A, 8, 0.0, 4 * A, 8, 5 * A, 1 << 16]
    for at, v in change.items():
        args[at] = v
    assert call("embedding_grad", *args) == want


@pytest.mark.parametrize("change,want", [({0: 2}, capi.INVALID_VALUE), ({1: 3}, capi.INVALID_VALUE), ({2: -1}, capi.INVALID_VALUE), ({3: 0}, capi.INVALID_VALUE),
                                         ({3: 2048, 5: 2048}, capi.NOT_SUPPORTED), ({7: 3}, capi.INVALID_VALUE), ({7: 0}, capi.INVALID_VALUE), ({8: 0}, capi.INVALID_VALUE),
                                         ({8: 9}, capi.INVALID_VALUE), ({9: 0}, capi.INVALID_VALUE), ({9: 40}, capi.NOT_SUPPORTED), ({9: 17}, capi.INVALID_VALUE),
                                         ({7: 64}, capi.NOT_SUPPORTED), ({4: None}, capi.NOT_INITIALIZED), ({12: None}, capi.NOT_INITIALIZED), ({14: None}, capi.NOT_INITIALIZED),
                                         ({5: 63}, capi.INVALID_VALUE), ({13: 7}, capi.INVALID_VALUE), ({14: A + 4}, capi.INVALID_VALUE), ({2: 0, 4: None}, capi.SUCCESS)])
def test_route(change, want):
    args = [capi.SCORE_SIGMOID, capi.TYPE_F32, 4, 64, A, 64, None, 8, 2, 8, 1, 1.0, 2 * A, 8, 3 * A, 8]
    if 9 in change and change[9] == 40:
        args[7] = args[8] = 1
    if change.get(7) == 64:
        args[8] = 64
    for at, v in change.items():
        args[at] = v
    assert call("route", *args) == want


def test_route_grad_and_the_calls_on_rows():
    assert call("route_grad", 0, 0, 4, 64, A, 64, 8, None, 8, 1, 1.0, 2 * A, 8, 3 * A, 64) == capi.NOT_INITIALIZED
    assert call("route_grad", 0, 0, 4, 64, A, 64, 8, 4 * A, 8, 1, 1.0, 2 * A, 8, A, 64) == capi.INVALID_VALUE
    assert call("route_grad", 0, 0, 4, 64, A, 64, 65, 4 * A, 65, 1, 1.0, 2 * A, 65, 3 * A, 64) == capi.INVALID_VALUE
    assert call("expert_plan", 4, 2, 8, A, 2, 2 * A, 3 * A, 2, None, 0) in (capi.EXECUTION_FAILED, capi.INVALID_POINTER)  # no device, or not its memory
    assert call("expert_plan", 4, 2, 8, A, 2, None, 3 * A, 2, None, 0) == capi.NOT_INITIALIZED
    assert call("expert_plan", 4, 2, 0, A, 2, 2 * A, 3 * A, 2, None, 0) == capi.INVALID_VALUE
    assert call("expert_plan", 4, 2, 2000, A, 2, 2 * A, 3 * A, 2, None, 0) == capi.NOT_SUPPORTED
    assert call("expert_plan", 1 << 30, 4, 8, A, 4, 2 * A, 3 * A, 4, None, 0) == capi.INVALID_VALUE
    assert call("expert_plan", 9000, 2, 8, A, 2, 2 * A, 3 * A, 2, 4 * A, 16) == capi.INVALID_VALUE      # workspace too small
    assert call("expert_dispatch", 0, 4, 2, 8, None, 8, A, 2, 8, 2 * A, 8) == capi.NOT_INITIALIZED
    assert call("expert_dispatch", 0, 4, 0, 8, 3 * A, 8, A, 2, 8, 2 * A, 8) == capi.INVALID_VALUE
    assert call("expert_dispatch", 0, 4, 2, 8, 3 * A, 8, A, 2, -1, 2 * A, 8) == capi.INVALID_VALUE
    assert call("expert_dispatch", 4, 4, 2, 8, 3 * A, 8, A, 2, 8, 2 * A, 8) == capi.INVALID_VALUE
    assert call("expert_combine", 0, 4, 2, 8, 8, A, 8, None, 2, None, 0, 0.0, 2 * A, 8) == capi.NOT_INITIALIZED
    assert call("expert_combine", 0, 4, 2, 8, 8, A, 8, 3 * A, 2, 4 * A, 1, 0.0, 2 * A, 8) == capi.INVALID_VALUE
    assert call("expert_combine_grad", 0, 4, 2, 8, 8, A, 8, 2 * A, 8, 3 * A, 2, None, 0, 2 * A, 8, 5 * A, 2) == capi.INVALID_VALUE
    assert call("expert_combine_grad", 0, 0, 2, 8, 8, None, 8, None, 8, None, 2, None, 0, None, 8, None, 2) == capi.SUCCESS


def test_columns_of_one_block_are_different_places():
    passed = (capi.EXECUTION_FAILED, capi.INVALID_POINTER)  # on to the check of the memory, which this is not
    lookup = lambda table, y, ldy=64, width=32: call("embedding", capi.INDEX_I64, capi.TYPE_F32, 4, 3 * A, 1, 9, width, 1.0, table, 64, y, ldy)  # noqa: E731
    assert lookup(A, A + 128) in passed and lookup(A + 128, A) in passed
    assert lookup(A, A + 128 + 256) in passed and lookup(A + 256, A + 128) in passed   # a row further down or up
    assert lookup(A, A + 124) == capi.INVALID_VALUE and lookup(A + 128, A + 4) == capi.INVALID_VALUE
    assert lookup(A, A + 132) == capi.INVALID_VALUE        # the last column is the first of the next row's
    assert lookup(A, A + 128, ldy=65) == capi.INVALID_VALUE
    assert lookup(A, A + 256) == capi.INVALID_VALUE and lookup(A, A) == capi.INVALID_VALUE


def test_workspace_sizes():
    n = C.c_size_t()
    assert call("embedding_grad_buffer_size", 10, 10, 10, None) == capi.NOT_INITIALIZED
    assert call("embedding_grad_buffer_size", -1, 10, 10, C.byref(n)) == capi.INVALID_VALUE
    sizes = [spblas.embedding_grad_buffer_size(t, v, w) for t, v, w in ((0, 1, 1), (100, 1, 1), (100, 5000, 1), (100, 5000, 4096), (1 << 31, 1, 1))]
    assert [s for s, _ in sizes] == [0, 0, 0, 0, capi.INVALID_VALUE]
    assert sizes[0][1] < sizes[1][1] < sizes[2][1] < sizes[3][1]
    assert call("expert_plan_buffer_size", 4, 2, 8, None) == capi.NOT_INITIALIZED
    assert spblas.expert_plan_buffer_size(4, 0, 8)[0] == capi.INVALID_VALUE
    assert spblas.expert_plan_buffer_size(10, 8, 64) == (capi.SUCCESS, 0)
    assert spblas.expert_plan_buffer_size(1 << 20, 8, 64)[1] > 0


def test_shapes_and_types_of_the_python_calls():
    f = np.zeros
    t, table, y = f(4, np.int64), f((9, 8), np.float32), f((4, 8), np.float32)
    assert spblas.embedding(t[None], table, 1.0, y) == capi.INVALID_VALUE
    assert spblas.embedding(t, table, 1.0, f((4, 7), np.float32)) == capi.INVALID_VALUE
    assert spblas.embedding(t, table, 1.0, f((5, 8), np.float32)) == capi.INVALID_VALUE
    assert spblas.embedding(t, table, 1.0, y.astype(np.float64)) == capi.INVALID_VALUE
    assert spblas.embedding(t, table[:, ::2], 1.0, f((4, 4), np.float32)) == capi.INVALID_VALUE     # columns apart
    assert spblas.embedding(t[::-1], table, 1.0, y) == capi.INVALID_VALUE                            # a negative stride
    assert spblas.embedding(t.astype(np.int16), table, 1.0, y) == capi.INVALID_VALUE
    i, w = f((4, 2), np.int32), f((4, 2), np.float32)
    assert spblas.route(0, y, None, 1, 1, True, 1.0, i.astype(np.int64), w) == capi.INVALID_VALUE
    assert spblas.route(0, y, None, 1, 1, True, 1.0, i, w.astype(np.float64)) == capi.INVALID_VALUE
    assert spblas.route(0, y, f(7, np.float32), 1, 1, True, 1.0, i, w) == capi.INVALID_VALUE
    assert spblas.route(0, y, None, 1, 1, True, 1.0, i[:3], w[:3]) == capi.INVALID_VALUE
    assert spblas.route_grad(0, y, i, True, 1.0, w, f((4, 7), np.float32)) == capi.INVALID_VALUE
    assert spblas.expert_plan(i, f((3, 3), np.int32), i.copy(), None) == capi.INVALID_VALUE
    assert spblas.expert_dispatch(y, i[:3], f((8, 8), np.float32)) == capi.INVALID_VALUE
    assert spblas.expert_combine(f((8, 8), np.float32), i, f((4, 3), np.float32), 0.0, y) == capi.INVALID_VALUE
    assert spblas.expert_combine_grad(y, f((8, 8), np.float32), i, w, f((8, 7), np.float32), w.copy()) == capi.INVALID_VALUE


@pytest.mark.parametrize("change,want", [({0: 2}, capi.INVALID_VALUE), ({1: 5}, capi.INVALID_VALUE), ({2: 0}, capi.INVALID_VALUE), ({2: 5000}, capi.NOT_SUPPORTED),
                                         ({3: -1}, capi.INVALID_VALUE), ({4: None}, capi.NOT_INITIALIZED), ({5: 1 << 25}, capi.INVALID_VALUE), ({7: None}, capi.NOT_INITIALIZED),
                                         ({9: None}, capi.NOT_INITIALIZED), ({12: None}, capi.NOT_INITIALIZED), ({8: 15}, capi.INVALID_VALUE), ({10: 15}, capi.INVALID_VALUE),
                                         ({11: 16 * 31}, capi.INVALID_VALUE), ({13: 31}, capi.INVALID_VALUE), ({12: A}, capi.INVALID_VALUE), ({12: 3 * A + 64}, capi.INVALID_VALUE),
                                         ({3: 0, 7: None, 12: None}, capi.SUCCESS), ({5: 0}, capi.SUCCESS)])
def test_expert_mm(change, want):
    args = [capi.TRANSPOSE, capi.TYPE_BF16, 4, 100, 2 * A, 32, 16, A, 16, 3 * A, 16, 512, 5 * A, 32]
    for at, v in change.items():
        args[at] = v
    assert call("expert_mm", *args) == want


@pytest.mark.parametrize("change,want", [({0: 5}, capi.INVALID_VALUE), ({1: capi.TYPE_F16}, capi.NOT_SUPPORTED), ({1: -1}, capi.INVALID_VALUE), ({4: None}, capi.NOT_INITIALIZED),
                                         ({7: None}, capi.NOT_INITIALIZED), ({12: None}, capi.NOT_INITIALIZED), ({13: 15}, capi.INVALID_VALUE), ({14: 100}, capi.INVALID_VALUE),
                                         ({12: A}, capi.INVALID_VALUE), ({5: 0, 12: None}, capi.SUCCESS)])
def test_expert_mm_grad(change, want):
    args = [capi.TYPE_BF16, capi.TYPE_F32, 4, 100, 2 * A, 32, 16, A, 32, 3 * A, 16, 0.0, 5 * A, 16, 512]
    for at, v in change.items():
        args[at] = v
    assert call("expert_mm_grad", *args) == want


def test_shapes_and_types_of_the_experts_products():
    f = np.zeros
    o, x, w, y = f(3, np.int32), f((6, 8), np.float16), f((2, 4, 8), np.float16), f((6, 4), np.float16)
    for args in ((capi.TRANSPOSE, o[:2], x, w, y), (capi.NON_TRANSPOSE, o, x, w, y), (capi.TRANSPOSE, o, x[:5], w, y), (capi.TRANSPOSE, o, x, w.astype(np.float32), y),
                 (capi.TRANSPOSE, o, x, w[0], y), (capi.TRANSPOSE, o, x[:, ::2], w, y)):
        assert spblas.expert_mm(*args) == capi.INVALID_VALUE
    assert spblas.expert_mm_grad(o, y, x, 0.0, f((2, 8, 4), np.float16)) == capi.INVALID_VALUE
    assert spblas.expert_mm_grad(o, y, x[:5], 0.0, w) == capi.INVALID_VALUE
    assert call("expert_mm_status", None, 0) == capi.NOT_INITIALIZED


def test_workspaces_whose_elements_are_apart():
    """What lies between them is not the call's to write."""
    f = np.zeros
    t, dy, d = f(4, np.int64), f((4, 8), np.float32), f((9, 8), np.float32)
    size = spblas.embedding_grad_buffer_size(4, 9, 8)[1]
    apart = f(2 * size + 64, np.uint8)[::2]
    assert apart.nbytes >= size and spblas.embedding_grad(t, dy, 1.0, 0.0, d, apart) == capi.INVALID_VALUE
    index, size = f((9000, 2), np.int32), spblas.expert_plan_buffer_size(9000, 2, 8)[1]
    apart = f((size, 2), np.uint8)[:, 0]
    assert apart.nbytes >= size and spblas.expert_plan(index, f(9, np.int32), index.copy(), apart) == capi.INVALID_VALUE
    whole = spblas.expert_plan(index, f(9, np.int32), index.copy(), f(size, np.uint8))
    assert whole in (capi.EXECUTION_FAILED, capi.INVALID_POINTER)  # on to the check of the memory, which is the host's
