"""Refusals of the row operators (layer norm, expert sort / dispatch / combine):
what they check before anything reaches a GPU, in the Python functions and at
the C entries."""
import ctypes
import re

import pytest
import torch

import hierarchicalkv_b200 as hkv

F32, F16, BF16 = 1, 5, 6
NULL = None
BUF = ctypes.c_void_p(1 << 20)   # an address that no refused call touches


def order(tokens=4, top_k=2, experts=3, **kw):
    return hkv.ExpertOrder(
        kw.get("offsets", torch.zeros(experts + 1, dtype=torch.int32)),
        kw.get("position", torch.zeros((tokens, top_k), dtype=torch.int32)),
        kw.get("source", torch.zeros(tokens * top_k, dtype=torch.int32)))


@pytest.mark.parametrize("ids,experts,fragment", [
    (torch.zeros(8, dtype=torch.int64), 4, "matrix"),
    (torch.zeros((4, 2)), 4, "int32 or int64"),
    (torch.zeros((4, 2), dtype=torch.int16), 4, "int32 or int64"),
    (torch.zeros((2, 4), dtype=torch.int64).t(), 4, "contiguous"),
    (torch.zeros((4, 2), dtype=torch.int64), 0, "num_experts"),
    (torch.zeros((4, 2), dtype=torch.int64), 1025, "num_experts"),
    (torch.zeros((4, 0), dtype=torch.int64), 4, "top_k"),
    (torch.zeros((4, 65), dtype=torch.int64), 4, "top_k"),
    (torch.zeros((4, 2), dtype=torch.int64), 4, "on a GPU"),
])
def test_expert_sort_refuses(product_lib, ids, experts, fragment):
    with pytest.raises(ValueError, match=fragment):
        hkv.expert_sort(ids, experts)


@pytest.mark.parametrize("x,fragment", [
    (torch.zeros(8), "two dimensions"),
    (torch.zeros((4, 0)), "no columns"),
    (torch.zeros((8, 4)).t(), "contiguous"),
    (torch.zeros((4, 8), dtype=torch.float64), "float32, float16 or bfloat16"),
    (torch.zeros((4, 8)), "on a GPU"),
])
def test_row_matrices_are_checked(product_lib, x, fragment):
    w, m = torch.ones(8), torch.ones(4)
    with pytest.raises(ValueError, match=fragment):
        hkv.layer_norm(x, w)
    with pytest.raises(ValueError, match=fragment):
        hkv.layer_norm_backward(x, x, w, m, m)
    with pytest.raises(ValueError, match=fragment):
        hkv.expert_combine(x, torch.ones((2, 2)), order(2))
    with pytest.raises(ValueError, match=fragment):
        hkv.expert_dispatch_backward(x, order(2))
    if x.dtype != torch.float64:    # dispatch moves rows of any type
        with pytest.raises(ValueError, match=fragment):
            hkv.expert_dispatch(x, order())


def test_calls_by_keyword_are_checked_too(product_lib):
    with pytest.raises(ValueError, match="on a GPU"):
        hkv.layer_norm(x=torch.zeros((4, 8)))
    with pytest.raises(ValueError, match="on a GPU"):
        hkv.layer_norm(torch.zeros((4, 8)), stream=0)


def lib_call(lib, name, *args):
    rc = getattr(lib, name)(*args)
    return rc, (lib.hkv_rows_last_error() or b"").decode()


@pytest.mark.parametrize("args,fragment", [
    ((4, 0, BUF, 8, 4, BUF, BUF, BUF, NULL, 0, NULL), "top_k"),
    ((4, 65, BUF, 8, 4, BUF, BUF, BUF, NULL, 0, NULL), "top_k"),
    ((4, 2, BUF, 2, 4, BUF, BUF, BUF, NULL, 0, NULL), "int32 or int64"),
    ((4, 2, BUF, 8, 0, BUF, BUF, BUF, NULL, 0, NULL), "experts"),
    ((4, 2, BUF, 8, 1025, BUF, BUF, BUF, NULL, 0, NULL), "experts"),
    ((1 << 30, 2, BUF, 8, 4, BUF, BUF, BUF, NULL, 0, NULL), "2\\^31"),
    ((4, 2, NULL, 8, 4, BUF, BUF, BUF, NULL, 0, NULL), "null"),
    ((4, 2, BUF, 8, 4, NULL, BUF, BUF, NULL, 0, NULL), "null"),
    ((4, 2, BUF, 8, 4, BUF, NULL, BUF, NULL, 0, NULL), "null"),
    ((1 << 20, 2, BUF, 8, 4, BUF, BUF, BUF, NULL, 0, NULL), "workspace"),
    ((1 << 20, 2, BUF, 8, 4, BUF, BUF, BUF, NULL, 1 << 30, NULL), "workspace"),
])
def test_sort_entry_refuses(product_lib, args, fragment):
    rc, msg = lib_call(product_lib, "hkv_expert_sort", *args)
    assert rc == 4 and re.search(fragment, msg), (rc, msg)


@pytest.mark.parametrize("name,args,fragment", [
    ("hkv_expert_dispatch", (4, 2, 0, BUF, 16, 3, BUF, BUF, BUF, 16, 0, NULL), "row_bytes"),
    ("hkv_expert_dispatch", (4, 2, 16, BUF, 16, 3, BUF, BUF, BUF, 8, 0, NULL), "overlap"),
    ("hkv_expert_dispatch", (4, 2, 16, NULL, 16, 3, BUF, BUF, BUF, 16, 0, NULL), "null"),
    ("hkv_expert_dispatch", (4, 2, 16, BUF, 16, 0, BUF, BUF, BUF, 16, 0, NULL), "experts"),
    ("hkv_expert_combine", (4, 2, 8, 2, BUF, 32, BUF, 1, BUF, BUF, 32, NULL), "float32, float16"),
    ("hkv_expert_combine", (4, 2, 8, F16, BUF, 16, BUF, BF16, BUF, BUF, 16, NULL), "weights"),
    ("hkv_expert_combine", (4, 2, 0, F32, BUF, 32, BUF, F32, BUF, BUF, 32, NULL), "dim"),
    ("hkv_expert_combine", (4, 2, 8, F32, BUF, 32, BUF, F32, BUF, BUF, 16, NULL), "overlap"),
    ("hkv_expert_combine", (4, 2, 8, F32, BUF, 34, BUF, F32, BUF, BUF, 32, NULL), "element size"),
    ("hkv_expert_combine", (4, 2, 8, F32, BUF, 32, BUF, F32, NULL, BUF, 32, NULL), "null"),
    ("hkv_expert_combine_backward", (4, 2, 8, F32, BUF, 32, BUF, 32, NULL, F32, 3, BUF, BUF, BUF, 32, 0,
                                     BUF, NULL), "null"),
    ("hkv_expert_combine_backward", (4, 2, 8, F32, BUF, 32, BUF, 32, BUF, F16, 3, BUF, BUF, BUF, 32, 0,
                                     BUF, NULL), "weights"),
    ("hkv_expert_combine_backward", (4, 2, 8, F32, BUF, 33, BUF, 32, BUF, F32, 3, BUF, BUF, BUF, 32, 0,
                                     BUF, NULL), "element size"),
    ("hkv_layer_norm", (4, 8, 7, BUF, 32, BUF, BUF, 7, 1e-5, BUF, 32, BUF, BUF, NULL), "float32, float16"),
    ("hkv_layer_norm", (4, 8, F16, BUF, 16, BUF, BUF, BF16, 1e-5, BUF, 16, BUF, BUF, NULL), "weight and bias"),
    ("hkv_layer_norm", (4, 0, F32, BUF, 32, BUF, BUF, F32, 1e-5, BUF, 32, BUF, BUF, NULL), "dim"),
    ("hkv_layer_norm", (4, 1 << 24, F32, BUF, 32, BUF, BUF, F32, 1e-5, BUF, 32, BUF, BUF, NULL), "dim"),
    ("hkv_layer_norm", (1 << 31, 8, F32, BUF, 32, BUF, BUF, F32, 1e-5, BUF, 32, BUF, BUF, NULL), "2\\^31"),
    ("hkv_layer_norm", (4, 8, F32, BUF, 32, BUF, BUF, F32, -1.0, BUF, 32, BUF, BUF, NULL), "eps"),
    ("hkv_layer_norm", (4, 8, F32, BUF, 32, BUF, BUF, F32, float("nan"), BUF, 32, BUF, BUF, NULL), "eps"),
    ("hkv_layer_norm", (4, 8, F32, BUF, 32, BUF, BUF, F32, float("inf"), BUF, 32, BUF, BUF, NULL), "eps"),
    ("hkv_layer_norm", (4, 8, F32, NULL, 32, BUF, BUF, F32, 1e-5, BUF, 32, BUF, BUF, NULL), "null"),
    ("hkv_layer_norm", (4, 8, F32, BUF, 32, BUF, BUF, F32, 1e-5, BUF, 31, BUF, BUF, NULL), "overlap"),
    ("hkv_layer_norm", (4, 8, F32, BUF, 33, BUF, BUF, F32, 1e-5, BUF, 32, BUF, BUF, NULL), "element size"),
    ("hkv_layer_norm_ptr", (4, 8, F32, NULL, BUF, BUF, F32, 1e-5, BUF, 32, BUF, BUF, NULL), "null"),
    ("hkv_layer_norm_backward", (4, 8, F32, NULL, 32, BUF, 32, BUF, F32, BUF, BUF, BUF, 32, BUF, BUF, BUF,
                                 1 << 20, NULL), "null"),
    ("hkv_layer_norm_backward", (4, 8, F32, BUF, 32, BUF, 32, BUF, F32, BUF, BUF, BUF, 32, BUF, BUF, BUF,
                                 8, NULL), "workspace"),
    ("hkv_layer_norm_backward", (4, 8, F32, BUF, 32, BUF, 32, BUF, F32, BUF, BUF, BUF, 32, NULL, BUF, NULL,
                                 1 << 20, NULL), "workspace"),
    ("hkv_layer_norm_backward", (4, 8, F32, BUF, 32, BUF, 32, BUF, F32, BUF, BUF, BUF, 16, BUF, BUF, BUF,
                                 1 << 20, NULL), "overlap"),
])
def test_entries_refuse(product_lib, name, args, fragment):
    rc, msg = lib_call(product_lib, name, *args)
    assert rc == 4 and re.search(fragment, msg), (rc, msg)


def test_entries_without_rows_do_nothing(product_lib):
    """No launch and no access: null buffers are fine where there are no rows."""
    assert product_lib.hkv_expert_dispatch(0, 2, 16, NULL, 16, 3, NULL, NULL, NULL, 16, 1, NULL) == 0
    assert product_lib.hkv_expert_combine(0, 2, 8, F32, NULL, 32, NULL, F32, NULL, NULL, 32, NULL) == 0
    assert product_lib.hkv_layer_norm(0, 8, F32, NULL, 32, NULL, NULL, F32, 1e-5, NULL, 32, NULL, NULL, NULL) == 0
    assert product_lib.hkv_layer_norm_ptr(0, 8, F32, NULL, NULL, NULL, F32, 1e-5, NULL, 32, NULL, NULL, NULL) == 0


def test_workspace_sizes(product_lib):
    assert product_lib.hkv_expert_sort_workspace_bytes(0, 2, 4) == 0
    assert product_lib.hkv_expert_sort_workspace_bytes(8, 8, 64) == 0
    assert product_lib.hkv_expert_sort_workspace_bytes(1 << 22, 2, 8) >= 4 * 8
    assert product_lib.hkv_expert_sort_workspace_bytes(1 << 22, 0, 8) == 0      # refused sizes need none
    assert product_lib.hkv_layer_norm_backward_workspace_bytes(0, 8, F32) == 0
    assert product_lib.hkv_layer_norm_backward_workspace_bytes(1, 8, F32) >= 2 * 8 * 4
