"""The row operators at the edges of what their documents allow: stream captures,
rows far from zero, batches and offsets past the sizes of the other tests."""
import os
import sys

import numpy as np
import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)

import hierarchicalkv_b200 as hkv  # noqa: E402
from tests.hkv_testlib import to_dev, unique_keys  # noqa: E402

pytestmark = pytest.mark.gpu


def make_table(dim, dtype=torch.float32, capacity=128 * 64, **options):
    t = hkv.HashTable(hkv.EvictStrategy.kLru, value_dtype=dtype)
    t.init(hkv.HashTableOptions(init_capacity=capacity, max_capacity=capacity, max_hbm_for_vectors=1 << 30, dim=dim,
                                **options))
    return t


# ---- find with layer norm ----------------------------------------------------------


@pytest.mark.parametrize("warm", [False, True], ids=["first", "later"])
def test_find_layer_norm_is_refused_inside_a_capture(warm):
    """Its scratch belongs to the table: a graph would keep the address of memory
    that a larger call gives back.  The refusal leaves the capture, the outputs and
    the table as they were."""
    dim, n = 16, 1000
    t = make_table(dim)
    keys, rows = to_dev(unique_keys(n, seed=2)), torch.randn((n, dim), device="cuda")
    t.insert_or_assign(n, keys, rows)
    out, found = torch.full((n, dim), 5.0, device="cuda"), torch.zeros(n, dtype=torch.bool, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    if warm:
        t.find_layer_norm(n, keys, torch.zeros_like(out), torch.zeros_like(found), stream=side)
    hkv.layer_norm(rows, stream=side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        with pytest.raises(hkv.MerlinException, match="stream capture"):
            t.find_layer_norm(n, keys, out, found)
        y = hkv.layer_norm(rows, stats=False)
    g.replay()
    torch.cuda.synchronize()
    want = hkv.layer_norm(rows, stats=False)
    assert torch.equal(y, want) and (out == 5).all() and not found.any()
    t.find_layer_norm(n, keys, out, found)
    assert found.all() and torch.equal(out, want)
    t.close()
