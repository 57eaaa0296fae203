"""What HashTable.find_layer_norm checks before anything reaches a GPU: tensors that a
kernel could not read or would read past their end."""
import ctypes

import pytest
import torch

import hierarchicalkv_b200 as hkv

N, DIM = 4, 8
BUF = ctypes.c_void_p(1 << 20)   # an address that no refused call touches


def gpu_like(t):
    """A CPU tensor that says it is on GPU 0: refused calls do not touch its memory."""
    class OnGpu(torch.Tensor):
        is_cuda = True

        def get_device(self):
            return 0
    return t.as_subclass(OnGpu)


def arguments(**other):
    args = dict(keys=torch.zeros(N, dtype=torch.int64), values=torch.zeros((N, DIM)),
                founds=torch.zeros(N, dtype=torch.bool))
    return {k: gpu_like(v) for k, v in {**args, **other}.items()}


@pytest.fixture
def table(product_lib):
    t = hkv.HashTable(hkv.EvictStrategy.kLru)
    t._opts = hkv.HashTableOptions(init_capacity=128, max_capacity=128, max_hbm_for_vectors=1 << 20, dim=DIM)
    return t                          # checked, but never created: what passes the checks meets a null handle


@pytest.mark.parametrize("other,fragment", [
    (dict(keys=torch.zeros(N, dtype=torch.int32)), "keys"),
    (dict(keys=torch.zeros(N)), "keys"),
    (dict(keys=torch.zeros(N - 1, dtype=torch.int64)), "keys"),
    (dict(founds=torch.zeros(N)), "founds"),
    (dict(founds=torch.zeros(N - 1, dtype=torch.bool)), "founds"),
    (dict(values=torch.zeros((N, DIM - 1))), "values"),
    (dict(values=torch.zeros((N, DIM), dtype=torch.float16)), "values"),
    (dict(mean=torch.zeros(N - 1)), "mean"),
    (dict(weight=torch.ones(DIM + 1)), "weight"),
])
def test_tensors_that_do_not_fit_are_refused(table, other, fragment):
    with pytest.raises(ValueError, match=fragment):
        table.find_layer_norm(N, **arguments(**other))


@pytest.mark.parametrize("name", ["keys", "values", "founds", "weight", "bias", "mean", "rstd"])
def test_memory_a_kernel_cannot_reach_is_refused(table, name):
    args = arguments(weight=torch.ones(DIM), bias=torch.ones(DIM), mean=torch.ones(N), rstd=torch.ones(N))
    plain = args[name].as_subclass(torch.Tensor)
    args[name] = plain                # pageable host memory
    with pytest.raises(ValueError, match=f"{name} must be on the GPU"):
        table.find_layer_norm(N, **args)

    class Elsewhere(torch.Tensor):
        is_cuda = True

        def get_device(self):
            return 1
    args[name] = plain.as_subclass(Elsewhere)
    with pytest.raises(ValueError, match="on the GPU"):
        table.find_layer_norm(N, **args)


def test_a_table_that_is_not_there(table, product_lib):
    with pytest.raises(ValueError, match="table"):
        table.find_layer_norm(N, **arguments(), stream=1)
    rc = product_lib.hkv_find_layer_norm(None, N, BUF, None, None, 1, 1e-5, BUF, BUF, None, None, None)
    assert rc == 4 and b"table" in product_lib.hkv_last_error()
