"""The C entries of the row operators refuse buffers that do not start at a multiple of
their element size: a kernel would fault on them."""
import ctypes

import pytest

F32, F16 = 1, 5
NULL = None
BUF = ctypes.c_void_p(1 << 20)   # addresses that no refused call touches
ODD, HALF, WORD = (ctypes.c_void_p((1 << 20) + k) for k in (1, 2, 4))


def sort(ids=BUF, id_bytes=8, offsets=BUF, position=BUF, source=BUF, tokens=4, work=NULL, work_bytes=0):
    return "hkv_expert_sort", (tokens, 2, ids, id_bytes, 4, offsets, position, source, work, work_bytes, NULL)


def dispatch(offsets=BUF, position=BUF):
    return "hkv_expert_dispatch", (4, 2, 16, BUF, 16, 3, offsets, position, BUF, 16, 0, NULL)


def combine(weights=BUF, kind=F32, position=BUF):
    return "hkv_expert_combine", (4, 2, 8, kind, BUF, 32, weights, kind, position, BUF, 32, NULL)


def combine_backward(weights=BUF, kind=F32, offsets=BUF, position=BUF, d_weights=BUF):
    return "hkv_expert_combine_backward", (4, 2, 8, F16, BUF, 32, BUF, 32, weights, kind, 3, offsets, position, BUF, 32,
                                           0, d_weights, NULL)


def norm(weight=BUF, bias=BUF, kind=F32, mean=BUF, rstd=BUF):
    return "hkv_layer_norm", (4, 8, F16, BUF, 16, weight, bias, kind, 1e-5, BUF, 16, mean, rstd, NULL)


def norm_ptr(ptrs=BUF, weight=BUF, bias=BUF, mean=BUF, rstd=BUF):
    return "hkv_layer_norm_ptr", (4, 8, F16, ptrs, weight, bias, F32, 1e-5, BUF, 16, mean, rstd, NULL)


def norm_backward(weight=BUF, kind=F32, mean=BUF, rstd=BUF, d_weight=BUF, d_bias=BUF, work=BUF):
    return "hkv_layer_norm_backward", (4, 8, F16, BUF, 16, BUF, 16, weight, kind, mean, rstd, BUF, 16, d_weight, d_bias,
                                       work, 1 << 20, NULL)


CALLS = [sort(ids=WORD), sort(ids=HALF, id_bytes=4), sort(offsets=HALF), sort(position=ODD), sort(source=HALF),
         sort(tokens=1 << 20, work=HALF, work_bytes=1 << 30),
         dispatch(offsets=HALF), dispatch(position=HALF),
         combine(weights=HALF), combine(weights=ODD, kind=F16), combine(position=HALF),
         combine_backward(weights=HALF), combine_backward(weights=ODD, kind=F16), combine_backward(offsets=HALF),
         combine_backward(position=ODD), combine_backward(d_weights=HALF),
         norm(weight=HALF), norm(bias=HALF), norm(weight=ODD, kind=F16), norm(mean=HALF), norm(rstd=ODD),
         norm_ptr(ptrs=WORD), norm_ptr(weight=HALF), norm_ptr(bias=ODD), norm_ptr(mean=HALF), norm_ptr(rstd=HALF),
         norm_backward(weight=HALF), norm_backward(weight=ODD, kind=F16), norm_backward(mean=HALF),
         norm_backward(rstd=HALF), norm_backward(d_weight=HALF), norm_backward(d_bias=ODD), norm_backward(work=HALF)]


@pytest.mark.parametrize("name,args", CALLS, ids=[f"{i}-{c[0][4:]}" for i, c in enumerate(CALLS)])
def test_misaligned_buffers_are_refused(product_lib, name, args):
    rc = getattr(product_lib, name)(*args)
    assert rc == 4 and b"element size" in product_lib.hkv_rows_last_error()
