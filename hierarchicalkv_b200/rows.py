"""Row operators of a model: what happens to the rows of a table next.

Layer norm of rows and its gradient, and the routing of token rows to experts
and back, with its gradients (hkv_layer_norm*, hkv_expert_* of the C ABI; the
reference has no such operators).  Where sharded.py sorts keys by the rank that
owns them, this module sorts tokens by the expert that takes them.

Tensors live on one GPU; a row matrix is 2-D, its rows contiguous and any
distance apart.  Rows are float32, float16 or bfloat16; weights and biases have
the rows' type or float32, and so have their gradients.  The calls run on the
current stream of the tensors' device, or on ``stream``, and do not synchronise.
``out`` arguments receive the result (they must not overlap an input); without
them it is a new tensor.  The functions are outside autograd: the gradients are
the functions whose names end in ``_backward``, to be called by the training
step, as accum_or_assign is.
"""
from __future__ import annotations

import functools
from typing import NamedTuple, Optional

import torch

from .table import _VALUE_KINDS, CudaException, load_library

_ROW_KINDS = {t: _VALUE_KINDS[t] for t in (torch.float32, torch.float16, torch.bfloat16)}


class ExpertOrder(NamedTuple):
    """Tokens sorted by expert (expert_sort).  Assignment ``t * top_k + j`` is
    token t's j-th expert."""

    offsets: torch.Tensor    # int32 [experts + 1]: expert e's rows are offsets[e] ... offsets[e + 1]
    position: torch.Tensor   # int32 [tokens, top_k]: the row of each assignment, -1 if dropped
    source: torch.Tensor     # int32 [tokens * top_k]: the assignment of each row, -1 behind the last


def _chk(lib, rc: int) -> None:
    if rc:
        msg = (lib.hkv_rows_last_error() or b"").decode()
        if rc == 2:
            raise CudaException(msg)
        raise ValueError(msg) if rc == 4 else RuntimeError(msg)


def _on_stream(fn):
    """Runs a call whose first tensor is on another device than the current one,
    or that names a stream, with that device and stream as the current ones, so
    that what it allocates belongs to them."""

    @functools.wraps(fn)
    def call(*args, stream=None, **kwargs):
        first = next((a for a in (*args, *kwargs.values()) if isinstance(a, torch.Tensor)), None)
        dev = first.device if first is not None else None
        if dev is None or dev.type != "cuda" or (stream is None and dev.index == torch.cuda.current_device()):
            return fn(*args, **kwargs)   # not on a GPU: the call itself refuses
        with torch.cuda.device(dev):
            if stream is None:
                stream = torch.cuda.current_stream(dev)
            elif isinstance(stream, int):
                stream = torch.cuda.ExternalStream(stream, dev) if stream else torch.cuda.default_stream(dev)
            with torch.cuda.stream(stream):
                return fn(*args, **kwargs)

    return call


def _current_stream(t: torch.Tensor) -> Optional[int]:
    return torch.cuda.current_stream(t.device).cuda_stream or None


def _rows(t: torch.Tensor, name: str, like: Optional[torch.Tensor] = None, shape=None, typed: bool = True) -> int:
    """Checks a row matrix; its stride in bytes."""
    if t.dim() != 2:
        raise ValueError(f"{name} must have two dimensions")
    n, dim = t.shape
    if shape is not None and (n, dim) != tuple(shape):
        raise ValueError(f"{name} must have the shape {tuple(shape)}")
    if dim < 1:
        raise ValueError(f"{name} has no columns")
    if dim > 1 and t.stride(1) != 1:
        raise ValueError(f"the rows of {name} must be contiguous")
    if like is None:
        if typed and t.dtype not in _ROW_KINDS:
            raise ValueError(f"{name} must be float32, float16 or bfloat16")
        if not t.is_cuda:
            raise ValueError(f"{name} must be on a GPU")
    elif t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"{name} must have the type and device of the other rows")
    # one row, or rows without a distance: what the stride says is of no account
    return (t.stride(0) if n > 1 else dim) * t.element_size()


def _out(out: Optional[torch.Tensor], shape, like: torch.Tensor, name: str = "out"):
    """The tensor a row matrix goes to, and its stride in bytes."""
    if out is None:
        out = torch.empty(shape, dtype=like.dtype, device=like.device)
        return out, shape[1] * out.element_size()
    stride = _rows(out, name, like, shape)
    if stride < shape[1] * out.element_size():
        raise ValueError(f"the rows of {name} overlap")
    return out, stride


def _vector(t: Optional[torch.Tensor], name: str, n: int, dtypes, device):
    if t is None:
        return None
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be " + " or ".join(str(d) for d in dict.fromkeys(dtypes)))
    if t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous and have {n} elements")
    if t.device != device:
        raise ValueError(f"{name} must be on the device of the rows")
    return t.data_ptr()


def _order(order: ExpertOrder, device):
    """(tokens, top_k, experts) of an order."""
    offsets, position = order[0], order[1]
    if position.dim() != 2 or position.dtype != torch.int32 or not position.is_contiguous():
        raise ValueError("order.position must be a contiguous int32 matrix [tokens, top_k]")
    if offsets.dim() != 1 or offsets.dtype != torch.int32 or not offsets.is_contiguous():
        raise ValueError("order.offsets must be a contiguous int32 vector [experts + 1]")
    if position.device != device or offsets.device != device:
        raise ValueError("the order must be on the device of the rows")
    return position.shape[0], position.shape[1], offsets.numel() - 1


@_on_stream
def expert_sort(expert_ids: torch.Tensor, num_experts: int) -> ExpertOrder:
    """Sorts token assignments by expert.  ``expert_ids``: int32 or int64
    [tokens, top_k]; an id outside [0, num_experts) drops its assignment.  The
    sort is stable: an expert's rows keep the order of the assignments."""
    if expert_ids.dim() != 2 or expert_ids.dtype not in (torch.int32, torch.int64):
        raise ValueError("expert_ids must be an int32 or int64 matrix [tokens, top_k]")
    if not expert_ids.is_contiguous():
        raise ValueError("expert_ids must be contiguous")
    if not 1 <= num_experts <= 1024:
        raise ValueError("num_experts must be between 1 and 1024")
    tokens, top_k = expert_ids.shape
    if not 1 <= top_k <= 64:
        raise ValueError("top_k must be between 1 and 64")
    if not expert_ids.is_cuda:
        raise ValueError("expert_ids must be on a GPU")
    lib = load_library()
    dev = expert_ids.device
    offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=dev)
    position = torch.empty((tokens, top_k), dtype=torch.int32, device=dev)
    source = torch.empty(tokens * top_k, dtype=torch.int32, device=dev)
    work_bytes = lib.hkv_expert_sort_workspace_bytes(tokens, top_k, num_experts)
    work = torch.empty(work_bytes, dtype=torch.uint8, device=dev) if work_bytes else None
    _chk(lib, lib.hkv_expert_sort(
        tokens, top_k, expert_ids.data_ptr(), expert_ids.element_size(), num_experts,
        offsets.data_ptr(), position.data_ptr(), source.data_ptr(),
        work.data_ptr() if work is not None else None, work_bytes, _current_stream(expert_ids)))
    return ExpertOrder(offsets, position, source)


@_on_stream
def expert_dispatch(x: torch.Tensor, order: ExpertOrder, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Copies of the token rows in the order of the experts: [tokens * top_k, dim]
    with row ``order.position[t, j]`` = x[t].  Rows behind the last expert's are
    zeros in a new tensor and left as they are in ``out``.  Any element type."""
    x_stride = _rows(x, "x", typed=False)
    tokens, top_k, experts = _order(order, x.device)
    if x.shape[0] != tokens:
        raise ValueError("x must have a row for every token of the order")
    new = out is None
    out, out_stride = _out(out, (tokens * top_k, x.shape[1]), x)
    lib = load_library()
    _chk(lib, lib.hkv_expert_dispatch(
        tokens, top_k, x.shape[1] * x.element_size(), x.data_ptr(), x_stride, experts,
        order[0].data_ptr(), order[1].data_ptr(), out.data_ptr(), out_stride, int(new),
        _current_stream(x)))
    return out


def _combine(rows, weights, order, out):
    stride = _rows(rows, "rows")
    tokens, top_k, _ = _order(order, rows.device)
    if rows.shape[0] != tokens * top_k:
        raise ValueError("rows must have a row for every assignment of the order")
    kind = _ROW_KINDS[rows.dtype]
    w = _vector(weights, "weights", tokens * top_k, (rows.dtype, torch.float32), rows.device)
    out, out_stride = _out(out, (tokens, rows.shape[1]), rows)
    lib = load_library()
    _chk(lib, lib.hkv_expert_combine(
        tokens, top_k, rows.shape[1], kind, rows.data_ptr(), stride, w,
        kind if weights is None else _ROW_KINDS[weights.dtype], order[1].data_ptr(), out.data_ptr(),
        out_stride, _current_stream(rows)))
    return out


@_on_stream
def expert_dispatch_backward(d_rows: torch.Tensor, order: ExpertOrder,
                             out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of expert_dispatch: every token sums the gradients of its copies
    [tokens, dim].  Rows behind the last expert's are not read."""
    return _combine(d_rows, None, order, out)


@_on_stream
def expert_combine(rows: torch.Tensor, weights: torch.Tensor, order: ExpertOrder,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The experts' rows back in token order: out[t] is the sum over j of
    weights[t, j] * rows[order.position[t, j]].  Dropped assignments add nothing,
    whatever their weight; a token without any gets zeros."""
    return _combine(rows, weights, order, out)


@_on_stream
def expert_combine_backward(d_out: torch.Tensor, rows: torch.Tensor, weights: torch.Tensor,
                            order: ExpertOrder, out: Optional[torch.Tensor] = None):
    """Gradients of expert_combine: (d_rows, d_weights).  The rows of d_rows
    behind the last expert's are zeros in a new tensor and left as they are in
    ``out``; the weights of dropped assignments get 0."""
    d_stride = _rows(d_out, "d_out")
    tokens, top_k, experts = _order(order, d_out.device)
    if d_out.shape[0] != tokens:
        raise ValueError("d_out must have a row for every token of the order")
    dim = d_out.shape[1]
    stride = _rows(rows, "rows", d_out, (tokens * top_k, dim))
    w = _vector(weights, "weights", tokens * top_k, (rows.dtype, torch.float32), d_out.device)
    new = out is None
    out, out_stride = _out(out, (tokens * top_k, dim), d_out)
    d_weights = torch.empty((tokens, top_k), dtype=weights.dtype, device=d_out.device)
    lib = load_library()
    _chk(lib, lib.hkv_expert_combine_backward(
        tokens, top_k, dim, _ROW_KINDS[rows.dtype], d_out.data_ptr(), d_stride, rows.data_ptr(),
        stride, w, _ROW_KINDS[weights.dtype], experts, order[0].data_ptr(), order[1].data_ptr(),
        out.data_ptr(), out_stride, int(new), d_weights.data_ptr(), _current_stream(d_out)))
    return out, d_weights


def _params(weight, bias, dim, dtype, device):
    """Addresses of weight and bias and their kind."""
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError("weight and bias must have one type")
    w = _vector(weight, "weight", dim, (dtype, torch.float32), device)
    b = _vector(bias, "bias", dim, (dtype, torch.float32), device)
    given = weight if weight is not None else bias
    return w, b, _ROW_KINDS[dtype if given is None else given.dtype]


@_on_stream
def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, eps: float = 1e-5, stats: bool = True,
               out: Optional[torch.Tensor] = None):
    """Layer norm of every row of x [n, dim].  Returns (y, mean, rstd), the
    statistics (float32 [n]) being what layer_norm_backward needs, or y alone
    with ``stats=False``."""
    stride = _rows(x, "x")
    n, dim = x.shape
    w, b, kind = _params(weight, bias, dim, x.dtype, x.device)
    y, y_stride = _out(out, (n, dim), x)
    mean = rstd = None
    if stats:
        mean = torch.empty(n, dtype=torch.float32, device=x.device)
        rstd = torch.empty(n, dtype=torch.float32, device=x.device)
    lib = load_library()
    _chk(lib, lib.hkv_layer_norm(
        n, dim, _ROW_KINDS[x.dtype], x.data_ptr(), stride, w, b, kind, eps, y.data_ptr(), y_stride,
        mean.data_ptr() if stats else None, rstd.data_ptr() if stats else None, _current_stream(x)))
    return (y, mean, rstd) if stats else y


@_on_stream
def layer_norm_ptr(n: int, row_ptrs: torch.Tensor, out: torch.Tensor,
                   weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                   eps: float = 1e-5, mean: Optional[torch.Tensor] = None,
                   rstd: Optional[torch.Tensor] = None) -> torch.Tensor:
    """layer_norm of n rows by address: ``row_ptrs`` (int64) as HashTable.find_ptr
    fills them, rows of the type and length of ``out``'s.  The rows are read where
    the table keeps them and must not change meanwhile (HashTable.find_layer_norm
    holds the table's lock over both steps).  Null addresses leave their row of
    ``out`` (and of ``mean`` and ``rstd``, float32, optional) as it is."""
    stride = _rows(out, "out")
    dim = out.shape[1]
    if not 0 <= n <= out.shape[0]:
        raise ValueError("out must have n rows")
    if stride < dim * out.element_size():
        raise ValueError("the rows of out overlap")
    if row_ptrs.dtype != torch.int64 or not row_ptrs.is_contiguous() or row_ptrs.numel() < n:
        raise ValueError("row_ptrs must be contiguous and hold n int64 addresses")
    if row_ptrs.device != out.device:
        raise ValueError("row_ptrs must be on the device of out")
    w, b, kind = _params(weight, bias, dim, out.dtype, out.device)
    for name, s in (("mean", mean), ("rstd", rstd)):
        if s is not None and (s.dtype != torch.float32 or s.numel() < n or not s.is_contiguous()
                              or s.device != out.device):
            raise ValueError(f"{name} must be contiguous, on the device of out and hold n float32 elements")
    lib = load_library()
    _chk(lib, lib.hkv_layer_norm_ptr(
        n, dim, _ROW_KINDS[out.dtype], row_ptrs.data_ptr(), w, b, kind, eps, out.data_ptr(), stride,
        mean.data_ptr() if mean is not None else None, rstd.data_ptr() if rstd is not None else None,
        _current_stream(out)))
    return out


@_on_stream
def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor],
                        mean: torch.Tensor, rstd: torch.Tensor, bias: bool = True,
                        out: Optional[torch.Tensor] = None):
    """Gradients of layer_norm: (dx, d_weight, d_bias).  d_weight is None where
    the layer has no ``weight``, d_bias where ``bias`` is false; both have the
    type of ``weight`` (of the rows where there is none)."""
    stride = _rows(x, "x")
    n, dim = x.shape
    dy_stride = _rows(dy, "dy", x, (n, dim))
    w, _, kind = _params(weight, None, dim, x.dtype, x.device)
    m = _vector(mean, "mean", n, (torch.float32,), x.device)
    r = _vector(rstd, "rstd", n, (torch.float32,), x.device)
    dx, dx_stride = _out(out, (n, dim), x)
    lib = load_library()
    ptype = x.dtype if weight is None else weight.dtype
    d_weight = torch.empty(dim, dtype=ptype, device=x.device) if weight is not None else None
    d_bias = torch.empty(dim, dtype=ptype, device=x.device) if bias else None
    work, work_bytes = None, 0
    if d_weight is not None or bias:
        work_bytes = lib.hkv_layer_norm_backward_workspace_bytes(n, dim, _ROW_KINDS[x.dtype])
        work = torch.empty(work_bytes, dtype=torch.uint8, device=x.device)
    _chk(lib, lib.hkv_layer_norm_backward(
        n, dim, _ROW_KINDS[x.dtype], dy.data_ptr(), dy_stride, x.data_ptr(), stride, w, kind, m, r,
        dx.data_ptr(), dx_stride, d_weight.data_ptr() if d_weight is not None else None,
        d_bias.data_ptr() if bias else None, work.data_ptr() if work is not None else None,
        work_bytes, _current_stream(x)))
    return dx, d_weight, d_bias
