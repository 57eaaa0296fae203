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
them it is a new tensor.  Inputs that were made on another stream than the one of
the call must be complete there, and stay allocated until it has run.

The functions are outside autograd: a tensor that requires gradients is taken for
its values, and the results carry no graph, whether gradients are enabled or not.
The gradients are the functions whose names end in ``_backward``, to be called by
the training step, as accum_or_assign is.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .table import _VALUE_KINDS, CudaException, load_library

_ROW_KINDS = {t: _VALUE_KINDS[t] for t in (torch.float32, torch.float16, torch.bfloat16)}
_F32 = torch.float32

# The host's part of a call is most of its time on a decoding step's few rows,
# so it asks torch for as little as it can: the raw handle of the current stream
# costs 0.1 us where the stream object costs 2.3 us, empty_like 1.4 us where
# empty with a shape, type and device costs 2.4 us.
_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
_raw_stream = torch._C._cuda_getCurrentRawStream


class ExpertOrder(NamedTuple):
    """Tokens sorted by expert (expert_sort).  Assignment ``t * top_k + j`` is
    token t's j-th expert."""

    offsets: torch.Tensor    # int32 [experts + 1]: expert e's rows are offsets[e] ... offsets[e + 1]
    position: torch.Tensor   # int32 [tokens, top_k]: the row of each assignment, -1 if dropped
    source: torch.Tensor     # int32 [tokens * top_k]: the assignment of each row, -1 behind the last


def _fail(lib, rc: int) -> None:
    msg = (lib.hkv_rows_last_error() or b"").decode()
    if rc == 2:
        raise CudaException(msg)
    raise ValueError(msg) if rc == 4 else RuntimeError(msg)


def _elsewhere(t: torch.Tensor, stream) -> bool:
    """Whether a call has to change the device or the stream first."""
    return t.is_cuda and (stream is not None or t.get_device() != _current_device())


def _run_there(fn, t: torch.Tensor, stream, *args):
    """Runs fn with the device of t and ``stream`` as the current ones, so that
    what it allocates belongs to them."""
    with torch.cuda.device(t.device):
        if stream is None:
            return fn(*args)
        if isinstance(stream, int):
            stream = torch.cuda.ExternalStream(stream, t.device) if stream else torch.cuda.default_stream(t.device)
        elif stream.device != t.device:
            raise ValueError(f"stream must be one of {t.device}, where the tensors are")
        with torch.cuda.stream(stream):
            return fn(*args)


def _rows(t: torch.Tensor, name: str):
    """Checks a row matrix: (rows, columns, distance of the rows in bytes)."""
    if t.dim() != 2:
        raise ValueError(f"{name} must have two dimensions")
    n, dim = t.shape
    if dim < 1:
        raise ValueError(f"{name} has no columns")
    stride, step = t.stride()
    if step != 1 and dim > 1:
        raise ValueError(f"the rows of {name} must be contiguous")
    if dim == 1 and t.is_neg():    # such views are two elements apart: longer rows are refused above
        raise ValueError(f"{name} is a negative view: resolve_neg it first")
    # of a single row, what the stride says is of no account
    return n, dim, (stride if n > 1 else dim) * t.element_size()


def _float_rows(t: torch.Tensor, name: str):
    """_rows of float rows on a GPU, and their kind."""
    checked = _rows(t, name)
    kind = _ROW_KINDS.get(t.dtype)
    if kind is None:
        raise ValueError(f"{name} must be float32, float16 or bfloat16")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a GPU")
    return *checked, kind


def _more_rows(t: torch.Tensor, name: str, n: int, dim: int, like: torch.Tensor) -> int:
    """Checks another row matrix of a call; its stride in bytes."""
    rows, columns, stride = _rows(t, name)
    if rows != n or columns != dim:
        raise ValueError(f"{name} must have the shape {(n, dim)}")
    if t.dtype is not like.dtype or t.get_device() != like.get_device():
        raise ValueError(f"{name} must have the type and device of the other rows")
    return stride


def _out(out: Optional[torch.Tensor], n: int, dim: int, like: torch.Tensor):
    """The matrix a result goes to, and its stride in bytes."""
    if out is None:
        same = like.shape[0] == n and like.is_contiguous()
        out = torch.empty_like(like) if same else like.new_empty((n, dim))
        return out, dim * out.element_size()
    stride = _more_rows(out, "out", n, dim, like)
    if stride < dim * out.element_size():
        raise ValueError("the rows of out overlap")
    if out.is_conj():
        raise ValueError("out is a conjugate view: resolve_conj it first")
    return out, stride


def _vector(t: Optional[torch.Tensor], name: str, n: int, like: torch.Tensor):
    """Address of n parameters in the type of the rows `like` or float32."""
    if t is None:
        return None
    if t.dtype is not _F32 and t.dtype is not like.dtype:
        raise ValueError(f"{name} must be float32 or have the type of the rows")
    if t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous and have {n} elements")
    if t.get_device() != like.get_device():
        raise ValueError(f"{name} must be on the device of the rows")
    return t.data_ptr()


def _statistic(t: Optional[torch.Tensor], name: str, n: int, like: torch.Tensor):
    """Address of the float32 statistics of n rows."""
    if t is None:
        return None
    if t.dtype is not _F32 or t.numel() < n or not t.is_contiguous() or t.get_device() != like.get_device():
        raise ValueError(f"{name} must be contiguous, on the device of the rows and hold {n} float32 elements")
    return t.data_ptr()


def _weights(t: Optional[torch.Tensor], order: ExpertOrder, like: torch.Tensor):
    """Address of the weights of an order's assignments."""
    if t is not None and t.shape != order[1].shape:
        raise ValueError("weights must have the shape of order.position, [tokens, top_k]")
    return _vector(t, "weights", order[1].numel(), like)


def _order(order: ExpertOrder, like: torch.Tensor):
    """(tokens, top_k, experts, addresses of offsets and position) of an order."""
    offsets, position = order[0], order[1]
    if position.dim() != 2 or position.dtype is not torch.int32 or not position.is_contiguous():
        raise ValueError("order.position must be a contiguous int32 matrix [tokens, top_k]")
    if offsets.dim() != 1 or offsets.dtype is not torch.int32 or not offsets.is_contiguous():
        raise ValueError("order.offsets must be a contiguous int32 vector [experts + 1]")
    dev = like.get_device()
    if position.get_device() != dev or offsets.get_device() != dev:
        raise ValueError("the order must be on the device of the rows")
    tokens, top_k = position.shape
    return tokens, top_k, offsets.shape[0] - 1, offsets.data_ptr(), position.data_ptr()


def expert_sort(expert_ids: torch.Tensor, num_experts: int, stream=None) -> ExpertOrder:
    """Sorts token assignments by expert.  ``expert_ids``: int32 or int64
    [tokens, top_k]; an id outside [0, num_experts) drops its assignment.  The
    sort is stable: an expert's rows keep the order of the assignments."""
    if _elsewhere(expert_ids, stream):
        return _run_there(expert_sort, expert_ids, stream, expert_ids, num_experts)
    if expert_ids.dim() != 2 or expert_ids.dtype not in (torch.int64, torch.int32):
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
    n = tokens * top_k
    position = torch.empty_like(expert_ids, dtype=torch.int32)
    source = expert_ids.new_empty(n, dtype=torch.int32)
    offsets = expert_ids.new_empty(num_experts + 1, dtype=torch.int32)
    work_bytes = lib.hkv_expert_sort_workspace_bytes(tokens, top_k, num_experts)
    work = expert_ids.new_empty(work_bytes, dtype=torch.uint8) if work_bytes else None
    rc = lib.hkv_expert_sort(
        tokens, top_k, expert_ids.data_ptr(), expert_ids.element_size(), num_experts,
        offsets.data_ptr(), position.data_ptr(), source.data_ptr(),
        work.data_ptr() if work_bytes else None, work_bytes, _raw_stream(expert_ids.get_device()))
    if rc:
        _fail(lib, rc)
    return ExpertOrder(offsets, position, source)


def expert_dispatch(x: torch.Tensor, order: ExpertOrder, out: Optional[torch.Tensor] = None,
                    stream=None) -> torch.Tensor:
    """Copies of the token rows in the order of the experts: [tokens * top_k, dim]
    with row ``order.position[t, j]`` = x[t].  Rows behind the last expert's are
    zeros in a new tensor and left as they are in ``out``.  Any element type.
    Records no graph: the gradient is expert_dispatch_backward."""
    if _elsewhere(x, stream):
        return _run_there(expert_dispatch, x, stream, x, order, out)
    n, dim, x_stride = _rows(x, "x")
    if x.is_conj():
        raise ValueError("x is a conjugate view: resolve_conj it first")
    if not x.is_cuda:
        raise ValueError("x must be on a GPU")
    tokens, top_k, experts, offsets, position = _order(order, x)
    if n != tokens:
        raise ValueError("x must have a row for every token of the order")
    new = out is None
    out, out_stride = _out(out, tokens * top_k, dim, x)
    lib = load_library()
    rc = lib.hkv_expert_dispatch(
        tokens, top_k, dim * x.element_size(), x.data_ptr(), x_stride, experts, offsets, position,
        out.data_ptr(), out_stride, new, _raw_stream(x.get_device()))
    if rc:
        _fail(lib, rc)
    return out


def _combine(rows, weights, order, out):
    n, dim, stride, kind = _float_rows(rows, "rows")
    tokens, top_k, _, _, position = _order(order, rows)
    if n != tokens * top_k:
        raise ValueError("rows must have a row for every assignment of the order")
    w = _weights(weights, order, rows)
    out, out_stride = _out(out, tokens, dim, rows)
    lib = load_library()
    rc = lib.hkv_expert_combine(
        tokens, top_k, dim, kind, rows.data_ptr(), stride, w,
        kind if weights is None else _ROW_KINDS[weights.dtype], position, out.data_ptr(), out_stride,
        _raw_stream(rows.get_device()))
    if rc:
        _fail(lib, rc)
    return out


def expert_dispatch_backward(d_rows: torch.Tensor, order: ExpertOrder,
                             out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """Gradient of expert_dispatch: every token sums the gradients of its copies
    [tokens, dim].  Rows behind the last expert's are not read."""
    if _elsewhere(d_rows, stream):
        return _run_there(_combine, d_rows, stream, d_rows, None, order, out)
    return _combine(d_rows, None, order, out)


def expert_combine(rows: torch.Tensor, weights: torch.Tensor, order: ExpertOrder,
                   out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """The experts' rows back in token order: out[t] is the sum over j of
    weights[t, j] * rows[order.position[t, j]].  Dropped assignments add nothing,
    whatever their weight; a token without any gets zeros.  Records no graph: the
    gradients are expert_combine_backward."""
    if _elsewhere(rows, stream):
        return _run_there(_combine, rows, stream, rows, weights, order, out)
    return _combine(rows, weights, order, out)


def expert_combine_backward(d_out: torch.Tensor, rows: torch.Tensor, weights: torch.Tensor,
                            order: ExpertOrder, out: Optional[torch.Tensor] = None, stream=None):
    """Gradients of expert_combine: (d_rows, d_weights).  The rows of d_rows
    behind the last expert's are zeros in a new tensor and left as they are in
    ``out``; the weights of dropped assignments get 0."""
    if _elsewhere(d_out, stream):
        return _run_there(expert_combine_backward, d_out, stream, d_out, rows, weights, order, out)
    if weights is None:
        raise ValueError("weights must be those of expert_combine")
    n, dim, d_stride, kind = _float_rows(d_out, "d_out")
    tokens, top_k, experts, offsets, position = _order(order, d_out)
    if n != tokens:
        raise ValueError("d_out must have a row for every token of the order")
    stride = _more_rows(rows, "rows", tokens * top_k, dim, d_out)
    w = _weights(weights, order, rows)
    new = out is None
    out, out_stride = _out(out, tokens * top_k, dim, rows)
    d_weights = weights.new_empty((tokens, top_k))
    lib = load_library()
    rc = lib.hkv_expert_combine_backward(
        tokens, top_k, dim, kind, d_out.data_ptr(), d_stride, rows.data_ptr(), stride, w,
        _ROW_KINDS[weights.dtype], experts, offsets, position, out.data_ptr(), out_stride, new,
        d_weights.data_ptr(), _raw_stream(d_out.get_device()))
    if rc:
        _fail(lib, rc)
    return out, d_weights


def _params(weight, bias, dim, like):
    """Addresses of weight and bias and their kind."""
    w = _vector(weight, "weight", dim, like)
    b = _vector(bias, "bias", dim, like)
    if weight is None:
        return w, b, _ROW_KINDS[like.dtype if bias is None else bias.dtype]
    if bias is not None and weight.dtype is not bias.dtype:
        raise ValueError("weight and bias must have one type")
    return w, b, _ROW_KINDS[weight.dtype]


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, eps: float = 1e-5, stats: bool = True,
               out: Optional[torch.Tensor] = None, stream=None):
    """Layer norm of every row of x [n, dim].  Returns (y, mean, rstd), the
    statistics (float32 [n]) being what layer_norm_backward needs, or y alone
    with ``stats=False``.  Records no graph: the gradients are layer_norm_backward."""
    if _elsewhere(x, stream):
        return _run_there(layer_norm, x, stream, x, weight, bias, eps, stats, out)
    n, dim, stride, kind = _float_rows(x, "x")
    w, b, param_kind = _params(weight, bias, dim, x)
    y, y_stride = _out(out, n, dim, x)
    mean = rstd = None
    if stats:
        mean, rstd = x.new_empty(n, dtype=_F32), x.new_empty(n, dtype=_F32)
    lib = load_library()
    rc = lib.hkv_layer_norm(
        n, dim, kind, x.data_ptr(), stride, w, b, param_kind, eps, y.data_ptr(), y_stride,
        mean.data_ptr() if stats else None, rstd.data_ptr() if stats else None,
        _raw_stream(x.get_device()))
    if rc:
        _fail(lib, rc)
    return (y, mean, rstd) if stats else y


def layer_norm_ptr(n: int, row_ptrs: torch.Tensor, out: torch.Tensor,
                   weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                   eps: float = 1e-5, mean: Optional[torch.Tensor] = None,
                   rstd: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """layer_norm of n rows by address: ``row_ptrs`` (int64) as HashTable.find_ptr
    fills them, rows of the type and length of ``out``'s.  The rows are read where
    the table keeps them and must not change meanwhile (HashTable.find_layer_norm
    holds the table's lock over both steps).  Null addresses leave their row of
    ``out`` (and of ``mean`` and ``rstd``, float32, optional) as it is, and so do
    addresses where no table row of this length starts: those that are no multiple
    of 16 bytes where the row's length is one, else of 4, else of the element."""
    if _elsewhere(out, stream):
        return _run_there(layer_norm_ptr, out, stream, n, row_ptrs, out, weight, bias, eps, mean, rstd)
    rows, dim, stride, kind = _float_rows(out, "out")
    if not 0 <= n <= rows:
        raise ValueError("out must have n rows")
    if stride < dim * out.element_size():
        raise ValueError("the rows of out overlap")
    if row_ptrs.dtype is not torch.int64 or not row_ptrs.is_contiguous() or row_ptrs.numel() < n:
        raise ValueError("row_ptrs must be contiguous and hold n int64 addresses")
    if row_ptrs.get_device() != out.get_device():
        raise ValueError("row_ptrs must be on the device of out")
    w, b, param_kind = _params(weight, bias, dim, out)
    m, r = _statistic(mean, "mean", n, out), _statistic(rstd, "rstd", n, out)
    lib = load_library()
    rc = lib.hkv_layer_norm_ptr(n, dim, kind, row_ptrs.data_ptr(), w, b, param_kind, eps, out.data_ptr(),
                                stride, m, r, _raw_stream(out.get_device()))
    if rc:
        _fail(lib, rc)
    return out


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor],
                        mean: torch.Tensor, rstd: torch.Tensor, bias: bool = True,
                        out: Optional[torch.Tensor] = None, stream=None):
    """Gradients of layer_norm: (dx, d_weight, d_bias).  d_weight is None where
    the layer has no ``weight``, d_bias where ``bias`` is false; both have the
    type of ``weight`` (of the rows where there is none)."""
    if _elsewhere(x, stream):
        return _run_there(layer_norm_backward, x, stream, dy, x, weight, mean, rstd, bias, out)
    n, dim, stride, kind = _float_rows(x, "x")
    dy_stride = _more_rows(dy, "dy", n, dim, x)
    w, _, param_kind = _params(weight, None, dim, x)
    m, r = _statistic(mean, "mean", n, x), _statistic(rstd, "rstd", n, x)
    if m is None or r is None:
        raise ValueError("mean and rstd must be those of layer_norm")
    dx, dx_stride = _out(out, n, dim, x)
    lib = load_library()
    d_weight = torch.empty_like(weight) if weight is not None else None
    d_bias = None
    if bias:
        d_bias = torch.empty_like(weight) if weight is not None else x.new_empty(dim)
    work, work_bytes = None, 0
    if bias or weight is not None:
        work_bytes = lib.hkv_layer_norm_backward_workspace_bytes(n, dim, kind)
        work = x.new_empty(work_bytes, dtype=torch.uint8)
    rc = lib.hkv_layer_norm_backward(
        n, dim, kind, dy.data_ptr(), dy_stride, x.data_ptr(), stride, w, param_kind, m, r,
        dx.data_ptr(), dx_stride, d_weight.data_ptr() if d_weight is not None else None,
        d_bias.data_ptr() if bias else None, work.data_ptr() if work is not None else None,
        work_bytes, _raw_stream(x.get_device()))
    if rc:
        _fail(lib, rc)
    return dx, d_weight, d_bias
