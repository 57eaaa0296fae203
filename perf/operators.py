"""Cases, plain forms and timed calls of the row operators that follow a table lookup in a model:

  dispatch       token assignments sorted by expert, the token rows copied into that order
  dispatch_grad  the gradient of that copy: every token sums the gradients of its copies
  combine        expert rows back in token order, weighted and summed
  combine_grad   its gradient: of the expert rows and of the weights
  norm           layer norm of rows, with the row statistics where a training step keeps them
  norm_ptr       layer norm of table rows read at the addresses a pointer lookup returned
  norm_grad      layer norm's gradient: of the rows, the weight and the bias

With `own` false, `run` is the plain form in elementary torch operations; with `own` true it makes the
calls a user of hierarchicalkv_b200 makes.
"""
import numpy as np
import torch

own = False

_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_EPS = 1e-5
_MAX_BYTES = 600 << 20      # of the largest matrix of a drawn case
_EXPERT_KINDS = ("dispatch", "dispatch_grad", "combine", "combine_grad")


def _expert(name, kind, tokens, top_k, experts, dim, dtype, ids="int64", weights="float32", drop=0.0, pad=0):
    return {"name": name, "kind": kind, "tokens": tokens, "top_k": top_k, "experts": experts, "dim": dim,
            "dtype": dtype, "ids": ids, "weights": weights, "drop": drop, "pad": pad}


def _norm(name, kind, rows, dim, dtype, params="same", bias=True, stats=True, misses=0.0, pad=0):
    return {"name": name, "kind": kind, "rows": rows, "dim": dim, "dtype": dtype, "params": params,
            "bias": bias, "stats": stats, "misses": misses, "pad": pad}


def listed():
    return [
        # one decoding step of a few requests: the launches and the host's part are the time
        _expert("dispatch_decode", "dispatch", 8, 8, 64, 2048, "bfloat16"),
        # a prompt batch: the copies are the time
        _expert("dispatch_prompt", "dispatch", 16384, 8, 128, 4096, "bfloat16"),
        # a training step with rows that are no multiple of 16 bytes apart and a tenth of the assignments dropped
        _expert("dispatch_grad_odd", "dispatch_grad", 30011, 6, 60, 1001, "float16", ids="int32", drop=0.1),
        # one decoding step, back
        _expert("combine_decode", "combine", 8, 8, 64, 2048, "bfloat16"),
        # the 65,536-key batch of the table's correctness workload at the hybrid table's row width, two experts each
        _expert("combine_rows", "combine", 65536, 2, 8, 128, "float32", ids="int32", drop=0.1),
        # a training step's way back
        _expert("combine_grad", "combine_grad", 8192, 8, 64, 2048, "bfloat16", weights="same"),
        # one token's activations at a decoding step of a few requests, nothing kept for a backward pass
        _norm("norm_decode", "norm", 16, 8192, "bfloat16", stats=False),
        # odd row width: rows start at addresses that are multiples of two bytes only
        _norm("norm_odd", "norm", 65537, 333, "float16", params="float32", pad=2),
        # the headline batch of the table (1,048,576 rows of 64 floats), read in the table through find*'s addresses
        _norm("norm_ptr_batch", "norm_ptr", 1048576, 64, "float32", misses=0.1, stats=False),
        # the headline batch's rows in a training step
        _norm("norm_grad_batch", "norm_grad", 1048576, 64, "float32"),
        # a training step of a dense layer's activations
        _norm("norm_grad_wide", "norm_grad", 16384, 8192, "bfloat16", params="float32"),
        # a small ragged training batch
        _norm("norm_grad_small", "norm_grad", 517, 1000, "bfloat16", bias=False),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return min(high, max(low, round(low * (high / low) ** rng.random())))


def draw(rng):
    kind = rng.choice(_EXPERT_KINDS + ("norm", "norm_ptr", "norm_grad"))
    dtype = rng.choice(sorted(_TYPES))
    size = 4 if dtype == "float32" else 2
    step = rng.choice((1, 8, 64))
    dim = max(1, _spread(rng, 8, 8192) // step) * step
    pad = rng.choice((0, 0, 0, 1, 8))
    if kind in _EXPERT_KINDS:
        experts = _spread(rng, 2, 512)
        top_k = rng.randint(1, min(8, experts))
        tokens = _spread(rng, 1, min(131072, max(1, _MAX_BYTES // (dim * size * top_k))))
        case = _expert("", kind, tokens, top_k, experts, dim, dtype, ids=rng.choice(("int32", "int64")),
                       weights=rng.choice(("same", "float32")), drop=rng.choice((0.0, 0.0, 0.1, 0.5)), pad=pad)
    else:
        rows = _spread(rng, 1, min(1048576, max(1, _MAX_BYTES // (2 * dim * size))))
        case = _norm("", kind, rows, dim, dtype, params=rng.choice(("same", "float32")), bias=rng.random() < 0.8,
                     stats=rng.random() < 0.5, misses=rng.choice((0.0, 0.1, 0.5)), pad=pad)
        if kind == "norm_ptr":
            case["pad"] = 0
        else:
            case["misses"] = 0.0
        if kind == "norm_grad":
            case["stats"] = True
    del case["name"]
    return case


def _ints(shape, low, high, g, dtype=torch.int64):
    return torch.randint(low, high, shape, generator=g, device="cuda", dtype=dtype)


def _normal(shape, g, dtype):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _padded(rows, pad):
    """The same rows as a slice of a matrix that is `pad` columns wider."""
    if not pad:
        return rows
    wide = torch.zeros((rows.shape[0], rows.shape[1] + pad), dtype=rows.dtype, device=rows.device)
    wide[:, :rows.shape[1]] = rows
    return wide[:, :rows.shape[1]]


def _plain_order(ids, experts):
    """Stable sort by expert; ids outside [0, experts) are dropped: they sort behind everything."""
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    by_expert, order = torch.sort(key, stable=True)
    edges = torch.arange(experts + 1, device=ids.device)
    offsets = torch.searchsorted(by_expert, edges)
    place = torch.arange(flat.numel(), device=ids.device)
    position = torch.empty_like(place)
    position[order] = place
    position = torch.where(key < experts, position, -1)
    source = torch.where(place < offsets[-1], order, -1)
    return offsets.int(), position.int().view(ids.shape), source.int()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    kind, dim, dtype = case["kind"], case["dim"], _TYPES[case["dtype"]]
    s = {"case": case}
    if kind in _EXPERT_KINDS:
        t, k, e = case["tokens"], case["top_k"], case["experts"]
        # a router's scores: some experts are asked for more often than others
        scores = torch.randn((t, e), generator=g, device="cuda") + torch.randn((e,), generator=g, device="cuda")
        top, ids = torch.topk(scores, k, dim=1)
        if case["drop"]:
            lost = torch.rand((t, k), generator=g, device="cuda") < case["drop"]
            lost |= torch.rand((t, 1), generator=g, device="cuda") < case["drop"] / 4    # tokens nobody takes
            ids = torch.where(lost, torch.where(_ints((t, k), 0, 2, g) > 0, -1, e), ids)
        s["ids"] = ids.to(getattr(torch, case["ids"]))
        s["weights"] = torch.softmax(top, 1).to(torch.float32 if case["weights"] == "float32" else dtype)
        if kind == "dispatch":
            s["x"] = _padded(_normal((t, dim), g, dtype), case["pad"])
            return s
        s["order"] = _plain_order(s["ids"], e)
        if kind != "dispatch_grad":
            s["y"] = _normal((t * k, dim), g, dtype)
        if kind == "combine_grad":
            s["d_out"] = _padded(_normal((t, dim), g, dtype), case["pad"])
        if kind == "dispatch_grad":
            s["d_rows"] = _normal((t * k, dim), g, dtype)
        # what lies behind the last expert's rows is nobody's: no result may depend on it
        behind = torch.arange(t * k, device="cuda") >= s["order"][0][-1]
        for name in ("y", "d_rows"):
            if name in s and case["drop"]:
                s[name][behind] = float("nan")
        return s
    n = case["rows"]
    ptype = torch.float32 if case["params"] == "float32" else dtype
    s["weight"] = (1 + 0.1 * torch.randn((dim,), generator=g, device="cuda")).to(ptype)
    s["bias"] = (0.1 * torch.randn((dim,), generator=g, device="cuda")).to(ptype) if case["bias"] else None
    if kind == "norm_ptr":
        table = _normal((2 * n, dim), g, dtype)
        at = _ints((n,), 0, 2 * n, g)
        at = torch.where(torch.rand((n,), generator=g, device="cuda") < case["misses"], -1, at)
        s["table"], s["at"] = table, at
        s["row_ptrs"] = torch.where(at >= 0, table.data_ptr() + at * (dim * table.element_size()), 0)
        s["out"] = torch.zeros((n, dim), dtype=dtype, device="cuda")    # rows of misses stay as they are
        return s
    # rows with a mean and a spread of their own
    x = torch.randn((n, dim), generator=g, device="cuda")
    x *= torch.rand((n, 1), generator=g, device="cuda") + 0.5
    x += torch.randn((n, 1), generator=g, device="cuda")
    s["x"] = _padded(x.to(dtype), case["pad"])
    if kind == "norm_grad":
        x64 = s["x"].double()
        s["mean"] = x64.mean(1).float()
        s["rstd"] = (x64.var(1, unbiased=False) + _EPS).rsqrt().float()
        s["dy"] = _normal((n, dim), g, dtype)
    return s


def _plain_norm(x, weight, bias):
    x = x.float()
    mean = x.mean(1)
    x = x - mean[:, None]
    rstd = 1 / torch.sqrt((x * x).mean(1) + _EPS)
    y = x * rstd[:, None] * weight.float()
    return (y if bias is None else y + bias.float()), mean, rstd


def _own(s):
    import hierarchicalkv_b200 as hkv

    kind = s["case"]["kind"]
    if kind == "dispatch":
        order = hkv.expert_sort(s["ids"], s["case"]["experts"])
        return [*order, hkv.expert_dispatch(s["x"], order)]
    if kind == "dispatch_grad":
        return hkv.expert_dispatch_backward(s["d_rows"], hkv.ExpertOrder(*s["order"]))
    if kind == "combine":
        return hkv.expert_combine(s["y"], s["weights"], hkv.ExpertOrder(*s["order"]))
    if kind == "combine_grad":
        return hkv.expert_combine_backward(s["d_out"], s["y"], s["weights"], hkv.ExpertOrder(*s["order"]))
    if kind == "norm":
        return hkv.layer_norm(s["x"], s["weight"], s["bias"], _EPS, stats=s["case"]["stats"])
    if kind == "norm_ptr":
        return hkv.layer_norm_ptr(s["case"]["rows"], s["row_ptrs"], s["out"], s["weight"], s["bias"], _EPS)
    return hkv.layer_norm_backward(s["dy"], s["x"], s["weight"], s["mean"], s["rstd"], bias=s["case"]["bias"])


def run(s):
    if own:
        return _own(s)
    case = s["case"]
    kind, dtype = case["kind"], _TYPES[case["dtype"]]
    if kind == "dispatch":
        offsets, position, source = _plain_order(s["ids"], case["experts"])
        kept = (source >= 0)[:, None]
        rows = torch.where(kept, s["x"][source.clamp(min=0).long() // case["top_k"]], 0)
        return [offsets, position, source, rows]
    if kind in _EXPERT_KINDS:
        offsets, position, source = s["order"]
        kept = (position >= 0)[:, :, None]
        at = position.clamp(min=0).long()
    if kind == "dispatch_grad":
        return torch.where(kept, s["d_rows"][at].float(), 0).sum(1).to(dtype)
    if kind == "combine":
        return torch.where(kept, s["y"][at].float() * s["weights"].float()[:, :, None], 0).sum(1).to(dtype)
    if kind == "combine_grad":
        from_token = (source >= 0)[:, None]
        src = source.clamp(min=0).long()
        d_rows = s["d_out"][src // case["top_k"]].float() * s["weights"].float().reshape(-1)[src][:, None]
        d_weights = torch.where(kept, s["y"][at].float() * s["d_out"].float()[:, None, :], 0).sum(2)
        return [torch.where(from_token, d_rows, 0).to(dtype), d_weights.to(s["weights"].dtype)]
    if kind == "norm":
        y, mean, rstd = _plain_norm(s["x"], s["weight"], s["bias"])
        return [y.to(dtype), mean, rstd] if case["stats"] else y.to(dtype)
    if kind == "norm_ptr":
        y, _, _ = _plain_norm(s["table"][s["at"].clamp(min=0)], s["weight"], s["bias"])
        return torch.where((s["at"] >= 0)[:, None], y.to(dtype), s["out"])
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    xhat = (s["x"].float() - s["mean"][:, None]) * rstd
    g = dy * s["weight"].float()
    dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    # over up to a million rows: summed in 64 bits
    d_weight = (dy * xhat).sum(0, dtype=torch.float64).to(s["weight"].dtype)
    d_bias = dy.sum(0, dtype=torch.float64).to(s["weight"].dtype)
    return [dx.to(dtype), d_weight, d_bias] if case["bias"] else [dx.to(dtype), d_weight]


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["kind"] in _EXPERT_KINDS:
        t, k, dim = case["tokens"], case["top_k"], case["dim"]
        n = t * k
        kept = n * (1 - case["drop"]) * (1 - case["drop"] / 4)
        wsize = 4 if case["weights"] == "float32" else size
        if case["kind"] == "dispatch":
            ids = n * (4 if case["ids"] == "int32" else 8)
            return {"bytes": ids + 4 * (2 * n + case["experts"] + 1) + (t + n) * dim * size, "flops": n}
        if case["kind"] == "dispatch_grad":
            return {"bytes": 4 * n + (t + kept) * dim * size, "flops": kept * dim}
        if case["kind"] == "combine":
            return {"bytes": (4 + wsize) * n + (t + kept) * dim * size, "flops": 2 * kept * dim}
        return {"bytes": (4 + 2 * wsize) * n + (t + kept + n) * dim * size, "flops": 3 * kept * dim}
    n, dim = case["rows"], case["dim"]
    psize = (4 if case["params"] == "float32" else size) * dim * (2 if case["bias"] else 1)
    if case["kind"] == "norm":
        return {"bytes": 2 * n * dim * size + psize + (8 * n if case["stats"] else 0), "flops": 7 * n * dim}
    if case["kind"] == "norm_ptr":
        hits = n * (1 - case["misses"])
        return {"bytes": 8 * n + 2 * hits * dim * size + psize, "flops": 7 * hits * dim}
    return {"bytes": 3 * n * dim * size + 8 * n + 2 * psize, "flops": 14 * n * dim}


def _exact_order(ids, experts):
    """Places by counting, on the host: an expert's rows start behind those of the experts before it."""
    flat = ids.cpu().numpy().reshape(-1).astype(np.int64)
    kept = np.flatnonzero((flat >= 0) & (flat < experts))
    counts = np.bincount(flat[kept], minlength=experts)
    offsets = np.concatenate([[0], np.cumsum(counts)])
    taken = kept[np.lexsort((kept, flat[kept]))]
    source = np.full(flat.size, -1, np.int32)
    source[:taken.size] = taken
    position = np.full(flat.size, -1, np.int32)
    position[taken] = np.arange(taken.size)
    return offsets.astype(np.int32), position.reshape(tuple(ids.shape)), source


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in _EXPERT_KINDS:
        k = case["top_k"]
        offsets, position, source = _exact_order(s["ids"], case["experts"])
        m = int(offsets[-1])
        src = torch.from_numpy(source[:m].astype(np.int64)).cuda()
        token = src // k
        weight = s["weights"].double().reshape(-1)[src][:, None]
        n = source.size
    if kind == "dispatch":
        rows = torch.zeros((n, case["dim"]), dtype=torch.float64, device="cuda")
        rows[:m] = s["x"].double()[token]
        return [offsets, position, source, rows]
    if kind == "dispatch_grad":
        out = torch.zeros((case["tokens"], case["dim"]), dtype=torch.float64, device="cuda")
        return out.index_add_(0, token, s["d_rows"][:m].double())
    if kind == "combine":
        out = torch.zeros((case["tokens"], case["dim"]), dtype=torch.float64, device="cuda")
        return out.index_add_(0, token, s["y"][:m].double() * weight)
    if kind == "combine_grad":
        d_out = s["d_out"].double()[token]
        d_rows = torch.zeros((n, case["dim"]), dtype=torch.float64, device="cuda")
        d_rows[:m] = d_out * weight
        d_weights = torch.zeros(n, dtype=torch.float64, device="cuda")
        d_weights[src] = torch.linalg.vecdot(d_out, s["y"][:m].double())
        return [d_rows, d_weights.view(-1, k)]
    w = s["weight"].double()
    b = s["bias"].double() if s["bias"] is not None else torch.zeros_like(w)
    if kind in ("norm", "norm_ptr"):
        x = s["x"] if kind == "norm" else s["table"][s["at"].clamp(min=0)]
        var, mean = torch.var_mean(x.double(), 1, correction=0)
        rstd = (var + _EPS) ** -0.5
        y = torch.addcmul(b, (x.double() - mean[:, None]) * rstd[:, None], w)
        if kind == "norm_ptr":
            y[s["at"] < 0] = s["out"].double()[s["at"] < 0]
            return y
        return [y, mean, rstd] if case["stats"] else y
    dim, dy, rstd = case["dim"], s["dy"].double(), s["rstd"].double()[:, None]
    xhat = (s["x"].double() - s["mean"].double()[:, None]) * rstd
    first = (dy @ w)[:, None] / dim                              # the mean of g = dy * weight
    second = torch.linalg.vecdot(dy * xhat, w.expand_as(dy))[:, None] / dim
    dx = rstd * (dy * w - first - xhat * second)
    grads = [dx, torch.linalg.vecdot(dy.mT, xhat.mT)]
    return grads + [dy.mT.sum(1)] if case["bias"] else grads
