"""The row operators on a GPU against plain 64-bit implementations: layer norm
and its gradients, expert sort / dispatch / combine and their gradients, the
table lookup with layer norm, and a training step of all of them together.

Tolerances.  u = 2^-24 bounds the relative error of one 32-bit operation.  A sum
of terms t passes every term through at most L additions, so it is off by at most
L * u * sum |t|: a thread adds at most max(64, D / 256) terms of a row, and 5
exchanges in the warp and 32 warps follow.  Results are rounded once, by at most
half a step of their type (finfo.eps / 2 of the value, or half the smallest
subnormal)."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)

import hierarchicalkv_b200 as hkv  # noqa: E402
from tests.hkv_testlib import to_dev, unique_keys  # noqa: E402

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]
SIZED = pytest.mark.parametrize("dtype", TYPES, ids=["f32", "f16", "bf16"])


def rounded(value, dtype):
    """How far rounding `value` to dtype may move it."""
    f = torch.finfo(dtype)
    return value.abs() * (f.eps / 2) + f.smallest_normal * f.eps / 2


def depth(dim):
    return max(64, dim // 256) + 48


def check(got, want, bound, what=""):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got.double() - want).abs()
    bad = ~(off <= bound)     # a NaN is bad
    assert not bad.any(), (what, int(bad.sum()), float(off[bad].max()), float((off / bound.clamp(min=1e-300)).max()))


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(shape, seed, dtype=torch.float32):
    return torch.randn(shape, generator=gen(seed), device="cuda").to(dtype)


def apart(rows, pad):
    """The rows as a slice of a wider matrix."""
    wide = torch.full((rows.shape[0], rows.shape[1] + pad), 7, dtype=rows.dtype, device=rows.device)
    wide[:, :rows.shape[1]] = rows
    return wide[:, :rows.shape[1]]


# ---- expert sort -----------------------------------------------------------------


def sort_oracle(ids, experts):
    flat = ids.cpu().numpy().reshape(-1).astype(np.int64)
    kept = np.flatnonzero((flat >= 0) & (flat < experts))
    taken = kept[np.argsort(flat[kept], kind="stable")]
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[kept], minlength=experts))])
    position = np.full(flat.size, -1, np.int64)
    position[taken] = np.arange(taken.size)
    source = np.full(flat.size, -1, np.int64)
    source[:taken.size] = taken
    return offsets, position.reshape(tuple(ids.shape)), source


def check_order(order, ids, experts):
    for got, want, name in zip(order, sort_oracle(ids, experts), order._fields):
        assert got.dtype == torch.int32
        np.testing.assert_array_equal(got.cpu().numpy(), want, err_msg=name)


def make_ids(tokens, top_k, experts, dtype=torch.int64, drop=0.0, seed=0):
    g = gen(seed)
    ids = torch.randint(0, experts, (tokens, top_k), generator=g, device="cuda")
    if drop:
        lost = torch.rand((tokens, top_k), generator=g, device="cuda") < drop
        wrong = torch.randint(0, 4, (tokens, top_k), generator=g, device="cuda")
        wrong = torch.tensor([-1, experts, -2 ** 31, 2 ** 31 - 1], device="cuda")[wrong]
        ids = torch.where(lost, wrong, ids)
    return ids.to(dtype)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("tokens,top_k", [(0, 2), (1, 1), (1, 8), (31, 1), (33, 3), (128, 8), (1025, 1), (513, 8),
                                          (4099, 2), (16384, 8), (9001, 13)])
@pytest.mark.parametrize("experts", [1, 2, 60, 257, 1024])
def test_sort_matches_a_stable_sort(tokens, top_k, experts, dtype):
    ids = make_ids(tokens, top_k, experts, dtype, drop=0.2, seed=tokens + experts)
    check_order(hkv.expert_sort(ids, experts), ids, experts)


@pytest.mark.parametrize("tokens,top_k,experts", [(131073, 1, 512), (200000, 6, 8), (70001, 8, 1024), (1 << 21, 1, 64)])
@pytest.mark.parametrize("drop", [0.0, 0.5])
def test_sort_of_large_batches(tokens, top_k, experts, drop):
    ids = make_ids(tokens, top_k, experts, drop=drop, seed=3)
    check_order(hkv.expert_sort(ids, experts), ids, experts)


@pytest.mark.parametrize("n", [5, 1000, 60000, 300000])
def test_sort_when_one_expert_takes_all_and_when_none_does(n):
    for fill in (3, -1, 7):
        ids = torch.full((n, 2), fill, device="cuda")
        check_order(hkv.expert_sort(ids, 7), ids, 7)


def test_sort_does_not_wrap_wide_ids():
    """An int64 id whose low half is an expert is still outside."""
    ids = torch.tensor([[1 << 32, 1], [(1 << 32) + 2, -(1 << 32)]], device="cuda")
    check_order(hkv.expert_sort(ids, 4), ids, 4)


# ---- dispatch and combine -----------------------------------------------------------


SHAPES = [(1, 1, 1, 1), (1, 8, 8, 64), (7, 3, 5, 33), (64, 2, 8, 8), (130, 5, 60, 100), (257, 8, 64, 1001),
          (33, 6, 4, 4096), (5, 64, 100, 16), (3, 2, 2, 20000)]


def token_rows(x, order, experts):
    """rows[p] = x[token of p] for the kept rows."""
    m = int(order.offsets[-1])
    return m, order.source[:m].long() // order.position.shape[1]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.uint8, torch.float64])
@pytest.mark.parametrize("tokens,top_k,experts,dim", SHAPES)
@pytest.mark.parametrize("pad", [0, 3])
def test_dispatch_copies_rows(tokens, top_k, experts, dim, dtype, pad):
    ids = make_ids(tokens, top_k, experts, drop=0.3, seed=dim)
    order = hkv.expert_sort(ids, experts)
    x = apart((randn((tokens, dim), 5) * 50).to(dtype), pad)
    m, token = token_rows(x, order, experts)
    got = hkv.expert_dispatch(x, order)
    assert torch.equal(got[:m], x[token])
    assert not got[m:].any()                               # a new tensor: zeros behind
    out = apart(torch.full_like(got, 9), pad)
    assert hkv.expert_dispatch(x, order, out=out) is out
    assert torch.equal(out[:m], x[token])
    assert (out[m:] == 9).all()                            # the caller's rows behind stay
    if pad:
        assert (out.as_strided((out.shape[0], pad), out.stride(), dim) == 7).all()   # and so does what lies between


@SIZED
@pytest.mark.parametrize("tokens,top_k,experts,dim", SHAPES)
@pytest.mark.parametrize("wide_weights", [False, True])
def test_combine_and_its_gradients(tokens, top_k, experts, dim, dtype, wide_weights):
    ids = make_ids(tokens, top_k, experts, drop=0.3, seed=dim + 1)
    order = hkv.expert_sort(ids, experts)
    n, m = tokens * top_k, int(order.offsets[-1])
    src = order.source[:m].long()
    token = src // top_k
    y = randn((n, dim), 1, dtype)
    y[m:] = float("nan")                                   # nobody's rows
    w = randn((tokens, top_k), 2, torch.float32 if wide_weights else dtype)
    w[order.position < 0] = float("inf")                   # weights of dropped assignments
    d_out = randn((tokens, dim), 4, dtype)
    w64, y64, d64 = w.double().reshape(-1)[src][:, None], y[:m].double(), d_out.double()[token]

    want = torch.zeros((tokens, dim), dtype=torch.float64, device="cuda").index_add_(0, token, y64 * w64)
    size = torch.zeros_like(want).index_add_(0, token, (y64 * w64).abs())
    got = hkv.expert_combine(y, w, order)
    check(got, want, (top_k + 1) * U * size + rounded(want, dtype), "combine")
    nobody = (order.position < 0).all(1)
    assert not got[nobody].any()

    d_rows, d_w = hkv.expert_combine_backward(d_out, y, w, order)
    assert d_rows.dtype == dtype and d_w.dtype == w.dtype
    want = d64 * w64
    check(d_rows[:m], want, U * want.abs() + rounded(want, dtype), "d_rows")
    assert not d_rows[m:].any()
    want = torch.zeros(n, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(want)
    want[src] = (d64 * y64).sum(1)
    size[src] = (d64 * y64).abs().sum(1)
    check(d_w.view(-1), want, depth(dim) * U * size + rounded(want, w.dtype), "d_weights")
    kept = apart(torch.full_like(d_rows, 9), 5)
    again, _ = hkv.expert_combine_backward(d_out, y, w, order, out=kept)
    assert again is kept and torch.equal(kept[:m], d_rows[:m]) and (kept[m:] == 9).all()

    # the gradient of dispatch: a token sums its copies'
    d_x = hkv.expert_dispatch_backward(y, order)
    want = torch.zeros((tokens, dim), dtype=torch.float64, device="cuda").index_add_(0, token, y64)
    size = torch.zeros_like(want).index_add_(0, token, y64.abs())
    check(d_x, want, top_k * U * size + rounded(want, dtype), "dispatch_backward")


@SIZED
@pytest.mark.parametrize("dim,pad", [(64, 1), (64, 4), (50, 8), (33, 1)])
def test_strided_and_unaligned_rows_give_the_same(dim, pad, dtype):
    """Another access width must not change a bit of the sums' order over k."""
    tokens, top_k, experts = 101, 3, 9
    order = hkv.expert_sort(make_ids(tokens, top_k, experts, seed=1), experts)
    y, w, d = randn((tokens * top_k, dim), 1, dtype), randn((tokens, top_k), 2), randn((tokens, dim), 3, dtype)
    assert torch.equal(hkv.expert_combine(apart(y, pad), w, order), hkv.expert_combine(y, w, order))
    assert torch.equal(hkv.expert_dispatch(apart(d, pad), order), hkv.expert_dispatch(d, order))
    rows, dw = hkv.expert_combine_backward(apart(d, pad), apart(y, pad), w, order)
    rows2, dw2 = hkv.expert_combine_backward(d, y, w, order)
    assert torch.equal(rows, rows2)
    size = (d[:, None].double() * y[order.position.long()].double()).abs().sum(2)
    check(dw, dw2.double(), 2 * depth(dim) * U * size + 1e-30, "d_weights")
    odd = torch.empty(tokens * dim + 1, dtype=dtype, device="cuda")[1:].view(tokens, dim)
    odd.copy_(d)
    assert torch.equal(hkv.expert_dispatch(odd, order), hkv.expert_dispatch(d, order))


def test_an_expert_twice_and_places_out_of_range():
    """One token may go to one expert several times; places outside the rows (an
    order that does not belong to them) count as dropped and reach no memory."""
    ids = torch.tensor([[2, 2, 2], [0, 2, 0]], device="cuda")
    order = hkv.expert_sort(ids, 3)
    check_order(order, ids, 3)
    y, w = randn((6, 8), 1), randn((2, 3), 2)
    want = (y[order.position.long()].double() * w.double()[:, :, None])
    check(hkv.expert_combine(y, w, order), want.sum(1), 4 * U * want.abs().sum(1))
    bad = hkv.ExpertOrder(order.offsets, order.position.clone(), order.source)
    bad.position[0, 1] = 6
    bad.position[1, 0] = -5
    bad.position[1, 2] = 2 ** 31 - 1
    ok = (bad.position >= 0) & (bad.position < 6)
    got = hkv.expert_combine(y, w, bad)
    check(got, torch.where(ok[:, :, None], want, 0).sum(1), 4 * U * want.abs().sum(1))
    rows = torch.full((6, 8), 9.0, device="cuda")
    x = randn((2, 8), 3)
    hkv.expert_dispatch(x, bad, out=rows)
    for t in range(2):
        for j in range(3):
            row = rows[order.position[t, j]]
            assert torch.equal(row, x[t]) if ok[t, j] else (row == 9).all()
    _, dw = hkv.expert_combine_backward(x, y, w, bad, out=rows)
    assert not dw[~ok].any() and dw[ok].all()
    # offsets that claim more rows than there are zero nothing, negative ones everything
    far = hkv.ExpertOrder(order.offsets + 100, torch.full_like(order.position, -1), order.source)
    assert hkv.expert_dispatch(x, far).shape == (6, 8)
    low = hkv.ExpertOrder(order.offsets - 100, torch.full_like(order.position, -1), order.source)
    assert not hkv.expert_dispatch(x, low).any()


def test_wide_rows_past_32_bit_offsets():
    """Rows whose byte offsets do not fit 32 bits."""
    tokens, top_k, dim = 70000, 2, 16384
    order = hkv.expert_sort(make_ids(tokens, top_k, 4, seed=2), 4)
    x = torch.arange(tokens, device="cuda").to(torch.int32)[:, None].expand(tokens, dim // 2).contiguous()
    rows = hkv.expert_dispatch(x, order)                    # 140,000 rows of 32 KiB: 4.6 GB
    assert rows.numel() * 4 > 2 ** 32
    token = order.source.long() // top_k
    assert torch.equal(rows[:, 0].long(), token) and torch.equal(rows[:, -1].long(), token)
    back = hkv.expert_combine(rows.view(torch.bfloat16), torch.zeros((tokens, top_k), device="cuda"), order)
    assert back.shape == (tokens, dim)


# ---- layer norm -----------------------------------------------------------------------


def norm_oracle(x, w, b, eps):
    x = x.double()
    mean = x.mean(1)
    d = x - mean[:, None]
    var = (d * d).mean(1)
    rstd = (var + eps) ** -0.5
    w = torch.ones(x.shape[1], device="cuda").double() if w is None else w.double()
    b = torch.zeros_like(w) if b is None else b.double()
    return d * rstd[:, None] * w + b, mean, rstd, d, w


def check_norm(got, x, w, b, eps, stats=None):
    y, mean, rstd, d, w64 = norm_oracle(x, w, b, eps)
    lu = depth(x.shape[1]) * U
    dm = ((lu + 3 * U) * x.double().abs().mean(1))          # of the mean
    # of rstd, relative: half of what the variance is off, which a wrong mean moves too
    rel = 0.5 * (lu + 6 * U) + (dm * rstd) + (dm * rstd) ** 2 + 4 * U
    xhat = d * rstd[:, None]
    off = w64.abs() * (rstd * dm)[:, None] * 2 + (w64 * xhat).abs() * (rel[:, None] + 4 * U) + 2 * U * y.abs()
    check(got, y, off + rounded(y, got.dtype), "y")
    if stats is not None:
        check(stats[0], mean, dm + U * mean.abs(), "mean")
        check(stats[1], rstd, (rel + U) * rstd, "rstd")


def norm_rows(n, dim, seed, dtype):
    x = torch.randn((n, dim), generator=gen(seed), device="cuda")
    x = x * (0.1 + 2 * torch.rand((n, 1), generator=gen(seed + 1), device="cuda"))
    return (x + 3 * torch.randn((n, 1), generator=gen(seed + 2), device="cuda")).to(dtype)


NORMS = [(1, 1), (3, 2), (5, 7), (1000, 8), (33, 31), (517, 64), (40, 100), (257, 128), (9, 333), (65, 512),
         (17, 1000), (3, 1023), (31, 1024), (700, 2048), (4, 4096), (5, 5000), (3, 8192), (2, 12289), (3, 16384),
         (2, 40000), (1, 70000)]


@SIZED
@pytest.mark.parametrize("n,dim", NORMS)
@pytest.mark.parametrize("wide_params", [False, True])
def test_layer_norm(n, dim, dtype, wide_params):
    x = norm_rows(n, dim, dim, dtype)
    pt = torch.float32 if wide_params else dtype
    w, b = (1 + 0.2 * randn((dim,), 7)).to(pt), randn((dim,), 8, pt)
    y, mean, rstd = hkv.layer_norm(x, w, b, 1e-5)
    check_norm(y, x, w, b, 1e-5, (mean, rstd))
    assert torch.equal(hkv.layer_norm(x, w, b, 1e-5, stats=False), y)
    check_norm(hkv.layer_norm(x, eps=0.5, stats=False), x, None, None, 0.5)
    check_norm(hkv.layer_norm(x, None, b, stats=False), x, None, b, 1e-5)


@SIZED
@pytest.mark.parametrize("dim", [64, 333, 2048])
def test_layer_norm_of_strided_rows_into_the_callers(dim, dtype):
    x = norm_rows(50, dim, 3, dtype)
    w = (1 + randn((dim,), 1)).to(dtype)
    for pad in (1, 2, 8):
        out = apart(torch.zeros_like(x), pad)
        y, mean, rstd = hkv.layer_norm(apart(x, pad), w, out=out)
        assert y is out
        check_norm(y, x, w, None, 1e-5, (mean, rstd))
        assert (out.as_strided((50, pad), out.stride(), dim) == 7).all()


def test_layer_norm_of_difficult_rows():
    """Far from zero, constant, with NaN, with infinity: each row for itself."""
    dim = 256
    x = norm_rows(8, dim, 1, torch.float32)
    x[1] += 3.0e4                      # the mean is large against the spread
    x[2] = 2.5                         # no spread at all
    x[3, 17] = float("nan")
    x[4, 200] = float("inf")
    x[5] *= 1e-30                      # the variance underflows: eps alone is left
    x[6] *= 1e15
    w, b = randn((dim,), 2), randn((dim,), 3)
    y, mean, rstd = hkv.layer_norm(x, w, b)
    fine = torch.tensor([0, 1, 2, 5, 6, 7], device="cuda")
    check_norm(y[fine], x[fine], w, b, 1e-5, (mean[fine], rstd[fine]))
    assert torch.equal(y[2], b)
    assert y[3].isnan().all() and y[4].isnan().any()
    y0 = hkv.layer_norm(x[2:3].contiguous(), w, b, eps=0.0, stats=False)
    assert y0.isnan().all()            # 0 / 0, as the formula says


def norm_grad_oracle(dy, x, w, mean, rstd):
    dy, x = dy.double(), x.double()
    mean, rstd = mean.double()[:, None], rstd.double()[:, None]
    w = torch.ones(x.shape[1], device="cuda").double() if w is None else w.double()
    xhat = (x - mean) * rstd
    g = dy * w
    m0, m1 = g.mean(1, keepdim=True), (g * xhat).mean(1, keepdim=True)
    dx = rstd * (g - m0 - xhat * m1)
    lu = depth(x.shape[1]) * U
    off = rstd * (8 * U * (g.abs() + m0.abs() + (xhat * m1).abs()) + (lu + 4 * U) * g.abs().mean(1, keepdim=True)
                  + xhat.abs() * (lu + 8 * U) * (g * xhat).abs().mean(1, keepdim=True))
    # a column: at most n / 64 rows in one thread, then the groups, the blocks and the warps
    lr = (x.shape[0] // 64 + 96) * U
    return ((dx, off), ((dy * xhat).sum(0), (lr + 6 * U) * (dy * xhat).abs().sum(0)), (dy.sum(0), lr * dy.abs().sum(0)))


def check_norm_grad(got, dy, x, w, mean, rstd):
    for name, value, (want, off) in zip(("dx", "d_weight", "d_bias"), got, norm_grad_oracle(dy, x, w, mean, rstd)):
        if value is not None:
            check(value, want, off + rounded(want, value.dtype), name)


@SIZED
@pytest.mark.parametrize("n,dim", NORMS + [(20011, 64), (5003, 320), (3001, 1001)])
@pytest.mark.parametrize("wide_params", [False, True])
def test_layer_norm_backward(n, dim, dtype, wide_params):
    x = norm_rows(n, dim, dim + 1, dtype)
    dy = randn((n, dim), 5, dtype)
    w = (1 + 0.2 * randn((dim,), 7)).to(torch.float32 if wide_params else dtype)
    _, mean, rstd = hkv.layer_norm(x, w)
    got = hkv.layer_norm_backward(dy, x, w, mean, rstd)
    assert got[0].dtype == dtype and got[1].dtype == got[2].dtype == w.dtype
    check_norm_grad(got, dy, x, w, mean, rstd)
    again = hkv.layer_norm_backward(dy, x, w, mean, rstd)
    assert all(torch.equal(p, q) for p, q in zip(got, again))     # no atomics: the same bits


@SIZED
@pytest.mark.parametrize("dim", [1, 2, 7, 8, 16, 24, 33, 40, 64, 66, 100, 130, 161, 200, 256, 258, 333, 390, 449, 511, 516,
                                 520, 776, 1001, 1032, 1160, 2049, 2240, 4104, 9000])
def test_more_rows_than_run_at_once(dim, dtype):
    """Batches that wait in queues, on every number of threads per row: whole, by
    address with misses, strided, and the gradient."""
    n = max(310000 // max(2, dim * torch.finfo(dtype).bits // 128), 3 * 148) + 3
    x = norm_rows(n, dim, dim, dtype)
    w, b = 1 + 0.2 * randn((dim,), 7), randn((dim,), 8)
    y, mean, rstd = hkv.layer_norm(x, w, b)
    check_norm(y, x, w, b, 1e-5, (mean, rstd))
    wide = apart(x, 1)
    padded, m, r = hkv.layer_norm(wide, w, b)
    check_norm(padded, x, w, b, 1e-5, (m, r))
    ptrs = x.data_ptr() + torch.arange(n, device="cuda") * (dim * x.element_size())
    miss = torch.arange(n, device="cuda") % 5 == 2
    ptrs[miss] = 0
    out = torch.full_like(x, 5)
    hkv.layer_norm_ptr(n, ptrs, out, w, b)
    check_norm(out[~miss], x[~miss], w, b, 1e-5)
    assert (out[miss] == 5).all()
    dy = randn((n, dim), 5, dtype)
    got = hkv.layer_norm_backward(dy, x, w, mean, rstd)
    check_norm_grad(got, dy, x, w, mean, rstd)
    check_norm_grad(hkv.layer_norm_backward(apart(dy, 1), wide, w, mean, rstd), dy, x, w, mean, rstd)


@SIZED
def test_layer_norm_backward_without_weight_or_bias_and_strided(dtype):
    n, dim = 77, 96
    x, dy = norm_rows(n, dim, 1, dtype), randn((n, dim), 5, dtype)
    _, mean, rstd = hkv.layer_norm(x)
    w = randn((dim,), 6, dtype)
    got = hkv.layer_norm_backward(dy, x, None, mean, rstd)
    assert got[1] is None
    check_norm_grad(got, dy, x, None, mean, rstd)
    got = hkv.layer_norm_backward(dy, x, None, mean, rstd, bias=False)
    assert got[1] is None and got[2] is None
    check_norm_grad(got, dy, x, None, mean, rstd)
    got = hkv.layer_norm_backward(dy, x, w, mean, rstd, bias=False)
    assert got[2] is None
    check_norm_grad(got, dy, x, w, mean, rstd)
    for pad in (1, 2, 8):
        out = apart(torch.zeros_like(x), pad)
        got = hkv.layer_norm_backward(apart(dy, pad), apart(x, pad), w, mean, rstd, out=out)
        assert got[0] is out
        check_norm_grad(got, dy, x, w, mean, rstd)
    # one gradient row for all rows: a distance of zero
    one = dy[:1].expand(n, dim)
    check_norm_grad(hkv.layer_norm_backward(one, x, w, mean, rstd), one, x, w, mean, rstd)


def test_no_rows():
    x, w = torch.empty((0, 16), device="cuda"), torch.ones(16, device="cuda")
    y, mean, rstd = hkv.layer_norm(x, w)
    assert y.shape == (0, 16) and mean.shape == rstd.shape == (0,)
    dx, dw, db = hkv.layer_norm_backward(x, x, w, mean, rstd)
    assert dx.shape == (0, 16) and not dw.any() and not db.any() and dw.shape == db.shape == (16,)
    order = hkv.expert_sort(torch.empty((0, 2), dtype=torch.int64, device="cuda"), 4)
    assert not order.offsets.any() and order.position.shape == (0, 2)
    assert hkv.expert_dispatch(x, order).shape == (0, 16)
    assert hkv.expert_combine(x, torch.empty((0, 2), device="cuda"), order).shape == (0, 16)
    d_rows, d_w = hkv.expert_combine_backward(x, x, torch.empty((0, 2), device="cuda"), order)
    assert d_rows.shape == (0, 16) and d_w.shape == (0, 2)
    ptrs = torch.empty(0, dtype=torch.int64, device="cuda")
    assert hkv.layer_norm_ptr(0, ptrs, x).shape == (0, 16)


def test_gradients_against_differences():
    """Directional differences of the forward kernels, f summed in 64 bits.  Along
    x + t v a row's y is (xhat + t a) / sqrt(1 + 2 t p + t^2 q) * w + b with
    a = rstd (v - mean(v)), q = mean(a^2), p = mean(xhat a): its t^3 term is at most
    (4 q^1.5 |xhat| + 2 q |a|) |w|, which the central difference shows times h^2 (twice that
    covers the terms behind it, as h sqrt(q) stays below 1/4).  The kernel's y is off by
    the sum's 18 additions of a mean, seen through rstd * mean|x|, and a few
    operations of its own: 32 u (1 + rstd mean|x|) (|y - b| + |b| + |w|)."""
    n, dim, h = 40, 48, 2.0 ** -6
    x, v, c = norm_rows(n, dim, 2, torch.float32), randn((n, dim), 3), randn((n, dim), 4)
    w, b = 1 + 0.2 * randn((dim,), 5), randn((dim,), 6)
    f = lambda t, w=w, b=b: (hkv.layer_norm(t, w, b, stats=False).double() * c.double())   # noqa: E731
    y, mean, rstd = hkv.layer_norm(x, w, b)
    dx, dw, db = hkv.layer_norm_backward(c, x, w, mean, rstd)
    r64 = rstd.double()[:, None]
    off = 32 * U * (1 + r64 * x.double().abs().mean(1, keepdim=True)) * ((y - b).abs() + b.abs() + w.abs()) * c.abs() / h
    a = r64 * (v - v.mean(1, keepdim=True))
    q = (a * a).mean(1, keepdim=True)
    assert float(h * q.sqrt().max()) < 0.25
    third = 2 * h * h * (4 * q ** 1.5 * ((y - b) / w).abs() + 2 * q * a.abs()) * (w * c).abs()
    slope = ((f(x + h * v) - f(x - h * v)) / (2 * h)).sum(1)
    check(dx.double().mul(v.double()).sum(1), slope, (off + third).sum(1))
    dv = randn((dim,), 7)
    slope = ((f(x, w + h * dv) - f(x, w - h * dv)) / (2 * h)).sum()
    assert abs(slope - (dw.double() * dv).sum()) <= 2 * off.sum()
    slope = ((f(x, w, b + h * dv) - f(x, w, b - h * dv)) / (2 * h)).sum()
    assert abs(slope - (db.double() * dv).sum()) <= 2 * off.sum()

    tokens, top_k, experts = 30, 3, 5                         # combine is bilinear: differences are exact
    order = hkv.expert_sort(make_ids(tokens, top_k, experts, drop=0.2, seed=4), experts)
    y, wt, c = randn((tokens * top_k, dim), 1), randn((tokens, top_k), 2), randn((tokens, dim), 3)
    dy, dwt = randn((tokens * top_k, dim), 4), randn((tokens, top_k), 5)
    f = lambda y, wt: (hkv.expert_combine(y, wt, order).double() * c.double()).sum()   # noqa: E731
    size = hkv.expert_combine(y.abs() + dy.abs(), wt.abs() + dwt.abs(), order).double().mul(c.abs()).sum()
    d_rows, d_w = hkv.expert_combine_backward(c, y, wt, order)
    assert abs((f(y + dy, wt) - f(y - dy, wt)) / 2 - (d_rows.double() * dy).sum()) <= 16 * U * size
    assert abs((f(y, wt + dwt) - f(y, wt - dwt)) / 2 - (d_w.double() * dwt).sum()) <= (16 + dim) * U * size


# ---- rows by address, and the lookup with layer norm ---------------------------------------


@SIZED
@pytest.mark.parametrize("n,dim", [(1, 1), (300, 64), (65, 33), (40, 512), (9, 2050), (3, 16384)])
def test_layer_norm_of_rows_by_address(n, dim, dtype):
    table = norm_rows(2 * n + 3, dim, 9, dtype)
    at = torch.randint(0, 2 * n + 3, (n,), generator=gen(1), device="cuda")
    ptrs = table.data_ptr() + at * (dim * table.element_size())
    miss = torch.rand(n, generator=gen(2), device="cuda") < 0.3
    ptrs[miss] = 0
    w, b = (1 + randn((dim,), 3)).to(dtype), randn((dim,), 4, dtype)
    out = torch.full((n + 2, dim), 5, dtype=dtype, device="cuda")
    mean, rstd = torch.full((n,), 5.0, device="cuda"), torch.full((n,), 5.0, device="cuda")
    assert hkv.layer_norm_ptr(n, ptrs, out, w, b, 1e-5, mean, rstd) is out
    hit = ~miss
    check_norm(out[:n][hit], table[at[hit]], w, b, 1e-5, (mean[hit], rstd[hit]))
    assert (out[:n][miss] == 5).all() and (out[n:] == 5).all()
    assert (mean[miss] == 5).all() and (rstd[miss] == 5).all()


@SIZED
@pytest.mark.parametrize("n,dim", [(7, 64), (7, 66), (7, 1025), (5000, 64), (5000, 66), (3, 20000)])
def test_addresses_where_no_row_starts_leave_their_row(n, dim, dtype):
    """An address that a row of this length cannot have counts as null: nothing is
    read there."""
    size = torch.finfo(dtype).bits // 8
    align = 16 if dim * size % 16 == 0 else 4 if dim * size % 4 == 0 else size
    table = norm_rows(n + 1, dim, 9, dtype)
    ptrs = table.data_ptr() + torch.arange(n, device="cuda") * (dim * size)
    odd = torch.arange(n, device="cuda") % 3 == 1
    ptrs[odd] += torch.arange(n, device="cuda")[odd] % (align - 1) + 1
    out = torch.full((n, dim), 5, dtype=dtype, device="cuda")
    mean, rstd = torch.full((n,), 5.0, device="cuda"), torch.full((n,), 5.0, device="cuda")
    hkv.layer_norm_ptr(n, ptrs, out, mean=mean, rstd=rstd)
    want, m, r = hkv.layer_norm(table[:n])
    assert torch.equal(out[~odd], want[~odd]) and torch.equal(mean[~odd], m[~odd]) and torch.equal(rstd[~odd], r[~odd])
    assert (out[odd] == 5).all() and (mean[odd] == 5).all() and (rstd[odd] == 5).all()


def make_table(dim, dtype=torch.float32, capacity=128 * 64, hbm=1 << 30, **options):
    t = hkv.HashTable(hkv.EvictStrategy.kLru, value_dtype=dtype)
    t.init(hkv.HashTableOptions(init_capacity=capacity, max_capacity=capacity, max_hbm_for_vectors=hbm, dim=dim,
                                **options))
    return t


@SIZED
@pytest.mark.parametrize("dim,hbm,options", [(64, 1 << 30, {}), (33, 1 << 30, {}), (64, 128 * 20 * 256, {}), (8, 0, {}),
                                             (16, 1 << 30, dict(max_bucket_size=64)), (16, 1 << 30, dict(slot_layout=1))])
def test_find_layer_norm_is_find_then_layer_norm(dim, hbm, options, dtype):
    t = make_table(dim, dtype, hbm=hbm, **options)
    keys = unique_keys(5000, seed=4)
    stored, rows = to_dev(keys[:4000]), norm_rows(4000, dim, 5, dtype)
    t.insert_or_assign(4000, stored, rows)
    n = 3000
    q = to_dev(np.concatenate([keys[1500:4000], keys[4500:]]))
    w, b = 1 + randn((dim,), 3), randn((dim,), 4)
    found = torch.zeros(n, dtype=torch.bool, device="cuda")
    out = torch.full((n, dim), 5, dtype=dtype, device="cuda")
    mean, rstd = torch.full((n,), 5.0, device="cuda"), torch.full((n,), 5.0, device="cuda")
    t.find_layer_norm(n, q, out, found, w, b, 1e-5, mean, rstd)
    plain, found2 = torch.zeros_like(out), torch.zeros_like(found)
    t.find(n, q, plain, found2)
    assert torch.equal(found, found2) and found[:2500].all() and not found[2500:].any()
    want, m, r = hkv.layer_norm(plain, w, b, 1e-5)
    assert torch.equal(out[found], want[found])
    assert torch.equal(mean[found], m[found]) and torch.equal(rstd[found], r[found])
    assert (out[~found] == 5).all() and (mean[~found] == 5).all() and (rstd[~found] == 5).all()
    only = torch.full((n, dim), 5, dtype=dtype, device="cuda")
    t.find_layer_norm(n, q, only, found)
    assert torch.equal(only[found], hkv.layer_norm(plain, stats=False)[found])
    t.find_layer_norm(0, q, only, found)
    t.close()


def test_find_layer_norm_refusals():
    t = make_table(8)
    k = torch.arange(4, device="cuda")
    v, f = torch.zeros((4, 8), device="cuda"), torch.zeros(4, dtype=torch.bool, device="cuda")
    w = torch.ones(8, device="cuda")
    for bad in (dict(weight=w[:7]), dict(weight=w.half()), dict(bias=w.double()), dict(weight=w, bias=w.half()),
                dict(mean=torch.zeros(3, device="cuda")), dict(rstd=w.half()), dict(eps=-1.0), dict(eps=float("nan"))):
        with pytest.raises(ValueError):
            t.find_layer_norm(4, k, v, f, **bad)
    with pytest.raises(ValueError):
        t.find_layer_norm(5, k, v, f)
    with pytest.raises(ValueError):
        t.find_layer_norm(4, k, v.half(), f)
    t.close()
    ints = make_table(8, torch.int64)
    with pytest.raises(hkv.MerlinException, match="float, half or bfloat16"):
        ints.find_layer_norm(4, k, torch.zeros((4, 8), dtype=torch.int64, device="cuda"), f)
    ints.close()
    dual = make_table(8, hbm=0, table_mode=1)
    with pytest.raises(hkv.MerlinException, match="MEMORY_MODE"):
        dual.find_layer_norm(4, k, v, f)
    dual.close()


def test_find_layer_norm_waits_for_updates_on_another_stream():
    """The lookup and the reading of the rows take the table's reader lock: each
    row is normalised as it was before or after an update, never half of each."""
    dim, n = 64, 8192
    t = make_table(dim, capacity=1 << 16)
    k = to_dev(unique_keys(n, seed=1))
    a, b = norm_rows(n, dim, 1, torch.float32), norm_rows(n, dim, 2, torch.float32)
    t.insert_or_assign(n, k, a)
    want = [hkv.layer_norm(v, stats=False) for v in (a, b)]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for turn in range(6):
        out = torch.zeros((n, dim), device="cuda")
        found = torch.zeros(n, dtype=torch.bool, device="cuda")
        side.wait_stream(torch.cuda.current_stream())
        t.find_layer_norm(n, k, out, found, stream=side)
        t.assign(n, k, b if turn % 2 == 0 else a)
        outs.append(out)
    torch.cuda.synchronize()
    for out in outs:
        either = (out == want[0]).all(1) | (out == want[1]).all(1)
        assert either.all()
    t.close()


# ---- streams and graphs ---------------------------------------------------------------------


def expert_pass(x, ids, w, experts):
    order = hkv.expert_sort(ids, experts)
    rows = hkv.expert_dispatch(x, order)
    out = hkv.expert_combine(rows, w, order)
    d_rows, d_w = hkv.expert_combine_backward(out, rows, w, order)
    return [*order, rows, out, d_rows, d_w, hkv.expert_dispatch_backward(d_rows, order)]


def norm_pass(x, w, b, dy):
    y, mean, rstd = hkv.layer_norm(x, w, b)
    return [y, mean, rstd, *hkv.layer_norm_backward(dy, x, w, mean, rstd)]


def test_streams_by_object_and_by_handle():
    x, w, dy = norm_rows(3000, 64, 1, torch.float32), randn((64,), 2), randn((3000, 64), 3)
    want = norm_pass(x, w, w, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for stream in (side, side.cuda_stream, 0):
        y, mean, rstd = hkv.layer_norm(x, w, w, stream=stream)
        got = [y, mean, rstd, *hkv.layer_norm_backward(dy, x, w, mean, rstd, stream=stream)]
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    with torch.cuda.stream(side):                            # the current stream is the one that runs
        got = norm_pass(x, w, w, dy)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_calls_that_do_not_fit_are_refused():
    x, ids = randn((6, 8), 1), make_ids(6, 2, 3)
    order = hkv.expert_sort(ids, 3)
    rows, w = hkv.expert_dispatch(x, order), randn((6, 2), 2)

    class Elsewhere:                                       # a stream of another GPU, without one
        device = torch.device("cuda", torch.cuda.device_count())

    with pytest.raises(ValueError, match="stream"):
        hkv.layer_norm(x, stream=Elsewhere())
    for bad in (w.t().contiguous(), w[:5], w.view(-1)):
        with pytest.raises(ValueError, match="shape of order.position"):
            hkv.expert_combine(rows, bad, order)
        with pytest.raises(ValueError, match="shape of order.position"):
            hkv.expert_combine_backward(x, rows, bad, order)
    for bad in (x[:5], x[:, :7], x.half(), torch.zeros((12, 8))):
        with pytest.raises(ValueError):
            hkv.expert_combine_backward(x, bad, w, order)
        with pytest.raises(ValueError):
            hkv.expert_dispatch(x, order, out=bad)
        with pytest.raises(ValueError):
            hkv.layer_norm(x, out=bad)
        with pytest.raises(ValueError):
            hkv.layer_norm_backward(bad, x, None, w[:, 0].contiguous(), w[:, 1].contiguous())
    with pytest.raises(ValueError, match="overlap"):
        hkv.layer_norm(x, out=x[:1].expand(6, 8))
    with pytest.raises(ValueError, match="top_k"):
        hkv.expert_dispatch(x, hkv.ExpertOrder(order.offsets, torch.zeros((6, 65), dtype=torch.int32, device="cuda"), None))


FIRST_CALLS = """
import torch
import hierarchicalkv_b200 as hkv
hkv.load_library()
x = torch.randn((5000, 64), device="cuda")
w, ids = torch.ones(64, device="cuda"), torch.randint(0, 6, (5000, 2), device="cuda")
wt = torch.ones((5000, 2), device="cuda")
def calls():
    y, mean, rstd = hkv.layer_norm(x, w, w)
    order = hkv.expert_sort(ids, 6)
    rows = hkv.expert_dispatch(y, order)
    out = hkv.expert_combine(rows, wt, order)
    d_rows, d_wt = hkv.expert_combine_backward(out, rows, wt, order)
    dy = hkv.expert_dispatch_backward(d_rows, order)
    return [y, mean, rstd, *order, rows, out, d_rows, d_wt, dy, *hkv.layer_norm_backward(dy, x, w, mean, rstd)]
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = calls()
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, calls()))
print("same")
"""


def test_a_process_s_first_calls_may_be_captured():
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stdout + r.stderr


def test_captured_calls_replay_on_new_inputs_and_graphs_do_not_share_scratch():
    n, dim, experts, top_k = 20000, 32, 6, 8               # 160,000 assignments: the sort with scratch
    x, w, dy = norm_rows(n, dim, 1, torch.float32), randn((dim,), 2), randn((n, dim), 3)
    ids, wt = make_ids(n, top_k, experts, drop=0.1), randn((n, top_k), 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                            # warm-up
        norm_pass(x, w, w, dy)
        expert_pass(x, ids, wt, experts)
    torch.cuda.synchronize()
    graphs, results = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(norm_pass(x, w, w, dy) + expert_pass(x, ids, wt, experts))
        graphs.append(g)
    for turn in range(3):
        x.copy_(norm_rows(n, dim, 10 + turn, torch.float32))
        ids.copy_(make_ids(n, top_k, experts, drop=0.1, seed=turn))
        want = norm_pass(x, w, w, dy) + expert_pass(x, ids, wt, experts)
        a, b = torch.cuda.Stream(), torch.cuda.Stream()
        for s, g in ((a, graphs[0]), (b, graphs[1])):        # both at once
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for got in results:
            assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_calls_at_the_same_time():
    xs = [norm_rows(40000, 64, s, torch.float32) for s in range(4)]
    w, dy = randn((64,), 2), randn((40000, 64), 3)
    ids = [make_ids(40000, 4, 16, seed=s) for s in range(4)]
    wt = randn((40000, 4), 5)
    want = [norm_pass(x, w, w, dy) + expert_pass(x, i, wt, 16) for x, i in zip(xs, ids)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(3):
        got = []
        for s, x, i in zip(streams, xs, ids):
            with torch.cuda.stream(s):
                got.append(norm_pass(x, w, w, dy) + expert_pass(x, i, wt, 16))
        torch.cuda.synchronize()
        for p, q in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(p, q))


# ---- together -----------------------------------------------------------------------------------


def test_a_training_step_of_table_norm_and_experts():
    """Keys -> rows of the table -> layer norm -> experts and back -> a loss, and the
    gradient of it all into the table with accum_or_assign, against autograd in 64
    bits.  Each step's own tolerance is tested above; here the chain of about ten
    steps is held to 2^-12 of the largest value, far above ten times their 2^-20 and
    far below what a wrong term would leave."""
    dim, n, experts, top_k = 32, 600, 5, 2
    t = make_table(dim)
    keys = to_dev(unique_keys(n, seed=9))
    rows = norm_rows(n, dim, 1, torch.float32)
    t.insert_or_assign(n, keys, rows)
    w, b = 1 + 0.2 * randn((dim,), 2), randn((dim,), 3)
    ids, gate = make_ids(n, top_k, experts, drop=0.15, seed=4), torch.rand((n, top_k), generator=gen(5), device="cuda")
    mats = randn((experts, dim, dim), 6) / dim ** 0.5
    target = randn((n, dim), 7)

    x, found = torch.zeros((n, dim), device="cuda"), torch.zeros(n, dtype=torch.bool, device="cuda")
    t.find(n, keys, x, found)
    assert found.all()
    h, mean, rstd = hkv.layer_norm(x, w, b)
    order = hkv.expert_sort(ids, experts)
    xs = hkv.expert_dispatch(h, order)
    ends = order.offsets.tolist()
    ys = torch.zeros_like(xs)
    for e in range(experts):
        ys[ends[e]:ends[e + 1]] = (xs[ends[e]:ends[e + 1]].double() @ mats[e].double()).float()
    out = hkv.expert_combine(ys, gate, order)
    d_out = out - target
    d_ys, d_gate = hkv.expert_combine_backward(d_out, ys, gate, order)
    d_xs = torch.zeros_like(d_ys)
    for e in range(experts):
        d_xs[ends[e]:ends[e + 1]] = (d_ys[ends[e]:ends[e + 1]].double() @ mats[e].double().t()).float()
    d_h = hkv.expert_dispatch_backward(d_xs, order)
    dx, dw, db = hkv.layer_norm_backward(d_h, x, w, mean, rstd)
    lr = 0.125
    t.accum_or_assign(n, keys, -lr * dx, torch.ones(n, dtype=torch.bool, device="cuda"))
    after = torch.zeros((n, dim), device="cuda")
    t.find(n, keys, after, found)
    t.close()

    leaf = [v.double().requires_grad_() for v in (rows, w, b, gate)]
    r, w64, b64, g64 = leaf
    d = r - r.mean(1, keepdim=True)
    h64 = d * ((d * d).mean(1, keepdim=True) + 1e-5) ** -0.5 * w64 + b64
    kept = (ids >= 0) & (ids < experts)
    y64 = torch.einsum("nd,nkde->nke", h64, mats.double()[ids.clamp(0, experts - 1)])
    out64 = (y64 * torch.where(kept, g64, 0)[:, :, None]).sum(1)
    (0.5 * (out64 - target.double()).square().sum()).backward()
    for got, want in ((out, out64.detach()), (dx, r.grad), (dw, w64.grad), (db, b64.grad), (d_gate, g64.grad),
                      (after, (r - lr * r.grad).detach())):
        check(got, want, 2.0 ** -12 * want.abs().max().expand_as(want))
