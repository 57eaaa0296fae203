"""The row operators at the edges of what their documents allow: stream captures,
rows far from zero, batches and offsets past the sizes of the other tests."""
import os
import sys
import threading

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


def test_find_layer_norm_on_several_streams_and_threads_at_once():
    """Readers share the table: the first takes the table's scratch, the others bring
    their own, and a batch that is larger than any before replaces the scratch while
    calls are under way.  Keys may come twice, and n may be one.  The bits are those of
    the same call alone (the order of a row's sums goes by the batch's size), and the
    rows those of the keys: their values are off by far less than 2^-12 of 1."""
    dim, stored = 48, 30000
    t = make_table(dim, capacity=1 << 16)
    keys, rows = to_dev(unique_keys(stored, seed=5)), torch.randn((stored, dim), device="cuda")
    t.insert_or_assign(stored, keys, rows)
    want = hkv.layer_norm(rows, stats=False)
    torch.cuda.synchronize()
    failed, results = [], []

    def ask(seed):
        try:
            g = torch.Generator(device="cuda").manual_seed(seed)
            stream = torch.cuda.Stream()
            kept = []
            with torch.cuda.stream(stream):
                for turn in range(12):
                    n = 1 if turn == 3 else 500 * (turn + 1) * (seed % 3 + 1)
                    at = torch.randint(0, stored, (n,), generator=g, device="cuda")
                    out = torch.zeros((n, dim), device="cuda")
                    found = torch.zeros(n, dtype=torch.bool, device="cuda")
                    t.find_layer_norm(n, keys[at], out, found)
                    kept.append((at, out, found))
                stream.synchronize()
                results.extend(kept)
        except BaseException as e:      # noqa: BLE001 - reported by the main thread
            failed.append(e)

    threads = [threading.Thread(target=ask, args=(seed,)) for seed in range(6)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not failed, failed
    assert len(results) == 6 * 12
    for at, out, found in results:
        alone, again = torch.zeros_like(out), torch.zeros_like(found)
        t.find_layer_norm(at.numel(), keys[at], alone, again)
        assert found.all() and torch.equal(out, alone)
        assert (out - want[at]).abs().max() < 2.0 ** -12
    t.close()


# ---- layer norm of rows far from zero --------------------------------------------------

U = 2.0 ** -24


def rounded(value, dtype):
    """How far rounding `value` to dtype may move it."""
    f = torch.finfo(dtype)
    return value.abs() * (f.eps / 2) + f.smallest_normal * f.eps / 2


def check(got, want, bound, what=""):
    off = (got.double() - want).abs()
    bad = ~(off <= bound)     # a NaN is bad
    assert not bad.any(), (what, int(bad.sum()), float(off[bad].max()), float((off / bound.clamp(min=1e-300)).max()))


def check_centred(x, w, b, eps, y, mean, rstd):
    """Layer norm of rows whose mean is corrected by the mean of the distances from it.

    L u bounds the relative error of a sum of the row (its terms pass at most L additions)
    with the division; the first mean is off by first = (L + 3) u mean|x|.  A distance from
    it is at most |x - m| + first and rounded to u of that, so the correction, itself at
    most first, is off by second = (L + 4) u (mean|x - m| + first).  Behind it a distance
    is off by 2 u (|x - m| + first) + second: the size of x counts in second order only.
    The variance, of corrected distances: (L + 5) u (var + second^2) + second^2; rsqrtf
    adds 4 u, the products and the last sum 4 u."""
    x = x.double()
    m = x.mean(1, keepdim=True)
    d = x - m
    var = (d * d).mean(1, keepdim=True)
    want_rstd = (var + eps) ** -0.5
    terms = (max(64, x.shape[1] // 256) + 48 + 3) * U
    first = terms * x.abs().mean(1, keepdim=True)
    second = (terms + U) * (d.abs().mean(1, keepdim=True) + first)
    centred = 2 * U * (d.abs() + first) + second
    rel = ((terms + 2 * U) * (var + second ** 2) + second ** 2) / (var + eps) + 4 * U
    w, b = w.double(), b.double()
    want = d * want_rstd * w + b
    off = w.abs() * want_rstd * centred * (1 + rel) + (w * d * want_rstd).abs() * (rel + 4 * U) + 2 * U * want.abs()
    check(y, want, off + rounded(want, y.dtype), "y")
    check(mean, m[:, 0], (second + 2 * U * first)[:, 0] + U * m[:, 0].abs(), "mean")
    check(rstd, want_rstd[:, 0], ((rel + U) * want_rstd)[:, 0], "rstd")


@pytest.mark.parametrize("n,dim", [(3, 7), (5, 333), (4, 1000), (3, 5000), (2, 12001), (2, 50000), (9000, 333),
                                   (4000, 1000), (3000, 1001), (500, 5000), (200, 12001), (20000, 100), (100000, 12)])
@pytest.mark.parametrize("spread", [0.0, 1.0])
@pytest.mark.parametrize("far", [1.0e3, 3.0e4, -7.0e6])
def test_layer_norm_of_rows_far_from_zero(n, dim, spread, far):
    """No length here is a power of two, so 1 / dim is rounded: constant rows come out as
    the bias, and rows that vary by 1 about a large value lose no more than the type does."""
    g = torch.Generator(device="cuda").manual_seed(dim)
    x = far + spread * torch.randn((n, dim), generator=g, device="cuda")
    w, b = 1 + 0.2 * torch.randn(dim, generator=g, device="cuda"), torch.randn(dim, generator=g, device="cuda")
    y, mean, rstd = hkv.layer_norm(x, w, b)
    check_centred(x, w, b, 1e-5, y, mean, rstd)
    out = torch.zeros_like(x)
    ptrs = x.data_ptr() + torch.arange(n, device="cuda") * (dim * 4)
    hkv.layer_norm_ptr(n, ptrs, out, w, b, 1e-5, mean, rstd)
    check_centred(x, w, b, 1e-5, out, mean, rstd)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("n,dim", [(4, 1000), (4000, 1000), (20, 333), (9000, 333), (2, 40002)])
def test_layer_norm_of_short_types_far_from_zero(n, dim, dtype):
    g = torch.Generator(device="cuda").manual_seed(dim)
    x = (2.0e4 + 100 * torch.randn((n, dim), generator=g, device="cuda")).to(dtype)
    x[0] = 3.0e4
    w, b = 1 + 0.2 * torch.randn(dim, generator=g, device="cuda"), torch.randn(dim, generator=g, device="cuda")
    check_centred(x, w, b, 1e-5, *hkv.layer_norm(x, w, b))


def test_layer_norm_of_huge_rows_stays_finite():
    """Where a rounding error's square overflows, rstd is 0 and the bias is left."""
    for dim in (1000, 333, 20000):
        x = torch.full((2, dim), 1.0e31, device="cuda")
        x[1] = -3.0e33
        b = torch.randn(dim, device="cuda")
        assert torch.equal(hkv.layer_norm(x, None, b, stats=False), b.expand(2, dim))


# ---- expert sort of batches with large tiles ---------------------------------------------


def check_order(order, ids, experts):
    flat = ids.cpu().numpy().reshape(-1).astype(np.int64)
    kept = np.flatnonzero((flat >= 0) & (flat < experts))
    taken = kept[np.argsort(flat[kept], kind="stable")]
    position = np.full(flat.size, -1, np.int32)
    position[taken] = np.arange(taken.size)
    source = np.full(flat.size, -1, np.int32)
    source[:taken.size] = taken
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[kept], minlength=experts))])
    np.testing.assert_array_equal(order.offsets.cpu().numpy(), offsets)
    np.testing.assert_array_equal(order.position.cpu().numpy().reshape(-1), position)
    np.testing.assert_array_equal(order.source.cpu().numpy(), source)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64], ids=["i32", "i64"])
@pytest.mark.parametrize("tokens,top_k,experts", [((1 << 21) + 1, 1, 64), (625001, 8, 8), (1100000, 1, 1024),
                                                  (1100009, 2, 1), (1400001, 3, 512)])
def test_sort_of_sixteen_ids_per_lane(tokens, top_k, experts, dtype):
    """Above 512 tiles of four ids per lane a tile has sixteen: uneven experts, a tenth
    dropped, and one expert for all, which brings the counters to their largest sums."""
    g = torch.Generator(device="cuda").manual_seed(tokens)
    ids = (torch.rand((tokens, top_k), generator=g, device="cuda") ** 2 * experts * 1.06).long() - 1
    ids = ids.to(dtype)
    check_order(hkv.expert_sort(ids, experts), ids, experts)
    ids.fill_(experts - 1)
    check_order(hkv.expert_sort(ids, experts), ids, experts)


# ---- offsets past 32 bits --------------------------------------------------------------


def far_apart(rows, stride):
    """The same rows, `stride` elements apart, 4 GiB and more in all."""
    assert rows.shape[0] * stride * rows.element_size() > 2 ** 32
    wide = torch.empty(rows.shape[0] * stride, dtype=rows.dtype, device="cuda")
    out = wide.as_strided(rows.shape, (stride, 1))
    out.copy_(rows)
    return out


WIDE = [(600, 1001, torch.bfloat16, 8000001), (600, 1024, torch.bfloat16, 8000000), (600, 2050, torch.float16, 8000002),
        (800, 333, torch.float32, 2000001), (40, 1001, torch.bfloat16, 80000001), (6, 40000, torch.float32, 200000000)]
BY_WIDTH = pytest.mark.parametrize("n,dim,dtype,stride", WIDE, ids=[f"{n}x{d}" for n, d, _, _ in WIDE])


@BY_WIDTH
def test_layer_norm_past_32_bit_offsets(n, dim, dtype, stride):
    """Rows far apart give the bits of the same rows side by side (which the other tests
    hold to the formula): the units, and with them the sums' order, are the same."""
    g = torch.Generator(device="cuda").manual_seed(dim)
    x = torch.randn((n, dim), generator=g, device="cuda").to(dtype)
    dy = torch.randn((n, dim), generator=g, device="cuda").to(dtype)
    w, b = 1 + 0.2 * torch.randn(dim, generator=g, device="cuda"), torch.randn(dim, generator=g, device="cuda")
    want = hkv.layer_norm(x, w, b)
    wide_x, out = far_apart(x, stride), far_apart(torch.zeros_like(x), stride)
    got = hkv.layer_norm(wide_x, w, b, out=out)
    assert got[0] is out and all(torch.equal(p, q) for p, q in zip(got, want))
    ptrs = wide_x.data_ptr() + torch.arange(n, device="cuda") * (stride * x.element_size())
    near = x.data_ptr() + torch.arange(n, device="cuda") * (dim * x.element_size())
    out.zero_()
    assert torch.equal(hkv.layer_norm_ptr(n, ptrs, out, w, b), hkv.layer_norm_ptr(n, near, torch.zeros_like(x), w, b))
    want = hkv.layer_norm_backward(dy, x, w, *want[1:])
    got = hkv.layer_norm_backward(far_apart(dy, stride), wide_x, w, *got[1:], out=out)
    assert got[0] is out and all(torch.equal(p, q) for p, q in zip(got, want))


@BY_WIDTH
def test_experts_past_32_bit_offsets(n, dim, dtype, stride):
    top_k, experts = 2, 5
    tokens = n // top_k
    g = torch.Generator(device="cuda").manual_seed(dim)
    order = hkv.expert_sort(torch.randint(-1, experts, (tokens, top_k), generator=g, device="cuda"), experts)
    m = int(order.offsets[-1])
    y = torch.randn((n, dim), generator=g, device="cuda").to(dtype)
    x = torch.randn((tokens, dim), generator=g, device="cuda").to(dtype)
    wt = torch.randn((tokens, top_k), generator=g, device="cuda")
    wide_y, wide_x = far_apart(y, stride), far_apart(x, stride * top_k)
    rows, out = far_apart(torch.zeros_like(y), stride), far_apart(torch.zeros_like(x), stride * top_k)
    assert torch.equal(hkv.expert_dispatch(wide_x, order, out=rows)[:m], hkv.expert_dispatch(x, order)[:m])
    assert torch.equal(hkv.expert_combine(wide_y, wt, order, out=out), hkv.expert_combine(y, wt, order))
    assert torch.equal(hkv.expert_dispatch_backward(wide_y, order, out=out), hkv.expert_dispatch_backward(y, order))
    d_rows, d_wt = hkv.expert_combine_backward(wide_x, wide_y, wt, order, out=rows)
    want_rows, want_wt = hkv.expert_combine_backward(x, y, wt, order)
    assert torch.equal(d_rows[:m], want_rows[:m]) and torch.equal(d_wt, want_wt)


def test_experts_of_a_batch_above_four_gigabytes():
    """Every row without a gap: whole numbers, whose sums are exact in any order."""
    tokens, top_k, dim = 70000, 2, 16384
    g = torch.Generator(device="cuda").manual_seed(1)
    order = hkv.expert_sort(torch.randint(0, 4, (tokens, top_k), generator=g, device="cuda"), 4)
    t = torch.arange(tokens, device="cuda")
    x = ((t % 5)[:, None] + (torch.arange(dim, device="cuda") % 2)).to(torch.bfloat16)
    rows = hkv.expert_dispatch(x, order)
    assert rows.numel() * 2 > 2 ** 32
    token = order.source.long() // top_k
    assert all(torch.equal(rows[i:i + 20000], x[token[i:i + 20000]]) for i in range(0, tokens * top_k, 20000))
    wt = torch.tensor([0.5, 2.0], device="cuda").expand(tokens, top_k).contiguous()
    assert torch.equal(hkv.expert_combine(rows, wt, order), x * 2.5)
    d_rows, d_wt = hkv.expert_combine_backward(x, rows, wt, order)
    factor = wt.view(-1)[order.source.long()].to(torch.bfloat16)[:, None]
    for i in range(0, tokens * top_k, 20000):
        assert torch.equal(d_rows[i:i + 20000], x[token[i:i + 20000]] * factor[i:i + 20000])
    dots = dim // 2 * ((t % 5) ** 2 + (t % 5 + 1) ** 2)
    assert torch.equal(d_wt, dots.float()[:, None].expand(tokens, top_k))


def test_find_layer_norm_with_pinned_buffers():
    """What a kernel can reach it may use, as find may: pinned host memory."""
    dim, n = 16, 500
    t = make_table(dim)
    keys, rows = to_dev(unique_keys(n, seed=2)), torch.randn((n, dim), device="cuda")
    t.insert_or_assign(n, keys, rows)
    out, found = torch.zeros((n, dim)).pin_memory(), torch.zeros(n, dtype=torch.bool).pin_memory()
    w = (1 + torch.rand(dim)).pin_memory()
    t.find_layer_norm(n, keys.cpu().pin_memory(), out, found, w)
    torch.cuda.synchronize()
    assert found.all() and torch.equal(out, hkv.layer_norm(rows, w.cuda(), stats=False).cpu())
    with pytest.raises(ValueError, match="founds must be on the GPU"):
        t.find_layer_norm(n, keys, rows, torch.zeros(n, dtype=torch.bool))
    t.close()


def test_find_layer_norm_refuses_misaligned_buffers_before_the_lookup():
    """At the C entry (tensors start at a multiple of their element): nothing has run."""
    dim, n = 8, 100
    t = make_table(dim)
    keys, rows = to_dev(unique_keys(n, seed=2)), torch.randn((n, dim), device="cuda")
    t.insert_or_assign(n, keys, rows)
    out, found = torch.full((n, dim), 5.0, device="cuda"), torch.zeros(n, dtype=torch.bool, device="cuda")
    spare = torch.full((n,), 5.0, device="cuda")
    fine = dict(keys=keys.data_ptr(), weight=spare.data_ptr(), bias=spare.data_ptr(), values=out.data_ptr(),
                mean=spare.data_ptr(), rstd=spare.data_ptr())
    stream = torch.cuda.current_stream().cuda_stream
    for name in fine:
        p = {**fine, name: fine[name] + (4 if name == "keys" else 2)}
        rc = t._lib.hkv_find_layer_norm(t._h, n, p["keys"], p["weight"], p["bias"], 1, 1e-5, p["values"],
                                        found.data_ptr(), p["mean"], p["rstd"], stream)
        assert rc == 4 and b"element size" in t._lib.hkv_last_error(), name
    torch.cuda.synchronize()
    assert not found.any() and (out == 5).all() and (spare == 5).all()
    t.close()


# ---- sums over many rows ---------------------------------------------------------------


def test_column_sums_of_many_long_rows():
    """One row of x and dy for 262,144 rows: every column adds a constant, whose rounding
    errors do not cancel.  A term passes 64 additions of a run, 64 runs, and 6 + 5 in the
    kernel that adds the 64 row splits; each product adds 3 roundings."""
    n, dim = 1 << 18, 8196
    g = torch.Generator(device="cuda").manual_seed(1)
    x, dy = torch.randn((1, dim), generator=g, device="cuda"), torch.randn((1, dim), generator=g, device="cuda")
    dy[0, :100] = 0.1
    _, mean, rstd = hkv.layer_norm(x)
    out = torch.empty((n, dim), device="cuda")
    _, dw, db = hkv.layer_norm_backward(dy.expand(n, dim), x.expand(n, dim), torch.ones(dim, device="cuda"),
                                        mean.expand(n).contiguous(), rstd.expand(n).contiguous(), out=out)
    xhat = (x[0].double() - mean.double()) * rstd.double()
    want_w, want_b = n * dy[0].double() * xhat, n * dy[0].double()
    chain = (64 + 64 + 11) * U
    check(dw, want_w, (chain + 3 * U) * want_w.abs() + rounded(want_w, dw.dtype), "d_weight")
    check(db, want_b, chain * want_b.abs() + rounded(want_b, db.dtype), "d_bias")


# ---- calls that no other test makes ------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("n,dim", [(6, 64), (5000, 64), (700, 333), (4, 20000)])
def test_one_row_for_all(n, dim, dtype):
    """Inputs whose rows are one row (a distance of zero) give the bits of their copies."""
    g = torch.Generator(device="cuda").manual_seed(dim)
    x = torch.randn((1, dim), generator=g, device="cuda").to(dtype).expand(n, dim)
    w = 1 + 0.2 * torch.randn(dim, generator=g, device="cuda")
    want = hkv.layer_norm(x.contiguous(), w, w)
    got = hkv.layer_norm(x, w, w)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    want = hkv.layer_norm_backward(x.contiguous(), x.contiguous(), w, *want[1:])
    got = hkv.layer_norm_backward(x, x, w, *got[1:])
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    tokens, experts = n // 2, 3
    order = hkv.expert_sort(torch.randint(-1, experts, (tokens, 2), generator=g, device="cuda"), experts)
    m = int(order.offsets[-1])
    one, wt = x[:tokens], torch.randn((tokens, 2), generator=g, device="cuda")
    assert torch.equal(hkv.expert_dispatch(one, order)[:m], one[:1].expand(m, dim))
    y = x[:1].expand(tokens * 2, dim)
    assert torch.equal(hkv.expert_combine(y, wt, order), hkv.expert_combine(y.contiguous(), wt, order))
    got = hkv.expert_combine_backward(one, y, wt, order)
    want = hkv.expert_combine_backward(one.contiguous(), y.contiguous(), wt, order)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("n", [300, 20000])
def test_layer_norm_by_address_captured_and_replayed(n):
    """The addresses are read when the graph runs: rows may move between replays, become
    misses and come back."""
    dim = 48
    g = torch.Generator(device="cuda").manual_seed(n)
    table = torch.randn((2 * n, dim), generator=g, device="cuda")
    want, mean, rstd = hkv.layer_norm(table)
    ptrs, out = torch.zeros(n, dtype=torch.int64, device="cuda"), torch.zeros((n, dim), device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        hkv.layer_norm_ptr(n, ptrs, out)
    for turn in range(3):
        at = torch.randint(0, 2 * n, (n,), generator=g, device="cuda")
        miss = torch.rand(n, generator=g, device="cuda") < 0.3
        ptrs.copy_(torch.where(miss, 0, table.data_ptr() + at * (dim * 4)))
        out.fill_(5)
        graph.replay()
        torch.cuda.synchronize()
        eager = hkv.layer_norm_ptr(n, ptrs, torch.full_like(out, 5))
        assert torch.equal(out, eager) and (out[miss] == 5).all()
        assert (out[~miss] - want[at[~miss]]).abs().max() < 2.0 ** -12
