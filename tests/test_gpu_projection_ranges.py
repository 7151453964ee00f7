"""Norm and projections at the ends of what their arguments may be, on the GPU against float64."""
from __future__ import annotations

import numpy as np
import pytest

import _serving as sv
from moe_mi355x import _lib
from moe_mi355x import projection as pj
from test_gpu_projection import SHAPES, Case, check_norm, norm64, run_norm, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [4, 40, 90, 300])
def test_scales_at_both_ends_of_fp32(mi355x, stream, rows):
    """Scales whose product leaves the range of fp32 where the result does not.  The sum's conversion and two products
    are a rounding each, the last one of half a subnormal step where the result is subnormal."""
    say(f"scales at the ends, {rows} rows")
    k, n = 2048, 42
    c = Case(7, rows, k, [n], np.float32)
    c.qs = np.resize(np.array([2.0 ** -126, 1.37 * 2.0 ** -110, 0.02, 1.21 * 2.0 ** 115], np.float32), rows)
    c.ws = [np.resize(np.array([2.0 ** -24, 1.5 * 2.0 ** -14, 0.75, 65504.0], np.float16), n)]
    c.w[0][5] = 0
    c.w[0][7] = 0  # under a scale of 65504
    got = c.run(mi355x, stream)[0].astype(np.float64)
    sums = c.q.astype(np.float64) @ c.w[0].astype(np.float64).T
    want = sums * (c.qs[:, None].astype(np.float64) * c.ws[0].astype(np.float64))
    huge = np.abs(want) > 2.0 ** 128
    assert np.array_equal(got[huge], np.sign(want[huge]) * np.inf)
    small = ~huge
    err = np.abs(got[small] - want[small])
    assert np.all(err <= 3.01 * 2.0 ** -24 * np.abs(want[small]) + 2.0 ** -150)
    assert np.all(got[:, [5, 7]] == 0)


@pytest.mark.parametrize("rows,hidden", [(3, 200), (5, 2048), (300, 2051), (300, 5120)])
def test_a_row_of_zeros_stays_one_without_eps(mi355x, stream, rows, hidden):
    """eps 0 divides a row of zeros by its own norm: it is zeros, with a scale of 1, as with any other eps; the rows
    beside it are the definition's."""
    say(f"zeros without eps, {rows} x {hidden}")
    rng = np.random.default_rng(3)
    x = rng.standard_normal((rows, hidden)).astype(np.float32)
    res = rng.standard_normal((rows, hidden)).astype(np.float32)
    w = (1 + 0.3 * rng.standard_normal(hidden)).astype(np.float32)
    x[1], x[2] = 0, -res[2]
    res[1] = 0
    q, s, h, total = got = run_norm(mi355x, stream, x, res, w, eps=0.0)
    for r in (1, 2):
        assert s[r] == 1 and not q[r].any() and not h[r].any() and not total[r].any()
    others = np.delete(np.arange(rows), [1, 2])
    v, y = norm64(x[others], res[others], w, True, 0.0)
    check_norm(y, v, tuple(a[others] for a in got), np.float32)


def test_an_infinite_eps_leaves_rows_of_zeros(mi355x, stream):
    say("infinite eps")
    x = np.random.default_rng(3).standard_normal((4, 256)).astype(np.float32)
    q, s, h, total = run_norm(mi355x, stream, x, None, None, eps=np.inf)
    assert np.all(s == 1) and not q.any() and not h.any() and np.array_equal(total, x)


def test_norm_of_more_rows_than_a_launch_holds(mi355x, stream):
    """Wide rows whose threads are more than 2^32 (103 GB): the first and last rows of every launch."""
    rows, hidden = (1 << 22) + 3, 8196
    say(f"norm {rows} x {hidden}")
    look = sorted({0, 1, rows - 1, *(r + d for r in (1 << 21, 1 << 22) for d in (-1, 0))})
    x = np.random.default_rng(5).standard_normal((len(look), hidden)).astype(np.float16)
    w = (1 + 0.3 * np.random.default_rng(6).standard_normal(hidden)).astype(np.float32)
    with sv.Arrays(mi355x, stream) as ar:
        ar.held += [mi355x.alloc_device(rows * n) for n in (2 * hidden, hidden, 4)]
        px, pq, ps = (int(b.handle) for b in ar.held)
        for i, r in enumerate(look):
            mi355x.copy_h2d_ptr_async(px + 2 * hidden * r, x[i].ctypes.data, x[i].nbytes, stream)
        mi355x.synchronize_stream(stream)
        pj.add_rmsnorm_i8(pj.norm_args(px, rows=rows, hidden=hidden, q=pq, q_scale=ps, norm_w=ar.put(w), dtype="float16"),
                          stream)
        q = np.stack([ar.get(pq + hidden * r, np.zeros(hidden, np.int8)) for r in look])
        s = np.concatenate([ar.get(ps + 4 * r, np.zeros(1, np.float32)) for r in look])
    v, y = norm64(x, None, w, True, 1e-6)
    check_norm(y, v, (q, s, None, None), np.float16)


def test_adapters_of_more_columns_than_a_launch_holds(mi355x, stream):
    """Four segments of the most columns there may be, 125 GB in all: 128 x 64 tiles, which as many adapters take
    otherwise, would be 2^32 threads.  Whole numbers; the first and last columns of every segment."""
    rows, k, n, rank, n_ad, edge = 897, 16, (1 << 24) - 1, 8, 17, 70
    say(f"adapters alone, {rows} rows onto 4 x {n}")
    rng = np.random.default_rng(8)
    x = rng.integers(-2, 3, (rows, k)).astype(np.float16)
    a = rng.integers(-2, 3, (n_ad, rank, k)).astype(np.float16)
    ids = np.full(rows, 3, np.int32)
    ids[[5, 896]], ids[7] = 16, -1
    edges = {c: rng.integers(-2, 3, (n_ad, edge, rank)).astype(np.float16) for c in (0, n - edge)}
    with sv.Arrays(mi355x, stream) as ar:
        ar.held += [mi355x.alloc_device(size) for size in [2 * n_ad * n * rank] + [2 * rows * n] * 4]
        pb, *py = (int(b.handle) for b in ar.held)
        for c, b in edges.items():
            for i in (3, 16):
                mi355x.copy_h2d_ptr_async(pb + 2 * rank * (i * n + c), b[i].ctypes.data, b[i].nbytes, stream)
        mi355x.synchronize_stream(stream)
        pa = ar.put(a)
        args = pj.projection_args([pj.segment(y, n, a=pa, b=pb) for y in py], rows=rows, k=k)
        ad = pj.adapter_args(ar.put(x), ar.put(np.arange(rows + 1, dtype=np.int32)), ar.put(ids),
                             ar.put(np.ones(n_ad, np.float32)), n_seqs=rows, n_adapters=n_ad, rank=rank, k=k)
        need = pj.workspace_bytes(args, ad)
        pj.project(args, stream, adapters=ad, workspace=(ar.put(np.zeros(need, np.uint8)), need))
        for r in (0, 5, 7, 127, 128, 640, 895, 896):
            t = x[r].astype(np.float64) @ a[ids[r]].astype(np.float64).T if ids[r] >= 0 else np.zeros(rank)
            for c, b in edges.items():
                want = t @ b[ids[r]].astype(np.float64).T
                for y in py:
                    assert np.array_equal(ar.get(y + 2 * (r * n + c), np.zeros(edge, np.float16)), want)


@pytest.mark.parametrize("rank", [8, 40, 72, 128])
@pytest.mark.parametrize("rows,each", [(20, 9), (90, 40), (200, 1), (700, 300)])
def test_an_infinity_in_a_row_reaches_its_outputs_as_one(mi355x, stream, rows, each, rank):
    """Adapters of positive weights, so that the definition's output is that infinity and no NaN, with ranks that fill
    no whole tile; the other rows do not see it."""
    say(f"infinite rows, {rows} rows, rank {rank}")
    lens = [each] * (rows // each)
    c = Case(6, rows, 272, [70], np.float32, lens=lens, ids=[i % 5 for i in range(len(lens))], rank=rank, n_adapters=5,
             base=False, res=True)
    c.a[0] = np.abs(c.a[0]) + np.float16(0.01)
    c.b[0] = np.abs(c.b[0]) + np.float16(0.01)
    clean = c.run(mi355x, stream)[0]
    c.x[3, 7], c.x[6, 271] = np.inf, -np.inf
    got = c.run(mi355x, stream)[0]
    assert np.all(got[3] == np.inf) and np.all(got[6] == -np.inf)
    others = np.delete(np.arange(rows), [3, 6])
    assert np.all(np.isfinite(clean)) and np.array_equal(got[others], clean[others])


@pytest.mark.parametrize("rows,each", [(60, 30), (90, 45), (200, 1), (700, 300)])
@pytest.mark.parametrize("rank", [16, 48])
def test_small_ranks_beside_loud_ones_keep_their_digits(mi355x, stream, rows, each, rank):
    """Every other rank 2^-24 of its neighbour, and columns that only the small ranks reach.  t is exact in fp32 (whole
    numbers below 2^24 times a power of two) and held to 2^-23 of itself; its products are summed in fp32, a rounding
    or a truncation for each."""
    say(f"small ranks, {rows} rows, rank {rank}")
    k, n, n_ad = 64, 70, 3
    lens = [each] * (rows // each)
    c = Case(5, rows, k, [n], np.float32, lens=lens, ids=[i % n_ad for i in range(len(lens))], rank=rank, n_adapters=n_ad,
             base=False, res=True)
    rng = np.random.default_rng(11)
    c.x = rng.integers(-1023, 1024, (rows, k)).astype(np.float16)
    few = (rng.integers(0, 8, (n_ad, rank, k)) == 0) * rng.integers(-255, 256, (n_ad, rank, k))
    few[:, 1::2] *= 2
    c.a[0] = (few * np.where(np.arange(rank) % 2, 2.0 ** -24, 1.0)[:, None]).astype(np.float16)
    assert np.array_equal(c.a[0][:, 1::2].astype(np.float64) * 2.0 ** 24, few[:, 1::2])  # subnormal, exact
    c.b[0][:, 1::2, 0::2] = 0
    c.res[0][:] = 0
    c.alpha[:] = 1
    got = c.run(mi355x, stream)[0].astype(np.float64)
    for a, r in c.adapter_rows():
        t = c.x[r].astype(np.float64) @ c.a[0][a].astype(np.float64).T
        assert np.abs(t[:, 0::2]).max() < 2 ** 24 and np.abs(t[:, 1::2]).max() < 1
        for cols in (slice(0, None, 2), slice(1, None, 2)):
            b = c.b[0][a, cols].astype(np.float64)
            size = np.abs(t) @ np.abs(b).T
            assert np.all(np.abs(got[r, cols] - t @ b.T) <= (1 + rank + 4) * 2.0 ** -23 * size)


def long_ring_case(rows, ns, **kw):
    """Nine stages of the reduction, the last in part: every ring of slots comes round, and ends inside a stage.  Whole
    numbers: 1104 products of 100 x 100 at most, times 1/8, and what the adapters add, stay below 2^24 steps of 1/8."""
    c = Case(rows, rows, 1104, ns, np.float32, whole=True, **kw)
    rng = np.random.default_rng(rows + 1)
    c.q = rng.integers(-100, 101, c.q.shape).astype(np.int8)
    c.w = [rng.integers(-100, 101, w.shape).astype(np.int8) for w in c.w]
    return c


@pytest.mark.parametrize("rows,ns", SHAPES)
def test_every_tile_over_many_stages(mi355x, stream, rows, ns):
    say(f"many stages, {rows} rows -> {ns}")
    c = long_ring_case(rows, ns)
    for i, o in enumerate(c.run(mi355x, stream)):
        assert np.array_equal(o, c.want(i)[0])


@pytest.mark.parametrize("rows,ns", SHAPES)
@pytest.mark.parametrize("rank,n_adapters,each", [(8, 33, 1), (72, 3, 70)])
def test_every_adapted_tile_over_many_stages(mi355x, stream, rows, ns, rank, n_adapters, each):
    say(f"many stages, adapted, {rows} rows -> {ns} rank={rank}")
    rng = np.random.default_rng(rows * rank)
    lens = []
    while sum(lens) < rows - 3:
        lens.append(min(int(rng.integers(0, 2 * each + 1)), rows - 3 - sum(lens)))
    c = long_ring_case(rows, ns, lens=lens, ids=rng.integers(-1, n_adapters, len(lens)).tolist(), rank=rank,
                       n_adapters=n_adapters)
    for i, o in enumerate(c.run(mi355x, stream)):
        assert np.array_equal(o, c.want(i)[0])


@pytest.mark.parametrize("rows", [2, 13, 40, 64, 70, 130])
def test_sums_past_24_bits_that_cancel(mi355x, stream, rows):
    """The longest reduction in runs of +127 x 127 and -127 x 127, inside a quarter of it and across, with small codes in
    between: partial sums reach 2^29, the sums stay below 2^24.  fp32 sums of 64 products each miss them."""
    say(f"cancelling sums, {rows} rows")
    k, n = 65536, 20
    c = Case(9, rows, k, [n], np.float32)
    rng = np.random.default_rng(9)
    sign = rng.choice([-127, 127], (1, k))
    c.w[0] = np.where(rng.random((n, k)) < 0.002, rng.integers(-127, 128, (n, k)), sign).astype(np.int8)
    runs = np.stack([np.where(np.arange(k) // run % 2, -1, 1) for run in (32768, 8192, 2048, 16384)])
    c.q = np.where(rng.random((rows, k)) < 0.002, rng.integers(-127, 128, (rows, k)),
                   runs[np.arange(rows) % 4] * sign).astype(np.int8)
    c.qs[:], c.ws = 1, [np.ones(n, np.float16)]
    part = np.einsum("rsk,nsk->srn", c.q.reshape(rows, -1, 64).astype(np.float64), c.w[0].reshape(n, -1, 64).astype(np.float64),
                     optimize=True)
    want = part.sum(0)  # whole numbers, exact
    near = np.zeros((rows, n), np.float32)
    for p in part.astype(np.float32):
        near += p
    assert np.abs(want).max() < 2 ** 24 and np.abs(part.cumsum(0)).max() > 2 ** 28
    assert np.mean(near != want) > 0.4  # (the runs of 2048 stay below 2^25)
    assert np.array_equal(c.run(mi355x, stream)[0], want)


@pytest.mark.parametrize("rows", [3, 90])
def test_the_largest_sum(mi355x, stream, rows):
    """-128 x -128 over the longest reduction: 2^30, within int32."""
    say(f"largest sum, {rows} rows")
    c = Case(9, rows, 65536, [20], np.float32)
    c.q[:], c.w[0][:] = -128, -128
    c.qs[:], c.ws = 1, [np.ones(20, np.float16)]
    assert np.all(c.run(mi355x, stream)[0] == 2.0 ** 30)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_more_weight_rows_than_a_launch_holds(mi355x, stream, dtype):
    say(f"weights of 2^24 + 5 rows, {dtype.__name__}")
    rows, cols = (1 << 24) + 5, 4
    w = np.random.default_rng(2).standard_normal((rows, cols), dtype=np.float32).astype(dtype)
    q, s = np.full((rows, cols), 99, np.int8), np.zeros(rows, np.float16)
    with sv.Arrays(mi355x, stream) as ar:
        pq, ps = ar.put(q), ar.put(s)
        _lib.check(_lib.load().mx_quantize_rows_i8(ar.put(w), _lib.MX_DT_F16 if dtype is np.float16 else _lib.MX_DT_F32,
                                                   rows, cols, pq, ps, stream), "mx_quantize_rows_i8")
        q, s = ar.get(pq, q), ar.get(ps, s)
    w = w.astype(np.float32)
    assert np.array_equal(s, (np.abs(w).max(1) / np.float32(127)).astype(np.float16))
    assert np.array_equal(q, np.clip(np.rint(w / s[:, None].astype(np.float32)), -127, 127))
