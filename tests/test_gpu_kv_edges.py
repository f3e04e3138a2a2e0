"""Paged attention at its edges: scores of minus infinity, scores that overflow, unused places of a cache
that hold anything, first launches inside a recorded step. Comparisons ask first that their tolerances are numbers: an infinite or undefined
one would accept any result."""
import os
import subprocess
import sys

import numpy as np
import pytest

import kvutil as K
from tuckmill_amd import hip as H

from q8util import require_gpu, upload_new
from test_gpu_kv import f32, prefill_case, run_decode, run_prefill, want_decode, want_prefill
from test_gpu_kv_many import many

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def ctx():
    c = require_gpu()
    yield c
    c.close()


def near(got, want, tol, what=""):
    assert np.isfinite(np.broadcast_to(tol, np.shape(want))[np.isfinite(want)]).all(), f"{what}: tolerances"
    K.near(got, want, tol, what)


def test_a_tolerance_that_is_no_number_is_refused():
    with pytest.raises(AssertionError, match="tolerances"):
        near(np.array([1e9]), np.array([0.5]), np.array([np.nan]))


# ---- a score of minus infinity takes its own position out, and no other ---------------------------

@pytest.mark.parametrize("type_id", [K.F16, K.F32])
@pytest.mark.parametrize("d", [64, 128, 256, 72])
def test_decode_one_infinite_score_takes_its_position_out(ctx, type_id, d):
    """A key with a channel of -infinity under positive queries: the softmax gives it a weight of
    exactly zero, so what is left is the attention over the other positions."""
    rng = np.random.default_rng(50 + d)
    lens, heads = [100, 33, 1, 700], 3
    out_of = [50, 0, 0, 699]
    paged = K.Paged(rng, type_id, 32, 1, d, lens)
    seen = [np.ones(n, bool) for n in lens]
    for s, j in enumerate(out_of):
        paged.keys[s][j, 0, 3] = -np.inf
        paged.put(s, j)
        seen[s][j] = False
    q = np.abs(rng.standard_normal((len(lens), heads * d))).astype(np.float32) + np.float32(0.1)
    got = run_decode(ctx, paged, q, heads, H.Attention(0.125))
    clean = K.Paged(rng, type_id, 32, 1, d, lens)
    clean.keys = [np.where(np.isinf(k), 0, k) for k in paged.keys]  # (where it is not looked at)
    clean.values = paged.values
    want, tol = want_decode(clean, q, heads, 0.125, seen=seen)
    near(got, want, tol)
    assert not got[2].any()  # the only position it had


@pytest.mark.parametrize("type_id,heads,d,news,lens", [
    (K.F16, 3, 64, [5, 2], [100, 40]), (K.F16, 2, 256, [20, 1], [100, 40]), (K.F32, 3, 64, [5, 2], [100, 40]),
    (K.F32, 2, 256, [20, 1], [100, 40]), (K.F16, 64, 64, [130, 6], [150, 40]), (K.F16, 64, 128, [130, 6], [150, 40]),
    (K.F16, 64, 256, [130, 6], [150, 40]), (K.F16, 64, 72, [130, 6], [150, 40]), (K.F16, 40, 64, [300, 40], [3000, 1100]),
    (K.F16, 16, 128, [600, 40], [1500, 1100])])
@pytest.mark.parametrize("cap,slopes", [(0.0, False), (5.0, False), (0.0, True)])
def test_rows_of_one_infinite_score_are_the_same_however_many_there_are(ctx, type_id, heads, d, news, lens, cap, slopes):
    """As above for ragged rows, few (as the kernel of single tokens takes them) and many (in tiles, and
    over positions shared between workgroups): which kernel runs does not show. Under a cap such a score is
    minus the cap."""
    rng = np.random.default_rng(55)
    out_of = [n - 30 for n in lens]
    paged = K.Paged(rng, type_id, 32, heads, d, lens)
    clean = K.Paged(rng, type_id, 32, heads, d, lens)
    clean.values, clean.keys = paged.values, [k.copy() for k in paged.keys]
    seen = [np.ones(n, bool) for n in lens]
    for s, j in enumerate(out_of):
        for p, low in ((paged, -np.inf), (clean, -6e4)):
            p.keys[s][j, :, 3] = low
            p.put(s, j)
        seen[s][j] = cap > 0  # (-6e4 is as far below the cap)
    starts, _, _ = prefill_case(rng, news, lens)
    q = np.abs(rng.standard_normal((sum(news), heads * d))).astype(np.float32) + np.float32(0.1)
    sl = (2.0 ** -(1 + np.arange(heads) / 8)).astype(np.float32) if slopes else None
    attn = H.Attention(0.125, cap, slopes=upload_new(ctx, sl) if slopes else None)
    got = run_prefill(ctx, paged, q, heads, attn, starts)
    want, tol = want_prefill(clean, q, heads, starts, news, 0.125, softcap=cap, slopes=sl, seen=seen)
    near(got, want, tol)


@pytest.mark.parametrize("every", [64, 700])
def test_rows_of_many_infinite_scores_beside_rows_that_are_nan(ctx, every):
    """Few and many positions to take out (and those of them in the first pages and the last), a query that
    is NaN, one that is infinite, and a key that is NaN to the rows that see it."""
    rng = np.random.default_rng(56)
    heads, d, rows, n = 64, 64, 600, 3000
    assert many(rows, 1, heads, heads)
    paged = K.Paged(rng, K.F16, 32, heads, d, [n])
    clean = K.Paged(rng, K.F16, 32, heads, d, [n])
    seen = np.ones(n, bool)
    seen[5::every] = False
    seen[n - rows + 20] = False  # a position that only some rows see
    clean.keys = [paged.keys[0].copy()]
    clean.values = paged.values
    paged.keys[0][~seen, :, 3] = -np.inf
    paged.keys[0][n - 40, :, 7] = np.nan
    for j in range(n):
        paged.put(0, j)
    q = np.abs(rng.standard_normal((rows, heads * d))).astype(np.float32) + np.float32(0.1)
    q[33] = np.nan
    q[77, 3::d] = np.inf
    got = run_prefill(ctx, paged, q, heads, H.Attention(0.125), np.array([0, rows]))
    p = np.arange(n - rows, n)
    fine = (p < n - 40) & ~np.isin(np.arange(rows), [33, 77])
    lo, hi = K.bounds(p, n)
    for r0 in range(0, rows, 37):  # (some of the rows: the reference is slow)
        r = np.array([r0, min(r0 + 1, rows - 1)])
        want, tol = K.attention(q[r].reshape(len(r), heads, d), clean.keys[0], clean.values[0], p[r], lo[r], hi[r], 0.125, seen=seen)
        near(got[r][fine[r]], want[fine[r]], tol[fine[r]], f"row {r0}")
    assert np.isnan(got[33]).all() and np.isnan(got[77]).all() and np.isnan(got[p >= n - 40]).all()
    assert not np.isnan(got[fine]).any()


@pytest.mark.parametrize("d,window,prefix,docs", [(64, 0, 0, 1), (128, 100, 0, 0), (64, 40, 1, 0), (256, 0, 1, 1)])
def test_infinite_scores_under_masks_with_shared_heads(ctx, d, window, prefix, docs):
    """Four query heads to a key-value head, odd strides, biases and every mask: what is taken out is what
    each row sees of it."""
    rng = np.random.default_rng(57)
    heads, kv_heads, news, lens = 32, 8, [270, 33], [500, 60]
    assert many(sum(news), 2, heads, kv_heads)
    paged = K.Paged(rng, K.F16, 16, kv_heads, d, lens)
    clean = K.Paged(rng, K.F16, 16, kv_heads, d, lens)
    clean.keys, clean.values = [k.copy() for k in paged.keys], paged.values
    seen = [rng.random(n) > 0.03 for n in lens]
    for s, n in enumerate(lens):
        paged.keys[s][~seen[s], :, 3] = -np.inf
        for j in range(n):
            paged.put(s, j)
    starts, first, pre = prefill_case(rng, news, lens, docs, prefix)
    w = heads * d
    q = np.abs(rng.standard_normal((sum(news), w))).astype(np.float32) + np.float32(0.1)
    flat = np.full((sum(news), w + 3), np.nan, np.float32)
    flat[:, :w] = q
    sl = (2.0 ** -(1 + np.arange(heads) / 8)).astype(np.float32)
    attn = H.Attention(0.125, 0.0, window, slopes=upload_new(ctx, sl), first=upload_new(ctx, K.u32(first)) if docs else None,
                       prefix=upload_new(ctx, K.u32(pre)) if prefix else None)
    out = upload_new(ctx, np.full((sum(news), w + 1), 7.0, np.float32))
    ctx.attn_prefill(attn, paged.upload(ctx), upload_new(ctx, flat), upload_new(ctx, paged.table), upload_new(ctx, K.u32(lens)),
                     upload_new(ctx, K.u32(starts)), out, sum(news), 2, heads, paged.stride, 0, 0, w + 3, w + 1)
    ctx.fence()
    got = f32(out, (sum(news), w + 1))
    want, tol = want_prefill(clean, q, heads, starts, news, 0.125, first, window, 0.0, sl, pre, seen)
    near(got[:, :w].reshape(want.shape), want, tol)
    assert (got[:, w:] == 7.0).all()


# ---- huge queries --------------------------------------------------------------------------------

def check_decided(got, scores, error, values, margin):
    """got [channel] where the largest of `scores` (each off by at most `error`) decides alone: the
    value at that position if no other's score comes within the two errors and `margin`, else
    something between the values."""
    order = np.argsort(scores)
    top, second = order[-1], order[-2]
    if scores[top] - scores[second] > error[top] + error[second] + margin:
        # (one weight, in two parts of 22 bits, and nothing beside it: half steps 2 for the parts, 1 for the
        # products, 2 for the sum of weights, 2 for the join, 1 for the division)
        assert np.abs(got - values[top]).max() <= 8 * K.EPS * np.abs(values[top]).max()
        return 1
    assert (got >= values.min(0) - 1e-5).all() and (got <= values.max(0) + 1e-5).all()
    return 0


@pytest.mark.parametrize("type_id,heads,rows", [(K.F16, 2, 1), (K.F32, 2, 1), (K.F16, 2, 6), (K.F32, 2, 6), (K.F16, 64, 140)])
@pytest.mark.parametrize("size", [1e10, 1e30])
def test_huge_queries_take_the_value_of_the_largest_score(ctx, type_id, heads, rows, size):
    rng = np.random.default_rng(60)
    d, n = 64, 300
    paged = K.Paged(rng, type_id, 16, heads, d, [n])
    q = (rng.standard_normal((rows, heads * d)) * size).astype(np.float32)
    attn = H.Attention(d ** -0.5)
    if rows == 1:
        got = run_decode(ctx, paged, q, heads, attn)
    else:
        assert many(rows, 1, heads, heads) == (rows > 100)
        got = run_prefill(ctx, paged, q, heads, attn, np.array([0, rows]))
    decided = 0
    for r in range(rows):
        upto = n - rows + r + 1
        for h in range(heads):
            k = paged.keys[0][:upto, h].astype(np.float64)
            qh = q[r].reshape(heads, d)[h].astype(np.float64)
            x = d ** -0.5 * (k @ qh)
            # f32 sums of d products, and q in 22 bits of its largest magnitude
            e = d ** -0.5 * (np.abs(k) @ np.abs(qh) * K.SIGMAS * np.sqrt(d) * K.EPS +
                             np.abs(k).sum(1) * np.abs(qh).max() * 2.0 ** -22) + 8 * K.EPS * np.abs(x)
            decided += check_decided(got[r, h], x, e, paged.values[0][:upto, h].astype(np.float64), 200.0)
    assert decided >= 0.9 * rows * heads  # (the check is not an empty one)


@pytest.mark.parametrize("rows,heads", [(1, 2), (6, 2), (200, 64)])
def test_rows_whose_scores_all_overflow_are_zero_whatever_they_see(ctx, rows, heads):
    """Scores below the range of f32 are -infinity, and where all of a row's are its result is zero,
    though a value that it sees is NaN; among positions shared between workgroups too."""
    rng = np.random.default_rng(61)
    d, n = 64, 3000
    paged = K.Paged(rng, K.F16, 64, heads, d, [n])
    paged.keys[0][:] = -np.abs(paged.keys[0]) - 1
    paged.values[0][10, :, 3] = np.nan
    paged.values[0][1500, :, 5] = np.inf
    for j in range(n):
        paged.put(0, j)
    assert many(rows, 1, heads, heads) == (rows == 200)
    q = np.full((rows, heads * d), 3e37, np.float32)  # (64 products of -3e37 and less, times 0.5)
    attn = H.Attention(0.5)
    got = run_decode(ctx, paged, q, heads, attn) if rows == 1 else run_prefill(ctx, paged, q, heads, attn, np.array([0, rows]))
    assert not np.isnan(got).any() and not got.any()


# ---- unused places of the cache --------------------------------------------------------------------

def test_what_lies_behind_a_sequence_costs_nothing(ctx):
    """Places of a last page that no position has yet hold anything: NaN there, or zeros, and the call
    takes as long (half as long again is allowed, a shortest of twelve calls each, in turns)."""
    rng = np.random.default_rng(70)
    heads, kv_heads, d, news, lens = 32, 8, 128, [1300, 700], [4001, 2009]
    assert many(sum(news), 2, heads, kv_heads)
    calls = []
    q = rng.standard_normal((sum(news), heads * d)).astype(np.float32)
    paged = K.Paged(rng, K.F16, 64, kv_heads, d, lens)
    shared = [upload_new(ctx, x) for x in (q, paged.table, K.u32(lens), K.u32([0, news[0], sum(news)]))]
    out = ctx.buffer(q.nbytes)
    for fill in (np.nan, 0.0):
        for pages in (paged.k, paged.v):
            pages[np.isnan(pages)] = 0.0
        if np.isnan(fill):
            for s, n in enumerate(lens):
                page, place = paged.table[s, n // 64], n % 64
                paged.k[page, :, place:] = fill
                paged.v[page, :, :, place:] = fill
        calls.append(paged.upload(ctx))
        if np.isnan(fill):
            for pages in (paged.k, paged.v):
                pages[np.isnan(pages)] = 0.0
    times, got = [[], []], [None, None]
    for _ in range(12):
        for i, cache in enumerate(calls):
            ctx.attn_prefill(H.Attention(d ** -0.5), cache, *shared, out, sum(news), 2, heads, paged.stride)
            ctx.fence()
            times[i].append(ctx.last_gpu_ms())
            got[i] = f32(out, (sum(news), heads * d)).view(np.uint32)
    assert np.array_equal(got[0], got[1])
    assert min(times[0]) <= 1.5 * min(times[1]), (min(times[0]), min(times[1]))


# ---- recorded steps -------------------------------------------------------------------------------

def test_first_launches_inside_a_recorded_step():
    """In a process of its own, so that nothing has launched these kernels before: the forms whose LDS has
    to be allowed first, recorded, replayed, and run again without a recording."""
    code = """
import sys
sys.path.insert(0, "tests")
import numpy as np
import kvutil as K
from tuckmill_amd import hip as H
from q8util import upload_new
from test_gpu_kv import f32, want_decode, want_prefill
ctx = H.HipContext.open()
rng = np.random.default_rng(80)
for type_id, heads, kv_heads, d, lens in ((K.F16, 16, 8, 128, [700, 65]), (K.F32, 4, 2, 128, [300, 9]), (K.F16, 4, 1, 256, [500, 40]),
                                          (K.F32, 4, 1, 256, [200, 31])):
    paged = K.Paged(rng, type_id, 64, kv_heads, d, lens)
    q = rng.standard_normal((2, heads * d)).astype(np.float32)
    out, cache, attn = ctx.buffer(q.nbytes), paged.upload(ctx), H.Attention(d ** -0.5)
    bufs = [upload_new(ctx, x) for x in (q, paged.table, K.u32(lens))]
    ctx.begin_group()
    ctx.attn_decode(attn, cache, *bufs, out, 2, heads, paged.stride)
    step = ctx.end_group_recorded()
    want, tol = want_decode(paged, q, heads, float(np.float32(d ** -0.5)))
    for turn in range(3):
        out.zero(0, out.len())
        step.run()
        ctx.fence()
        got = f32(out, want.shape)
        K.near(got, want, tol, f"decode {type_id} {d} {turn}")
    ctx.attn_decode(attn, cache, *bufs, out, 2, heads, paged.stride)
    ctx.fence()
    assert np.array_equal(f32(out, want.shape).view(np.uint32), got.view(np.uint32))
for type_id, heads, d, news, lens in ((K.F16, 64, 128, [100, 60], [150, 60]), (K.F16, 64, 256, [100, 60], [150, 60]),
                                      (K.F16, 4, 128, [5, 3], [150, 60]), (K.F32, 4, 256, [5, 30], [150, 60])):
    paged = K.Paged(rng, type_id, 64, heads, d, lens)
    starts = np.concatenate([[0], np.cumsum(news)])
    q = rng.standard_normal((int(starts[-1]), heads * d)).astype(np.float32)
    out, cache, attn = ctx.buffer(q.nbytes), paged.upload(ctx), H.Attention(d ** -0.5)
    bufs = [upload_new(ctx, x) for x in (q, paged.table, K.u32(lens), K.u32(starts))]
    ctx.begin_group()
    ctx.attn_prefill(attn, cache, *bufs, out, len(q), 2, heads, paged.stride)
    step = ctx.end_group_recorded()
    want, tol = want_prefill(paged, q, heads, starts, news, float(np.float32(d ** -0.5)))
    for turn in range(3):
        out.zero(0, out.len())
        step.run()
        ctx.fence()
        got = f32(out, want.shape)
        K.near(got, want, tol, f"prefill {type_id} {d} {turn}")
    ctx.attn_prefill(attn, cache, *bufs, out, len(q), 2, heads, paged.stride)
    ctx.fence()
    assert np.array_equal(f32(out, want.shape).view(np.uint32), got.view(np.uint32))
print("recorded ok")
"""
    res = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100, cwd=ROOT)
    assert res.returncode == 0 and "recorded ok" in res.stdout, res.stderr[-2000:]
