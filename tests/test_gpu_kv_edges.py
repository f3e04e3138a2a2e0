"""Paged attention at its edges."""
import numpy as np
import pytest

import kvutil as K
from tuckmill_amd import hip as H

from q8util import require_gpu, upload_new
from test_gpu_kv import f32, run_decode, run_prefill
from test_gpu_kv_many import many

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = require_gpu()
    yield c
    c.close()


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
