"""GPU parity of the operators between a step's products (include/tm_hip.h): rotary
positions with the store into the paged cache, attention of single tokens and of ragged
chunks, logits; each against a plain 64-bit form. Whatever no sequence holds in a cache
is NaN, so that anything read past a mask shows."""
import os
import subprocess
import sys

import numpy as np
import pytest

import kvutil as K
import oracle as O
from tuckmill_amd import hip as H
from tuckmill_amd import synth as S

from q8util import require_gpu, upload_new

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = require_gpu()
    yield c
    c.close()


def f32(buf, shape):
    return buf.download_f32(0, int(np.prod(shape))).reshape(shape)


# ---- decode ------------------------------------------------------------------------------

LENS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 333, 700]


def run_decode(ctx, paged, q, heads, attn, extra=0, **more):
    seqs, d = len(paged.lens), paged.head_dim
    cache = paged.upload(ctx)
    qb, tb, lb = upload_new(ctx, q), upload_new(ctx, paged.table), upload_new(ctx, K.u32(paged.lens + extra))
    out = upload_new(ctx, np.full((seqs, heads * d), 7.0, np.float32))
    ctx.attn_decode(attn, cache, qb, tb, lb, out, seqs, heads, paged.stride, **more)
    ctx.fence()
    got = f32(out, (seqs, heads, d))
    ctx.attn_decode(attn, cache, qb, tb, lb, out, seqs, heads, paged.stride, **more)
    ctx.fence()
    assert np.array_equal(got.view(np.uint32), f32(out, (seqs, heads, d)).view(np.uint32))  # same bits
    return got


def want_decode(paged, q, heads, scale, first=None, window=0, softcap=0.0, slopes=None, seen=None):
    want, tol = [], []
    for s, n in enumerate(paged.lens):
        p = np.array([n - 1])
        lo, hi = K.bounds(p, n, None if first is None else first[s:s + 1], window)
        w, t = K.attention(q[s].reshape(1, heads, -1), paged.keys[s], paged.values[s], p, lo, hi, scale, softcap, slopes,
                           None if seen is None else seen[s])
        want.append(w[0])
        tol.append(t[0])
    return np.array(want), np.array(tol)


@pytest.mark.parametrize("type_id", [K.F16, K.F32])
@pytest.mark.parametrize("heads,kv_heads,d,page", [
    (16, 8, 128, 16), (4, 1, 256, 128), (3, 3, 64, 32), (12, 1, 64, 16), (40, 8, 128, 64), (17, 1, 80, 16), (2, 1, 8, 16),
    (32, 2, 96, 256), (6, 2, 200, 16), (33, 1, 128, 32)])
def test_decode_matches_the_plain_form(ctx, type_id, heads, kv_heads, d, page):
    rng = np.random.default_rng(heads * 1000 + d + page + type_id)
    paged = K.Paged(rng, type_id, page, kv_heads, d, LENS)
    q = rng.standard_normal((len(LENS), heads * d)).astype(np.float32)
    got = run_decode(ctx, paged, q, heads, H.Attention(d ** -0.5))
    want, tol = want_decode(paged, q, heads, np.float32(d ** -0.5))
    K.near(got, want, tol)
    assert not got[0].any()  # the empty sequence


@pytest.mark.parametrize("type_id", [K.F16, K.F32])
@pytest.mark.parametrize("window,cap,slopes,first", [(1, 0, 0, 0), (50, 0, 0, 0), (0, 5.0, 0, 0), (0, 50.0, 1, 0), (0, 0, 1, 1),
                                                     (100, 3.0, 1, 1), (4000000000, 0, 0, 0)])
def test_decode_masks_caps_and_biases(ctx, type_id, window, cap, slopes, first):
    rng = np.random.default_rng(5)
    heads, kv_heads, d = 8, 2, 64
    paged = K.Paged(rng, type_id, 16, kv_heads, d, LENS, scale=3.0)
    q = rng.standard_normal((len(LENS), heads * d)).astype(np.float32)
    sl = (2.0 ** -(1 + np.arange(heads))).astype(np.float32) if slopes else None
    fi = np.array([rng.integers(0, n + 2) for n in LENS]) if first else None
    if first:
        fi[-1] = 1 << 31  # beyond everything: an empty row
    attn = H.Attention(d ** -0.5, cap, window, slopes=upload_new(ctx, sl) if slopes else None,
                       first=upload_new(ctx, K.u32(fi)) if first else None)
    got = run_decode(ctx, paged, q, heads, attn)
    want, tol = want_decode(paged, q, heads, np.float32(d ** -0.5), fi, window, cap, sl)
    K.near(got, want, tol)


@pytest.mark.parametrize("type_id", [K.F16, K.F32])
def test_decode_long_sequences_are_split_and_joined(ctx, type_id):
    rng = np.random.default_rng(8)
    lens = [20001, 3, 0, 9000]
    paged = K.Paged(rng, type_id, 64, 2, 64, lens)
    q = rng.standard_normal((4, 4 * 64)).astype(np.float32)
    got = run_decode(ctx, paged, q, 4, H.Attention(0.125))
    want, tol = want_decode(paged, q, 4, 0.125)
    K.near(got, want, tol)
    # one sequence's bits do not depend on what else is in the call's table beyond its row
    one = K.Paged(rng, type_id, 64, 2, 64, [777])
    qq = rng.standard_normal((1, 4 * 64)).astype(np.float32)
    K.near(run_decode(ctx, one, qq, 4, H.Attention(0.125)), *want_decode(one, qq, 4, 0.125))


@pytest.mark.parametrize("type_id", [K.F16, K.F32])
def test_decode_extreme_scores(ctx, type_id):
    """Scores from -1e4 to 1e4, ties, scores that are all far below zero, tiny and huge q."""
    rng = np.random.default_rng(9)
    lens, heads, d = [65, 300, 300, 300, 300, 40], 2, 64
    paged = K.Paged(rng, type_id, 16, 1, d, lens)
    q = rng.standard_normal((len(lens), heads * d)).astype(np.float32)
    q[0] *= 3000.0
    paged.keys[1][:] = paged.keys[1][0]  # every score the same
    paged.keys[2][:, :, 0] = 100.0  # all scores near -1e4
    q[2] = 0.0
    q[2, ::d] = -800.0
    q[3] *= 1e-30
    q[4] *= 1e30
    q[5] = 0.0
    for s in (1, 2):
        for j in range(lens[s]):
            paged.put(s, j)
    got = run_decode(ctx, paged, q, heads, H.Attention(d ** -0.5))
    want, tol = want_decode(paged, q, heads, np.float32(d ** -0.5))
    # (a score of 1e30 decides by its largest value alone; it is finite in f32)
    K.near(got, want, tol)


@pytest.mark.parametrize("type_id", [K.F16, K.F32])
def test_decode_infinities_and_nan(ctx, type_id):
    rng = np.random.default_rng(10)
    lens, heads, d = [100, 100, 100, 100, 100], 1, 64
    paged = K.Paged(rng, type_id, 32, 1, d, lens)
    q = np.abs(rng.standard_normal((len(lens), heads * d))).astype(np.float32) + 0.1
    paged.keys[0][7] = np.nan     # before `first`: no influence
    paged.values[0][7] = np.inf
    paged.keys[1][:, 0, 0] = -np.inf  # every visible score -inf: zeros
    paged.keys[2][50, 0, 0] = -np.inf  # one position out
    paged.values[3][60] = np.nan  # a visible NaN
    paged.keys[4][60, 0, 0] = np.inf  # a score of +inf
    for s in range(5):
        for j in range(100):
            paged.put(s, j)
    first = np.array([8, 0, 0, 0, 0])
    attn = H.Attention(0.125, first=upload_new(ctx, K.u32(first)))
    got = run_decode(ctx, paged, q, heads, attn)
    want, tol = want_decode(paged, q, heads, 0.125, first)
    K.near(got[:3], want[:3], tol[:3])
    assert not got[1].any() and np.isnan(got[3]).all() and np.isnan(got[4]).all()


@pytest.mark.parametrize("type_id", [K.F16, K.F32])
def test_decode_pages_that_are_not_in_the_cache_are_not_seen(ctx, type_id):
    rng = np.random.default_rng(11)
    paged = K.Paged(rng, type_id, 16, 2, 64, [100, 64, 40])
    seen = [np.ones(n, bool) for n in (100, 64, 40)]
    paged.table[0, 2] = 0xffffffff
    seen[0][32:48] = False
    paged.table[1, :] = paged.pages  # none of its pages
    seen[1][:] = False
    q = rng.standard_normal((3, 4 * 64)).astype(np.float32)
    got = run_decode(ctx, paged, q, 4, H.Attention(0.125))
    want, tol = want_decode(paged, q, 4, 0.125, seen=seen)
    K.near(got, want, tol)
    assert not got[1].any()


def test_decode_lengths_beyond_the_table_are_cut(ctx):
    rng = np.random.default_rng(12)
    paged = K.Paged(rng, K.F16, 16, 1, 64, [64, 64])
    paged.stride -= 1
    paged.table = np.ascontiguousarray(paged.table[:, :-1])
    q = rng.standard_normal((2, 2 * 64)).astype(np.float32)
    got = run_decode(ctx, paged, q, 2, H.Attention(0.125), extra=np.array([3000000000, 1]))
    want, tol = want_decode(paged, q, 2, 0.125)
    K.near(got, want, tol)


@pytest.mark.parametrize("type_id", [K.F16, K.F32])
@pytest.mark.parametrize("q_off,out_off,q_more,out_more", [(0, 0, 0, 0), (3, 5, 7, 2), (64, 4, 128, 64)])
def test_decode_offsets_and_strides(ctx, type_id, q_off, out_off, q_more, out_more):
    rng = np.random.default_rng(13)
    lens, heads, d = [5, 90, 17], 4, 64
    paged = K.Paged(rng, type_id, 16, 2, d, lens)
    w = heads * d
    q = rng.standard_normal((3, w)).astype(np.float32)
    flat = np.full(q_off + 3 * (w + q_more), np.nan, np.float32)
    for s in range(3):
        flat[q_off + s * (w + q_more):][:w] = q[s]
    cache = paged.upload(ctx)
    out = upload_new(ctx, np.full(out_off + 3 * (w + out_more) + 9, 7.0, np.float32))
    ctx.attn_decode(H.Attention(0.125), cache, upload_new(ctx, flat), upload_new(ctx, paged.table),
                    upload_new(ctx, K.u32(lens)), out, 3, heads, paged.stride, q_off, out_off, w + q_more, w + out_more)
    ctx.fence()
    got = f32(out, (out_off + 3 * (w + out_more) + 9,))
    want, tol = want_decode(paged, q, heads, 0.125)
    written = np.zeros(got.shape, bool)
    for s in range(3):
        at = slice(out_off + s * (w + out_more), out_off + s * (w + out_more) + w)
        K.near(got[at].reshape(heads, d), want[s], tol[s])
        written[at] = True
    assert (got[~written] == 7.0).all()


# ---- prefill -----------------------------------------------------------------------------

def prefill_case(rng, news, lens, docs=False, prefix=False):
    """Row descriptions of a ragged batch."""
    starts = np.concatenate([[0], np.cumsum(news)])
    first = np.zeros(starts[-1], np.int64)
    pre = np.array([rng.integers(0, n + 3) for n in lens]) if prefix else None
    if docs:
        for s, (n, length) in enumerate(zip(news, lens)):
            cuts = np.array(sorted({0} | {int(rng.integers(0, length + 1)) for _ in range(3)}))
            p = np.arange(length - n, length)
            first[starts[s]:starts[s + 1]] = cuts[np.searchsorted(cuts, np.maximum(p, 0), side="right") - 1]
    return starts, first if docs else None, pre


def want_prefill(paged, q, heads, starts, news, scale, first=None, window=0, softcap=0.0, slopes=None, prefix=None, seen=None):
    want, tol = np.zeros((q.shape[0], heads, paged.head_dim)), np.zeros((q.shape[0], heads, paged.head_dim))
    for s, n in enumerate(news):
        r = slice(int(starts[s]), int(starts[s]) + int(n))
        length = int(paged.lens[s])
        p = np.arange(length - n, length)
        lo, hi = K.bounds(p, length, None if first is None else first[r], window, 0 if prefix is None else min(int(prefix[s]), length))
        want[r], tol[r] = K.attention(q[r].reshape(n, heads, paged.head_dim), paged.keys[s], paged.values[s], p, lo, hi, scale, softcap,
                                      slopes, None if seen is None else seen[s])
    return want, tol


def run_prefill(ctx, paged, q, heads, attn, starts, lens=None):
    rows, d = q.shape[0], paged.head_dim
    cache = paged.upload(ctx)
    bufs = [upload_new(ctx, x) for x in (q, paged.table, K.u32(paged.lens if lens is None else lens), K.u32(starts))]
    out = upload_new(ctx, np.full((rows, heads * d), 7.0, np.float32))
    got = []
    for _ in range(2):
        ctx.attn_prefill(attn, cache, *bufs, out, rows, len(starts) - 1, heads, paged.stride)
        ctx.fence()
        got.append(f32(out, (rows, heads, d)))
    assert np.array_equal(got[0].view(np.uint32), got[1].view(np.uint32))  # same bits
    return got[0]


NEWS = [1, 0, 2, 17, 33, 64, 65, 130]
CACHED = [0, 9, 40, 0, 95, 0, 31, 200]


@pytest.mark.parametrize("type_id", [K.F16, K.F32])
@pytest.mark.parametrize("heads,kv_heads,d,page", [
    (16, 8, 128, 16), (4, 1, 256, 128), (3, 3, 64, 32), (5, 1, 64, 16), (10, 2, 128, 64), (9, 3, 80, 16), (2, 1, 8, 16),
    (16, 1, 96, 256), (4, 2, 200, 16)])
def test_prefill_matches_the_plain_form(ctx, type_id, heads, kv_heads, d, page):
    rng = np.random.default_rng(heads * 1000 + d + page + type_id)
    lens = [n + c for n, c in zip(NEWS, CACHED)]
    paged = K.Paged(rng, type_id, page, kv_heads, d, lens)
    starts, _, _ = prefill_case(rng, NEWS, lens)
    q = rng.standard_normal((int(starts[-1]) + 3, heads * d)).astype(np.float32)
    got = run_prefill(ctx, paged, q, heads, H.Attention(d ** -0.5), starts)
    want, tol = want_prefill(paged, q, heads, starts, NEWS, np.float32(d ** -0.5))
    K.near(got[:-3], want[:-3], tol[:-3])
    assert (got[-3:] == 7.0).all()  # rows behind the last sequence


@pytest.mark.parametrize("type_id", [K.F16, K.F32])
@pytest.mark.parametrize("window,cap,slopes,docs,prefix", [
    (1, 0, 0, 0, 0), (40, 0, 0, 0, 0), (0, 4.0, 0, 0, 0), (0, 50.0, 1, 0, 0), (0, 0, 0, 1, 0), (0, 0, 0, 0, 1), (30, 0, 1, 0, 1),
    (64, 5.0, 1, 1, 1)])
def test_prefill_masks_caps_and_biases(ctx, type_id, window, cap, slopes, docs, prefix):
    rng = np.random.default_rng(21)
    heads, kv_heads, d = 4, 2, 64
    lens = [n + c for n, c in zip(NEWS, CACHED)]
    paged = K.Paged(rng, type_id, 16, kv_heads, d, lens, scale=3.0)
    starts, first, pre = prefill_case(rng, NEWS, lens, docs, prefix)
    if docs:
        first[4] = 0xffffffff  # a row that sees nothing
    q = rng.standard_normal((int(starts[-1]), heads * d)).astype(np.float32)
    sl = (2.0 ** -(1 + np.arange(heads))).astype(np.float32) if slopes else None
    attn = H.Attention(d ** -0.5, cap, window, slopes=upload_new(ctx, sl) if slopes else None,
                       first=upload_new(ctx, K.u32(first)) if docs else None,
                       prefix=upload_new(ctx, K.u32(pre)) if prefix else None)
    got = run_prefill(ctx, paged, q, heads, attn, starts)
    want, tol = want_prefill(paged, q, heads, starts, NEWS, np.float32(d ** -0.5), first, window, cap, sl, pre)
    K.near(got, want, tol)


@pytest.mark.parametrize("type_id", [K.F16, K.F32])
def test_prefill_few_rows_over_long_caches(ctx, type_id):
    rng = np.random.default_rng(22)
    news, lens = [4, 1, 5], [6000, 3000, 20]
    paged = K.Paged(rng, type_id, 16, 2, 64, lens)
    starts, _, _ = prefill_case(rng, news, lens)
    q = rng.standard_normal((10, 4 * 64)).astype(np.float32)
    got = run_prefill(ctx, paged, q, 4, H.Attention(0.125), starts)
    want, tol = want_prefill(paged, q, 4, starts, news, 0.125)
    K.near(got, want, tol)


@pytest.mark.parametrize("type_id", [K.F16, K.F32])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("at", [45, 100, 17])
def test_prefill_rows_do_not_see_what_lies_ahead(ctx, type_id, bad, at):
    """A key and a value that are not finite reach the rows from their position on, and no other
    (nor those whose document begins later)."""
    rng = np.random.default_rng(23)
    paged = K.Paged(rng, type_id, 16, 1, 64, [150])
    paged.keys[0][at, 0, 3] = bad
    paged.values[0][at] = bad
    paged.put(0, at)
    q = rng.standard_normal((130, 2 * 64)).astype(np.float32)
    first = np.zeros(130, np.int64)
    first[110:] = at + 1
    attn = H.Attention(0.125, first=upload_new(ctx, K.u32(first)))
    got = run_prefill(ctx, paged, q, 2, attn, np.array([0, 130]))
    with np.errstate(all="ignore"):
        want, tol = want_prefill(paged, q, 2, np.array([0, 130]), [130], 0.125, first)
    p = np.arange(20, 150)
    clean = (p < at) | (first > at)
    K.near(got[clean], want[clean], tol[clean])
    # (an infinite key may also give a score of -infinity, which takes the position out, or its
    # value's infinity times a weight of zero)
    if np.isnan(bad):
        assert np.isnan(got[~clean]).all()


@pytest.mark.parametrize("type_id", [K.F16, K.F32])
def test_prefill_bad_pages_lengths_and_bounds(ctx, type_id):
    rng = np.random.default_rng(24)
    news, lens = [20, 30, 10, 6], [50, 30, 10, 100]
    paged = K.Paged(rng, type_id, 16, 2, 64, lens)
    seen = [np.ones(n, bool) for n in lens]
    paged.table[0, 1] = 0xfffffff0
    seen[0][16:32] = False
    paged.table[3, :] = paged.pages
    seen[3][:] = False
    starts, _, _ = prefill_case(rng, news, lens)
    q = rng.standard_normal((66, 4 * 64)).astype(np.float32)
    got = run_prefill(ctx, paged, q, 4, H.Attention(0.125), starts)
    want, tol = want_prefill(paged, q, 4, starts, news, 0.125, seen=seen)
    K.near(got, want, tol)
    assert not got[60:].any()
    # a sequence of fewer cached tokens than rows: the first rows lie before its beginning
    short = paged.lens.copy()
    short[1] = 25
    got = run_prefill(ctx, paged, q, 4, H.Attention(0.125), starts, short)
    assert not got[20:25].any()
    part, ptol = K.attention(q[25:50].reshape(25, 4, 64), paged.keys[1][:25], paged.values[1][:25], np.arange(25),
                             *K.bounds(np.arange(25), 25), 0.125)
    K.near(got[25:50], part, ptol)
    # bounds that do not ascend, or leave the batch, leave their rows as they were
    got = run_prefill(ctx, paged, q, 4, H.Attention(0.125), np.array([0, 20, 10, 60, 4000000000]))
    K.near(got[:20], want[:20], tol[:20])
    assert (got[60:] == 7.0).all()


@pytest.mark.parametrize("type_id", [K.F16, K.F32])
def test_prefill_one_row_each_is_decode(ctx, type_id):
    rng = np.random.default_rng(25)
    lens = [1, 77, 300]
    paged = K.Paged(rng, type_id, 16, 2, 64, lens)
    q = rng.standard_normal((3, 8 * 64)).astype(np.float32)
    want, tol = want_decode(paged, q, 8, 0.125)
    K.near(run_prefill(ctx, paged, q, 8, H.Attention(0.125), np.arange(4)), want, tol)
    K.near(run_decode(ctx, paged, q, 8, H.Attention(0.125)), want, tol)


@pytest.mark.parametrize("type_id", [K.F16, K.F32])
def test_prefill_offsets_and_strides(ctx, type_id):
    rng = np.random.default_rng(26)
    heads, d, rows = 4, 64, 40
    paged = K.Paged(rng, type_id, 16, 2, d, [70])
    w, q_off, out_off, qs, os = heads * d, 3, 5, heads * d + 7, heads * d + 2
    q = rng.standard_normal((rows, w)).astype(np.float32)
    flat = np.full(q_off + rows * qs, np.nan, np.float32)
    for r in range(rows):
        flat[q_off + r * qs:][:w] = q[r]
    out = upload_new(ctx, np.full(out_off + rows * os + 9, 7.0, np.float32))
    ctx.attn_prefill(H.Attention(0.125), paged.upload(ctx), upload_new(ctx, flat), upload_new(ctx, paged.table),
                     upload_new(ctx, K.u32([70])), upload_new(ctx, K.u32([0, rows])), out, rows, 1, heads, paged.stride, q_off,
                     out_off, qs, os)
    ctx.fence()
    got = f32(out, (out_off + rows * os + 9,))
    want, tol = want_prefill(paged, q, heads, np.array([0, rows]), [rows], 0.125)
    written = np.zeros(got.shape, bool)
    for r in range(rows):
        at = slice(out_off + r * os, out_off + r * os + w)
        K.near(got[at].reshape(heads, d), want[r], tol[r])
        written[at] = True
    assert (got[~written] == 7.0).all()


# ---- positions and store --------------------------------------------------------------------

@pytest.mark.parametrize("type_id", [K.F16, K.F32])
@pytest.mark.parametrize("tokens,heads,kv_heads,d,rot,sections,interleaved,adjacent,page", [
    (1, 16, 8, 128, 128, [64], False, False, 16), (37, 4, 1, 256, 256, [128], False, True, 128),
    (19, 3, 3, 64, 32, [6, 5, 5], True, False, 16), (130, 8, 2, 80, 80, [24, 8, 8], False, True, 32),
    (5, 2, 1, 8, 2, [1], False, False, 16), (64, 6, 2, 96, 64, [8, 0, 20, 4], True, True, 64),
    (300, 5, 1, 128, 126, [21, 21, 21], True, False, 256)])
def test_rope_store_matches_the_plain_form(ctx, type_id, tokens, heads, kv_heads, d, rot, sections, interleaved, adjacent, page):
    rng = np.random.default_rng(tokens + d)
    pages = -(-tokens // page) + 2
    q, k, v = (rng.standard_normal((tokens, h * d)).astype(np.float32) for h in (heads, kv_heads, kv_heads))
    k[0, :3] = [1e6, -70000.0, 1e-9]  # beyond f16 both ways
    pos = rng.integers(0, 1 << 22, (len(sections), tokens))
    pos[:, 0] = (1 << 32) - 1
    pos[:, -1] = 0
    freqs = (1e6 ** (-2.0 * np.arange(rot // 2) / rot)).astype(np.float32)
    slots = rng.permutation(pages * page)[:tokens].astype(np.int64)
    if tokens > 10:
        slots[3] = -1
        slots[4] = pages * page  # just outside
        slots[6] = slots[9]  # the later one stays
    cache = H.KvCache.new(ctx, type_id, pages, page, kv_heads, d)
    old = rng.standard_normal((pages, kv_heads, page, d)).astype(K.DT[type_id])
    cache.k.upload(0, old)
    cache.v.upload(0, old)
    out = ctx.buffer(q.nbytes)
    rope = H.Rope(upload_new(ctx, freqs), rot, sections, interleaved, adjacent)
    args = [upload_new(ctx, x) for x in (q, k, v)] + [out, upload_new(ctx, K.u32(pos)), upload_new(ctx, K.u32(slots))]
    ctx.rope_store(rope, cache, *args, tokens, heads)
    ctx.fence()
    axis = K.axis_of_pairs(sections, interleaved)
    want, tol = K.rope(q.reshape(tokens, heads, d), pos, freqs, axis, rot, adjacent)
    K.near(f32(out, (tokens, heads, d)), want, tol, "q")
    wk, tk = K.rope(k.reshape(tokens, kv_heads, d), pos, freqs, axis, rot, adjacent)
    dt = K.DT[type_id]
    kc = cache.k.download(0, old.nbytes).view(dt).reshape(old.shape)
    vc = cache.v.download(0, old.nbytes).view(dt).reshape(pages, kv_heads, d, page)
    ek, ev = old.copy().astype(np.float64), old.reshape(vc.shape).copy().astype(np.float64)
    et = np.zeros(ek.shape)
    for t in range(tokens):
        s = int(slots[t])
        if 0 <= s < pages * page:
            ek[s // page, :, s % page], et[s // page, :, s % page] = wk[t], tk[t]
            ev[s // page, :, :, s % page] = v[t].reshape(kv_heads, d).astype(dt)
    if type_id == K.F16:  # one rounding to f16, of a value that may be off by the tolerance
        with np.errstate(over="ignore"):
            low, high = (ek - et).astype(np.float16), (ek + et).astype(np.float16)
        assert ((kc >= low) & (kc <= high)).all()
    else:
        K.near(kc, ek, et, "k")
    assert np.array_equal(vc.astype(np.float64), ev)
    # in place, and from the rows of one fused projection: the same bits
    both = np.concatenate([q, k, v], axis=1)
    fused, w, kw = upload_new(ctx, both), heads * d, kv_heads * d
    again = H.KvCache.new(ctx, type_id, pages, page, kv_heads, d)
    again.k.upload(0, old)
    again.v.upload(0, old)
    ctx.rope_store(rope, again, fused, fused, fused, fused, *args[4:], tokens, heads, 0, w, w + kw, 0, w + 2 * kw, w + 2 * kw,
                   w + 2 * kw, w + 2 * kw)
    ctx.fence()
    got = f32(fused, both.shape)
    assert np.array_equal(got[:, :w].view(np.uint32), f32(out, (tokens, w)).view(np.uint32))
    assert np.array_equal(got[:, w:], both[:, w:])
    assert np.array_equal(again.k.download(0, old.nbytes), cache.k.download(0, old.nbytes))
    assert np.array_equal(again.v.download(0, old.nbytes), cache.v.download(0, old.nbytes))


def test_rope_odd_offsets_and_strides(ctx):
    rng = np.random.default_rng(31)
    tokens, heads, kv_heads, d = 9, 3, 1, 24
    w, kw = heads * d, kv_heads * d
    offs = dict(q_off=1, k_off=2, v_off=3, out_off=5, q_stride=w + 3, k_stride=kw + 1, v_stride=kw + 5, out_stride=w + 1)
    rows = {n: rng.standard_normal((tokens, x)).astype(np.float32) for n, x in (("q", w), ("k", kw), ("v", kw))}
    bufs = {}
    for n, x in rows.items():
        flat = np.full(offs[n + "_off"] + tokens * offs[n + "_stride"], np.nan, np.float32)
        for t in range(tokens):
            flat[offs[n + "_off"] + t * offs[n + "_stride"]:][:x.shape[1]] = x[t]
        bufs[n] = upload_new(ctx, flat)
    freqs = np.array([1.0, 0.1, 0.01], np.float32)
    pos = rng.integers(0, 5000, (1, tokens))
    out = upload_new(ctx, np.full(5 + tokens * (w + 1), 7.0, np.float32))
    cache = H.KvCache.new(ctx, K.F32, 1, 16, kv_heads, d)
    ctx.rope_store(H.Rope(upload_new(ctx, freqs), 6), cache, bufs["q"], bufs["k"], bufs["v"], out, upload_new(ctx, K.u32(pos)),
                   upload_new(ctx, K.u32(np.arange(tokens))), tokens, heads, **offs)
    ctx.fence()
    got = f32(out, (5 + tokens * (w + 1),))
    want, tol = K.rope(rows["q"].reshape(tokens, heads, d), pos, freqs, [0] * 3, 6, False)
    for t in range(tokens):
        K.near(got[5 + t * (w + 1):][:w].reshape(heads, d), want[t], tol[t])
        assert got[5 + t * (w + 1) + w:][:1].size == 0 or got[5 + t * (w + 1) + w] == 7.0
    vc = cache.v.download_f32(0, 16 * d).reshape(d, 16)
    assert np.array_equal(vc[:, :tokens], rows["v"].T) and not vc[:, tokens:].any()


# ---- logits -------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,vocab,hist,biases,mask", [
    (1, 1, 1, 1, 1), (3, 33, 50, 4, 1), (2, 4096, 100, 0, 0), (5, 4097, 0, 7, 1), (1, 151936, 700, 0, 0), (4, 20011, 3000, 300, 1),
    (2, 8191, 9, 0, 1), (3, 8195, 1, 1, 0)])
def test_logits_adjust_matches_the_plain_form(ctx, rows, vocab, hist, biases, mask):
    rng = np.random.default_rng(vocab)
    x = (rng.standard_normal((rows, vocab)) * 5).astype(np.float32)
    x[0, 0] = 0.0
    if vocab > 20:
        x[0, 1:6] = [np.inf, -np.inf, np.nan, -0.0, 1e-40]
    kw, ref = {}, {}
    if hist:
        ids = (rng.random((rows, hist)) ** 3 * vocab).astype(np.int64)
        ids[:, ::7] = 3 % vocab
        ids[:, 1::11] = [vocab]  # outside the vocabulary
        ids[0, 0] = 0xffffffff
        lens = np.array([rng.integers(0, hist + 1) for _ in range(rows)])
        lens[0] = hist + 5  # cut at the stride
        pen = np.stack([rng.uniform(0.8, 1.6, rows), rng.uniform(-1, 1, rows), rng.uniform(0, 0.3, rows)], 1).astype(np.float32)
        ref.update(history=ids, history_len=lens, penalties=pen)
        kw.update(history=upload_new(ctx, K.u32(ids)), history_len=upload_new(ctx, K.u32(lens)), penalties=upload_new(ctx, pen),
                  history_stride=hist)
    if biases:
        bid = rng.integers(0, vocab, (rows, biases))
        bid[:, ::5] = 2 % vocab  # the same id again: the last one counts
        if biases > 3:
            bid[0, 1] = vocab + 1
        bval = rng.standard_normal((rows, biases)).astype(np.float32)
        blen = np.array([rng.integers(0, biases + 1) for _ in range(rows)])
        blen[0] = 0xffffffff
        ref.update(bias_ids=bid, bias_values=bval, bias_len=blen)
        kw.update(bias_ids=upload_new(ctx, K.u32(bid)), bias_values=upload_new(ctx, bval), bias_len=upload_new(ctx, K.u32(blen)),
                  bias_stride=biases)
    if mask:
        words = -(-vocab // 32) + 1
        al = rng.integers(0, 1 << 32, (rows, words), dtype=np.uint64).astype(np.uint32)
        al[rows - 1] = 0  # nothing allowed
        ref.update(allowed=al)
        kw.update(allowed=upload_new(ctx, al), allowed_stride=words)
    spec = H.LogitsAdjust(**kw)
    want, tol = K.adjust(x, **ref)
    xb, out = upload_new(ctx, x), upload_new(ctx, np.full(rows * vocab + 8, 7.0, np.float32))
    ctx.logits_adjust(spec, xb, out, rows, vocab, 0, 4)
    ctx.fence()
    got = f32(out, (rows * vocab + 8,))
    K.near(got[4:-4].reshape(rows, vocab), want, tol)
    assert (got[:4] == 7.0).all() and (got[-4:] == 7.0).all()
    if not (hist or biases or mask):
        assert np.array_equal(got[4:-4].view(np.uint32), x.reshape(-1).view(np.uint32))
    ctx.logits_adjust(spec, xb, xb, rows, vocab)  # in place
    ctx.fence()
    assert np.array_equal(f32(xb, (rows * vocab,)).view(np.uint32), got[4:-4].view(np.uint32))


# ---- together ---------------------------------------------------------------------------------

def test_a_decode_step_of_recorded_operators_over_several_tokens(ctx):
    """A layer's attention half and the pick of a token, as a program encodes them: norm, the three
    projections, positions and store, attention, output projection, residual, norm, vocabulary,
    penalties, argmax; recorded once and replayed for every token with new positions, slots and
    lengths, against a plain form of the whole. Another operator runs between the replays."""
    rng = np.random.default_rng(41)
    hidden, heads, kv_heads, d, vocab, page, steps = 256, 4, 2, 64, 512, 16, 5
    seqs = 2
    w, kw = heads * d, kv_heads * d
    mats = {}
    for i, (n, rows, cols) in enumerate((("q", w, hidden), ("k", kw, hidden), ("v", kw, hidden), ("o", hidden, w), ("vocab", vocab, hidden))):
        raw = S.make_weights(rows, cols, 50 + i)
        mats[n] = (H.Matrix.load(ctx, raw, cols, rows), raw, rows, cols)
    dense = {n: np.stack([O.gemm_q8_0_f32(raw, rows, cols, np.eye(cols, dtype=np.float32)[i], 1)[0] for i in range(cols)], 1)
             for n, (_, raw, rows, cols) in mats.items()}
    lens = np.array([20, 3])
    paged = K.Paged(rng, K.F16, page, kv_heads, d, lens + steps)
    cache = paged.upload(ctx)
    norm = upload_new(ctx, np.ones(hidden, np.float32))
    freqs = (1e4 ** (-np.arange(d // 2) / (d // 2))).astype(np.float32)
    hist0 = rng.integers(0, vocab, (seqs, 40))
    pen = np.array([[1.3, 0.5, 0.2], [1.1, 0.0, 0.1]], np.float32)
    b = {n: ctx.buffer(4 * size) for n, size in (("x", seqs * hidden), ("n", seqs * hidden), ("q", seqs * w), ("qr", seqs * w),
                                                ("k", seqs * kw), ("v", seqs * kw), ("a", seqs * w), ("o", seqs * hidden),
                                                ("l", seqs * vocab), ("pos", seqs), ("slots", seqs), ("lens", seqs), ("pick", 8),
                                                ("one", vocab), ("hlen", seqs))}
    partial = ctx.buffer(H.ARGMAX_PARTIAL_BYTES)
    table, history = upload_new(ctx, paged.table), upload_new(ctx, K.u32(hist0))
    rope, attn = H.Rope(upload_new(ctx, freqs), d), H.Attention(d ** -0.5)
    adjust = H.LogitsAdjust(history, b["hlen"], upload_new(ctx, pen), history_stride=40)

    def encode():
        ctx.rmsnorm(b["x"], norm, b["n"], seqs, hidden, 1e-6)
        for n in ("q", "k", "v"):
            mats[n][0].gemm(ctx, b["n"], b[n], seqs, exact=True)
        ctx.rope_store(rope, cache, b["q"], b["k"], b["v"], b["qr"], b["pos"], b["slots"], seqs, heads)
        ctx.attn_decode(attn, cache, b["qr"], table, b["lens"], b["a"], seqs, heads, paged.stride)
        mats["o"][0].gemm(ctx, b["a"], b["o"], seqs, exact=True)
        ctx.f32_axpy(b["o"], b["x"], 1.0, seqs * hidden)
        ctx.rmsnorm(b["x"], norm, b["n"], seqs, hidden, 1e-6)
        mats["vocab"][0].gemm(ctx, b["n"], b["l"], seqs, exact=True)
        ctx.logits_adjust(adjust, b["l"], b["l"], seqs, vocab)
        for s in range(seqs):
            ctx.copy_f32(b["l"], s * vocab, b["one"], 0, vocab)
            ctx.argmax_f32(b["one"], vocab, partial, b["pick"], s)

    ctx.begin_group()
    encode()
    step = ctx.end_group_recorded()
    x0 = rng.standard_normal((seqs, hidden)).astype(np.float32)
    keys = [list(paged.keys[s][:lens[s]].astype(np.float64)) for s in range(seqs)]
    values = [list(paged.values[s][:lens[s]].astype(np.float64)) for s in range(seqs)]
    rms = lambda y: y / np.sqrt((y * y).mean(1, keepdims=True) + 1e-6)  # noqa: E731
    for i in range(steps):
        at = lens + i
        pages = [paged.table[s, at[s] // page] for s in range(seqs)]
        x = (x0 * (1 + 0.3 * i)).astype(np.float32)
        b["x"].upload(0, x)
        b["pos"].upload(0, K.u32(at))
        b["slots"].upload(0, K.u32([int(pages[s]) * page + at[s] % page for s in range(seqs)]))
        b["lens"].upload(0, K.u32(at + 1))
        b["hlen"].upload(0, K.u32([10 + i, 30 + i]))
        step.run()
        ctx.fence()
        n = rms(x.astype(np.float64))
        q, k, v = (n @ dense[m].T.astype(np.float64) for m in ("q", "k", "v"))
        q, _ = K.rope(q.reshape(seqs, heads, d), at[None], freqs, [0] * (d // 2), d, False)
        k, _ = K.rope(k.reshape(seqs, kv_heads, d), at[None], freqs, [0] * (d // 2), d, False)
        a = np.zeros((seqs, heads, d))
        for s in range(seqs):
            keys[s].append(k[s].astype(np.float16).astype(np.float64))
            values[s].append(v[s].reshape(kv_heads, d).astype(np.float16).astype(np.float64))
            m = len(keys[s])
            a[s] = K.attention(q[s:s + 1], np.array(keys[s]), np.array(values[s]), np.array([m - 1]), np.array([0]), np.array([m]),
                               d ** -0.5)[0][0]
        got = f32(b["a"], (seqs, heads, d))
        # a key or value whose f32 value lies next to a border of f16 may round the other way: one f16
        # step (2^-10) of one of m cached tokens; the rest is f32
        scale = np.abs(a).max()
        assert np.abs(got - a).max() <= scale * 2.0 ** -10, i
        y = x + a.reshape(seqs, -1) @ dense["o"].T.astype(np.float64)
        logits = rms(y) @ dense["vocab"].T.astype(np.float64)
        want, _ = K.adjust(logits.astype(np.float32), hist0, [10 + i, 30 + i], pen)
        got = f32(b["l"], (seqs, vocab))
        assert np.abs(got - want).max() <= np.abs(want).max() * 2.0 ** -9, i
        assert np.array_equal(b["pick"].download(0, 4 * seqs).view(np.uint32), got.argmax(1).astype(np.uint32))
        ctx.f32_scale(b["l"], b["one"], 2.0, vocab)  # something else in between
        replay = f32(b["a"], (seqs, heads, d)).copy()
        b["x"].upload(0, x)
        ctx.begin_group()
        encode()
        ctx.end_group()
        ctx.fence()
        assert np.array_equal(f32(b["a"], replay.shape).view(np.uint32), replay.view(np.uint32))  # replayed or not


def test_two_recorded_steps_share_the_context(ctx):
    """Two recorded steps whose attention needs workspace of different sizes, replayed in turns."""
    rng = np.random.default_rng(42)
    made = []
    for lens in ([3000], [700, 9000]):
        paged = K.Paged(rng, K.F16, 64, 2, 64, lens)
        q = rng.standard_normal((len(lens), 4 * 64)).astype(np.float32)
        out = ctx.buffer(q.nbytes)
        cache, bufs = paged.upload(ctx), [upload_new(ctx, x) for x in (q, paged.table, K.u32(lens))]
        ctx.begin_group()
        ctx.attn_decode(H.Attention(0.125), cache, *bufs, out, len(lens), 4, paged.stride)
        made.append((ctx.end_group_recorded(), out, want_decode(paged, q, 4, 0.125), cache, bufs))
    for turn in range(3):
        for step, out, (want, tol), _, _ in made:
            out.zero(0, out.len())
            step.run()
        for step, out, (want, tol), _, _ in made:
            ctx.fence()
            K.near(f32(out, want.shape), want, tol, f"turn {turn}")


def test_two_contexts_at_once(ctx):
    rng = np.random.default_rng(43)
    other = H.HipContext.open()
    try:
        outs = []
        paged = K.Paged(rng, K.F16, 64, 2, 64, [5000, 8])
        q = rng.standard_normal((2, 4 * 64)).astype(np.float32)
        for c in (ctx, other):
            cache, bufs, out = paged.upload(c), [upload_new(c, x) for x in (q, paged.table, K.u32(paged.lens))], c.buffer(q.nbytes)
            outs.append((c, cache, bufs, out))
        for _ in range(20):
            for c, cache, bufs, out in outs:
                c.attn_decode(H.Attention(0.125), cache, *bufs, out, 2, 4, paged.stride)
        want, tol = want_decode(paged, q, 4, 0.125)
        for c, cache, bufs, out in outs:
            c.fence()
            K.near(f32(out, want.shape), want, tol)
        for o in outs:  # (the other context's buffers go before it does)
            if o[0] is other:
                for x in [o[1].k, o[1].v, o[3], *o[2]]:
                    x.free()
    finally:
        other.close()


def test_buffer_contents_as_a_device_array(ctx):
    """In a process of its own: torch brings a HIP runtime along and has to be imported before this
    library loads one."""
    with pytest.raises(H.TuckmillError):
        ctx.buffer(64, shared=False).contents()
    code = """
import torch
assert torch.cuda.is_available()
import numpy as np
from tuckmill_amd import hip as H
ctx = H.HipContext.open()
buf = ctx.buffer(400)
buf.upload(0, np.arange(100, dtype=np.float32))
ctx.fence()
view = torch.as_tensor(buf, device="cuda").view(torch.float32)
assert view.data_ptr() == buf.contents() and view.shape == (100,)
view.mul_(2.0)
torch.cuda.synchronize()
assert np.array_equal(buf.download_f32(0, 100), np.arange(100, dtype=np.float32) * 2)
print("view ok")
"""
    res = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100,
                         cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert res.returncode == 0 and "view ok" in res.stdout, res.stderr[-2000:]
