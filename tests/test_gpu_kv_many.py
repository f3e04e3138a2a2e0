"""Paged attention where a call has many rows, many sequences or long ones: ragged batches
of f16 pages with enough rows for the kernel with tiles of 128 (more than 1056 tiles of eight
rows over all key-value heads), and the shares that the other kernel cuts positions into."""
import numpy as np
import pytest

import kvutil as K
from tuckmill_amd import hip as H

from q8util import require_gpu, upload_new
from test_gpu_kv import CACHED, NEWS, f32, prefill_case, run_decode, run_prefill, want_decode, want_prefill

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = require_gpu()
    yield c
    c.close()


def many(rows, seqs, heads, kv_heads):
    """Whether the rows are enough for tiles of 128."""
    return (rows * (heads // kv_heads) // 8 + seqs) * kv_heads > 1056


@pytest.mark.parametrize("heads,kv_heads,d,page", [
    (64, 64, 64, 16), (32, 16, 128, 32), (30, 10, 256, 64), (64, 64, 8, 16), (32, 32, 72, 128), (32, 16, 136, 256), (72, 12, 40, 16),
    (32, 32, 128, 64)])
def test_tiles_of_rows_match_the_plain_form(ctx, heads, kv_heads, d, page):
    rng = np.random.default_rng(heads * 1000 + d + page)
    lens = [n + c for n, c in zip(NEWS, CACHED)]
    paged = K.Paged(rng, K.F16, page, kv_heads, d, lens)
    starts, _, _ = prefill_case(rng, NEWS, lens)
    assert many(int(starts[-1]) + 3, len(NEWS), heads, kv_heads)
    q = rng.standard_normal((int(starts[-1]) + 3, heads * d)).astype(np.float32)
    got = run_prefill(ctx, paged, q, heads, H.Attention(d ** -0.5), starts)
    want, tol = want_prefill(paged, q, heads, starts, NEWS, np.float32(d ** -0.5))
    K.near(got[:-3], want[:-3], tol[:-3])
    assert (got[-3:] == 7.0).all()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window,cap,slopes,docs,prefix,scale", [
    (1, 0, 0, 0, 0, 1.0), (50, 5.0, 0, 0, 0, 1.0), (0, 50.0, 1, 1, 0, 1.0), (64, 0, 1, 1, 1, 1.0), (0, 0, 0, 0, 1, 1.0),
    (0, 0, 0, 0, 0, -1.0), (0, 5.0, 1, 0, 0, -0.5), (0, 0, 0, 1, 0, 0.0)])
def test_tiles_of_rows_with_masks_caps_and_biases(ctx, d, window, cap, slopes, docs, prefix, scale):
    rng = np.random.default_rng(31)
    heads = kv_heads = 32
    lens = [n + c for n, c in zip(NEWS, CACHED)]
    paged = K.Paged(rng, K.F16, 16, kv_heads, d, lens, scale=3.0)
    starts, first, pre = prefill_case(rng, NEWS, lens, docs, prefix)
    if docs:
        first[4] = 0xffffffff  # a row that sees nothing
    assert many(int(starts[-1]), len(NEWS), heads, kv_heads)
    q = rng.standard_normal((int(starts[-1]), heads * d)).astype(np.float32)
    sl = (2.0 ** -(1 + np.arange(heads) / 4)).astype(np.float32) if slopes else None
    by = float(np.float32(d ** -0.5 * scale))
    attn = H.Attention(by, cap, window, slopes=upload_new(ctx, sl) if slopes else None,
                       first=upload_new(ctx, K.u32(first)) if docs else None,
                       prefix=upload_new(ctx, K.u32(pre)) if prefix else None)
    got = run_prefill(ctx, paged, q, heads, attn, starts)
    want, tol = want_prefill(paged, q, heads, starts, NEWS, by, first, window, cap, sl, pre)
    K.near(got, want, tol)


@pytest.mark.parametrize("kv_heads,d", [(32, 64), (16, 128), (16, 256)])
def test_tiles_of_rows_over_long_caches_share_positions(ctx, kv_heads, d):
    rng = np.random.default_rng(32)
    news, lens = [200, 330], [1500, 1100]
    paged = K.Paged(rng, K.F16, 64, kv_heads, d, lens)
    starts, _, _ = prefill_case(rng, news, lens)
    assert many(530, 2, kv_heads, kv_heads)
    q = rng.standard_normal((530, kv_heads * d)).astype(np.float32)
    got = run_prefill(ctx, paged, q, kv_heads, H.Attention(d ** -0.5, window=900), starts)
    want, tol = want_prefill(paged, q, kv_heads, starts, news, float(np.float32(d ** -0.5)), window=900)
    K.near(got, want, tol)


@pytest.mark.parametrize("kv_heads", [1, 64])
@pytest.mark.parametrize("type_id", [K.F16, K.F32])
@pytest.mark.parametrize("d", [64, 128, 256, 24])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("at", [45, 100])
def test_values_that_are_not_finite_stay_with_the_rows_that_see_them(ctx, kv_heads, type_id, d, bad, at):
    rng = np.random.default_rng(33)
    paged = K.Paged(rng, type_id, 16, kv_heads, d, [150])
    paged.keys[0][at, 0, 3] = bad
    paged.values[0][at] = bad
    paged.values[0][at + 7, :, d - 2] = -bad
    paged.put(0, at)
    paged.put(0, at + 7)
    q = rng.standard_normal((130, kv_heads * d)).astype(np.float32)
    first = np.zeros(130, np.int64)
    first[115:] = at + 8
    attn = H.Attention(0.125, first=upload_new(ctx, K.u32(first)))
    got = run_prefill(ctx, paged, q, kv_heads, attn, np.array([0, 130]))
    with np.errstate(all="ignore"):
        want, tol = want_prefill(paged, q, kv_heads, np.array([0, 130]), [130], 0.125, first)
    p = np.arange(20, 150)
    clean = (p < at) | (first > at + 7)
    K.near(got[clean], want[clean], tol[clean])
    assert np.isnan(got[clean]).sum() == 0
    if np.isnan(bad):
        assert np.isnan(got[~clean]).all()


@pytest.mark.parametrize("type_id", [K.F16, K.F32])
def test_tiles_of_rows_with_bad_pages_lengths_and_bounds(ctx, type_id):
    rng = np.random.default_rng(34)
    news, lens, heads = [20, 30, 10, 60], [50, 30, 10, 100], 64
    paged = K.Paged(rng, type_id, 16, heads, 64, lens)
    seen = [np.ones(n, bool) for n in lens]
    paged.table[0, 1] = 0xfffffff0
    seen[0][16:32] = False
    paged.table[3, :] = paged.pages
    seen[3][:] = False
    starts, _, _ = prefill_case(rng, news, lens)
    q = rng.standard_normal((120, heads * 64)).astype(np.float32)
    got = run_prefill(ctx, paged, q, heads, H.Attention(0.125), starts)
    want, tol = want_prefill(paged, q, heads, starts, news, 0.125, seen=seen)
    K.near(got, want, tol)
    assert not got[60:].any()
    short = paged.lens.copy()
    short[1] = 25
    got = run_prefill(ctx, paged, q, heads, H.Attention(0.125), starts, short)
    assert not got[20:25].any()
    part, ptol = K.attention(q[25:50].reshape(25, heads, 64), paged.keys[1][:25], paged.values[1][:25], np.arange(25),
                             *K.bounds(np.arange(25), 25), 0.125)
    K.near(got[25:50], part, ptol)
    got = run_prefill(ctx, paged, q, heads, H.Attention(0.125), np.array([0, 20, 10, 60, 4000000000]))
    K.near(got[:20], want[:20], tol[:20])
    assert (got[60:] == 7.0).all()


def test_tiles_of_rows_at_odd_offsets_and_strides(ctx):
    rng = np.random.default_rng(35)
    heads, d, rows = 64, 64, 140
    paged = K.Paged(rng, K.F16, 16, heads, d, [170])
    w, q_off, out_off, qs, os = heads * d, 3, 5, heads * d + 7, heads * d + 2
    q = rng.standard_normal((rows, w)).astype(np.float32)
    flat = np.full(q_off + rows * qs, np.nan, np.float32)
    for r in range(rows):
        flat[q_off + r * qs:][:w] = q[r]
    out = upload_new(ctx, np.full(out_off + rows * os + 9, 7.0, np.float32))
    ctx.attn_prefill(H.Attention(0.125), paged.upload(ctx), upload_new(ctx, flat), upload_new(ctx, paged.table),
                     upload_new(ctx, K.u32([170])), upload_new(ctx, K.u32([0, rows])), out, rows, 1, heads, paged.stride, q_off,
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


@pytest.mark.parametrize("type_id", [K.F16, K.F32])
@pytest.mark.parametrize("seqs", [64, 65, 200, 513, 700])
def test_decode_of_many_ragged_sequences(ctx, type_id, seqs):
    rng = np.random.default_rng(seqs + type_id)
    lens = [int(n) for n in 10 ** rng.uniform(-1, 2.3, seqs)]
    lens[0], lens[seqs // 2], lens[-1] = 3000, 0, 2500
    paged = K.Paged(rng, type_id, 16, 2, 64, lens)
    q = rng.standard_normal((seqs, 4 * 64)).astype(np.float32)
    got = run_decode(ctx, paged, q, 4, H.Attention(0.125, window=2000))
    want, tol = want_decode(paged, q, 4, 0.125, window=2000)
    K.near(got, want, tol)


@pytest.mark.parametrize("type_id", [K.F16, K.F32])
def test_ragged_rows_of_many_sequences(ctx, type_id):
    rng = np.random.default_rng(36)
    news = [int(n) for n in rng.integers(0, 4, 150)]
    lens = [n + int(10 ** rng.uniform(0, 2.5)) for n in news]
    lens[70] += 2000
    paged = K.Paged(rng, type_id, 16, 1, 128, lens)
    starts, _, _ = prefill_case(rng, news, lens)
    q = rng.standard_normal((int(starts[-1]), 3 * 128)).astype(np.float32)
    got = run_prefill(ctx, paged, q, 3, H.Attention(0.1), starts)
    want, tol = want_prefill(paged, q, 3, starts, news, float(np.float32(0.1)))
    K.near(got, want, tol)


@pytest.mark.parametrize("type_id", [K.F16, K.F32])
@pytest.mark.parametrize("scale,cap", [(-0.125, 0.0), (0.0, 0.0), (-0.5, 4.0), (0.0, 4.0)])
def test_decode_scales_below_and_at_zero(ctx, type_id, scale, cap):
    rng = np.random.default_rng(37)
    paged = K.Paged(rng, type_id, 16, 2, 64, [40, 1, 333])
    q = rng.standard_normal((3, 8 * 64)).astype(np.float32)
    got = run_decode(ctx, paged, q, 8, H.Attention(scale, cap))
    want, tol = want_decode(paged, q, 8, scale, softcap=cap)
    K.near(got, want, tol)


@pytest.mark.parametrize("type_id", [K.F16, K.F32])
@pytest.mark.parametrize("scattered", [0, 1])
def test_of_rows_far_apart_that_name_one_slot_the_last_is_stored(ctx, type_id, scattered):
    rng = np.random.default_rng(38)
    tokens, heads, kv_heads, d, page = 2500, 2, 2, 16, 16
    pages = 64
    slots = rng.integers(0, pages * page, tokens) if scattered else np.arange(tokens) % (pages * page - 5)
    q, k, v = (rng.standard_normal((tokens, h * d)).astype(np.float32) for h in (heads, kv_heads, kv_heads))
    cache = H.KvCache.new(ctx, type_id, pages, page, kv_heads, d)
    cache.k.upload(0, np.zeros((pages, kv_heads, page, d), K.DT[type_id]))
    cache.v.upload(0, np.zeros((pages, kv_heads, d, page), K.DT[type_id]))
    rope = H.Rope(upload_new(ctx, np.zeros(d // 2, np.float32)), d, [d // 2], False, False)  # (turns by nothing)
    ctx.rope_store(rope, cache, *[upload_new(ctx, x) for x in (q, k, v)], ctx.buffer(q.nbytes),
                   upload_new(ctx, K.u32(np.arange(tokens))), upload_new(ctx, K.u32(slots)), tokens, heads)
    ctx.fence()
    ek, ev = np.zeros((pages, kv_heads, page, d), K.DT[type_id]), np.zeros((pages, kv_heads, d, page), K.DT[type_id])
    for t, s in enumerate(slots):
        ek[s // page, :, s % page] = k[t].reshape(kv_heads, d)
        ev[s // page, :, :, s % page] = v[t].reshape(kv_heads, d)
    assert np.array_equal(cache.k.download(0, ek.nbytes).view(ek.dtype).reshape(ek.shape), ek)
    assert np.array_equal(cache.v.download(0, ev.nbytes).view(ev.dtype).reshape(ev.shape), ev)


@pytest.mark.parametrize("type_id,heads,kv_heads", [(K.F16, 8, 4), (K.F32, 8, 4), (K.F16, 64, 64)])
@pytest.mark.parametrize("cap", [0.0, 2.0 ** -140])
def test_steep_biases_and_a_cap_of_next_to_nothing(ctx, type_id, heads, kv_heads, cap):
    rng = np.random.default_rng(39)
    news, lens = [130, 6], [230, 40]
    paged = K.Paged(rng, type_id, 16, kv_heads, 64, lens)
    paged.keys[0][100] = 0  # scores of zero
    paged.put(0, 100)
    starts, _, _ = prefill_case(rng, news, lens)
    q = rng.standard_normal((136, heads * 64)).astype(np.float32)
    slopes = (2.0 ** rng.integers(-3, 6, heads) * 1.1).astype(np.float32)
    attn = H.Attention(0.125, cap, slopes=upload_new(ctx, slopes))
    got = run_prefill(ctx, paged, q, heads, attn, starts)
    want, tol = want_prefill(paged, q, heads, starts, news, 0.125, softcap=cap, slopes=slopes)
    K.near(got, want, tol)
    if many(136, 2, heads, kv_heads):
        return
    got = run_decode(ctx, paged, q[:2], heads, attn)
    want, tol = want_decode(paged, q[:2], heads, 0.125, softcap=cap, slopes=slopes)
    K.near(got, want, tol)


@pytest.mark.parametrize("rows,vocab", [(3, 3000), (40, 60001)])
@pytest.mark.parametrize("hist,biases", [(65535, 65534), (65536, 5), (5, 65535), (70000, 70000)])
def test_logits_with_long_lists(ctx, rows, vocab, hist, biases):
    rng = np.random.default_rng(40)
    x = (rng.standard_normal((rows, vocab)) * 5).astype(np.float32)
    history = rng.integers(0, vocab + 3, (rows, hist)).astype(np.uint32)
    history[0] = 7  # one id, as often as there are entries
    ids = rng.integers(0, vocab + 3, (rows, biases)).astype(np.uint32)
    ids[1] = 8  # one id: the last entry counts
    values = rng.standard_normal((rows, biases)).astype(np.float32)
    hl, bl = np.full(rows, hist + 9), np.full(rows, biases)
    hl[2], bl[2] = hist // 2, biases // 2
    pen = np.tile(np.array([1.3, 0.4, 1e-3], np.float32), (rows, 1))
    bufs = [upload_new(ctx, v) for v in (history, K.u32(hl), pen, ids, values, K.u32(bl))]
    adjust = H.LogitsAdjust(*bufs, history_stride=hist, bias_stride=biases)
    xb = upload_new(ctx, x)
    out = ctx.buffer(x.nbytes)
    ctx.logits_adjust(adjust, xb, out, rows, vocab)
    ctx.fence()
    want, tol = K.adjust(x, history, hl, pen, ids, values, bl)
    K.near(f32(out, x.shape), want, tol)


@pytest.mark.parametrize("type_id,heads,kv_heads", [(K.F16, 4, 2), (K.F32, 4, 2), (K.F16, 64, 64)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_infinite_queries_keep_to_themselves(ctx, type_id, heads, kv_heads, d):
    rng = np.random.default_rng(41)
    news, lens = [130, 6], [150, 40]
    paged = K.Paged(rng, type_id, 16, kv_heads, d, lens)
    for s in range(2):
        paged.keys[s][:, :, 5] = -np.abs(paged.keys[s][:, :, 5]) - 1
        for j in range(lens[s]):
            paged.put(s, j)
    starts, _, _ = prefill_case(rng, news, lens)
    q = rng.standard_normal((136, heads, d)).astype(np.float32)
    q[17] = 0
    q[17, :, 5] = np.inf  # every score is -infinity
    q[40, :, 5] = -np.inf  # every score is infinity
    q[41] *= 1e30
    q[42] *= 1e-30
    with np.errstate(all="ignore"):
        want, tol = want_prefill(paged, q.reshape(136, -1), heads, starts, news, 0.01)
        got = run_prefill(ctx, paged, q.reshape(136, -1), heads, H.Attention(0.01), starts)
    rest = np.ones(136, bool)
    rest[[17, 40, 41]] = False
    K.near(got[rest], want[rest], tol[rest])
    assert not got[17].any() or np.isnan(got[17]).all()  # (zero times infinity is NaN, as in a plain product)
    assert np.isnan(got[40]).all()
    near_one = np.abs(got[41]) <= np.abs(paged.values[0]).max() * (1 + 2.0 ** -20)  # (one weight is all, whichever)
    assert near_one.all()


@pytest.mark.parametrize("type_id,kv_heads,news", [(K.F16, 32, 200), (K.F16, 2, 5), (K.F32, 2, 5)])
def test_nan_that_is_seen_shows_where_its_weight_is_nothing(ctx, type_id, kv_heads, news):
    """Among positions shared between workgroups, in a part whose scores are far below the rest."""
    rng = np.random.default_rng(42)
    paged = K.Paged(rng, type_id, 64, kv_heads, 64, [3000])
    paged.keys[0][:1000, :, 0] = -3000
    paged.keys[0][1000:, :, 0] = 0
    paged.values[0][10, :, 3] = np.nan
    for j in range(3000):
        paged.put(0, j)
    q = rng.standard_normal((news, kv_heads, 64)).astype(np.float32)
    q[:, :, 0] = 5
    got = run_prefill(ctx, paged, q.reshape(news, -1), kv_heads, H.Attention(0.125), np.array([0, news]))
    assert np.isnan(got[..., 3]).all()
    paged.values[0][10, :, 3] = 0  # (in the reference; the cache holds it still)
    want, tol = want_prefill(paged, q.reshape(news, -1), kv_heads, np.array([0, news]), [news], 0.125)
    K.near(np.delete(got, 3, -1), np.delete(want, 3, -1), np.delete(tol, 3, -1))
    if news == 5:
        got = run_decode(ctx, paged, q[0].reshape(1, -1), kv_heads, H.Attention(0.125))
        assert np.isnan(got[..., 3]).all() and np.isfinite(np.delete(got, 3, -1)).all()
