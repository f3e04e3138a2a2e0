"""References in 64 bits for the operators over the paged key-value cache and for the
logits, and the tolerances that go with them (not collected by pytest).

Tolerances count roundings. EPS is half a step of f32 relative to the value. A dot
product or sum of n f32 terms is off by a random walk of its roundings: SIGMAS *
sqrt(n) half steps of the sum of the terms' magnitudes (n of them in a row is the
bound that never happens; six deviations is what is asked here).
"""
from __future__ import annotations

import numpy as np

from tuckmill_amd import hip as H

EPS = 2.0 ** -24
SIGMAS = 6.0
F16, F32 = 1, 0
DT = {F16: np.float16, F32: np.float32}


class Paged:
    """Sequences of `lens` tokens in shuffled pages. Everything no sequence holds is
    NaN: stale pages, the rest of last pages. Table entries nobody needs are garbage."""

    def __init__(self, rng, type_id, page, kv_heads, head_dim, lens, scale=1.0, spare=2):
        self.type_id, self.page, self.kv_heads, self.head_dim = type_id, page, kv_heads, head_dim
        self.lens = np.array(lens, np.int64)
        need = [-(-int(n) // page) for n in lens]
        self.pages = max(1, sum(need) + spare)
        self.stride = max(need + [1]) + 1
        order = rng.permutation(self.pages)
        self.table = rng.integers(1 << 20, 1 << 32, (len(lens), self.stride), dtype=np.uint64).astype(np.uint32)
        self.k = np.full((self.pages, kv_heads, page, head_dim), np.nan, DT[type_id])
        self.v = np.full((self.pages, kv_heads, head_dim, page), np.nan, DT[type_id])
        self.keys, self.values = [], []  # [seq][token, head, channel] as cached
        at = 0
        for s, n in enumerate(lens):
            self.table[s, :need[s]] = order[at:at + need[s]]
            at += need[s]
            k = (rng.standard_normal((n, kv_heads, head_dim)) * scale).astype(DT[type_id])
            v = rng.standard_normal((n, kv_heads, head_dim)).astype(DT[type_id])
            self.keys.append(k)
            self.values.append(v)
            for j in range(int(n)):
                self.put(s, j)

    def put(self, s, j):
        page, place = self.table[s, j // self.page], j % self.page
        self.k[page, :, place] = self.keys[s][j]
        self.v[page, :, :, place] = self.values[s][j]

    def upload(self, ctx):
        kb, vb = ctx.buffer(self.k.nbytes), ctx.buffer(self.v.nbytes)
        kb.upload(0, self.k)
        vb.upload(0, self.v)
        return H.KvCache(kb, vb, self.type_id, self.pages, self.page, self.kv_heads, self.head_dim)


def attention(q, keys, values, p, lo, hi, scale, softcap=0.0, slopes=None, seen=None):
    """One sequence: q [row, head, channel] at positions p, row r sees lo[r] <= j < hi[r]
    (and seen[j]). Returns the result in 64 bits and how far an f32 one may be off."""
    rows, heads, d = q.shape
    n, kv_heads, _ = keys.shape
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    j = np.arange(n)
    with np.errstate(all="ignore"):
        for h in range(heads):
            k = keys[:, h // (heads // kv_heads)].astype(np.float64)
            v = values[:, h // (heads // kv_heads)].astype(np.float64)
            qh = q[:, h].astype(np.float64)
            for r in range(rows):
                vis = (j >= lo[r]) & (j < hi[r])
                if seen is not None:
                    vis &= seen
                if not vis.any():
                    continue
                x = scale * (k[vis] @ qh[r])
                e = abs(scale) * (np.abs(k[vis]) @ np.abs(qh[r])) * SIGMAS * np.sqrt(d) * EPS
                if softcap:
                    e = e + 8 * EPS * np.abs(x)  # a division, a tanh of a few half steps, a product
                    x = softcap * np.tanh(x / softcap)
                if slopes is not None:
                    b = float(slopes[h]) * np.abs(p[r] - j[vis])
                    e = e + 2 * EPS * (b + np.abs(x))
                    x = x - b
                top = x.max()
                if top == -np.inf:
                    continue
                # exp2 of (x - reference) log2 e: roundings of x, the factor and the difference
                e = e + 4 * EPS * (np.abs(x) + np.abs(x - top) + 16) + 4 * EPS
                w = np.exp(x - top)
                total = w.sum()
                out[r, h] = (w @ v[vis]) / total
                m = w.size
                # every weight off by e; both sums a walk of m terms; weights in 22 bits; the division
                each = e + SIGMAS * np.sqrt(m) * EPS * 2 + 8 * EPS
                tol[r, h] = ((w * each) @ np.abs(v[vis])) / total + np.abs(out[r, h]) * ((w * each).sum() / total)
    return out, tol


def bounds(p, length, first=None, window=0, prefix=0):
    """lo, hi of the rows at positions p (arrays)."""
    lo = np.zeros(len(p), np.int64) if first is None else np.asarray(first, np.int64)
    if window:
        lo = np.maximum(lo, p - window + 1)
    return lo, np.minimum(length, np.maximum(p + 1, prefix))


def rope(x, positions, freqs, axis, rot, adjacent):
    """x [row, head, channel] turned in 64 bits, and how far an f32 result may be off."""
    y = x.astype(np.float64).copy()
    angle = positions[np.asarray(axis)].T.astype(np.float64) * freqs.astype(np.float64)  # [row, pair]
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    a, b = (np.s_[..., 0:rot:2], np.s_[..., 1:rot:2]) if adjacent else (np.s_[..., :rot // 2], np.s_[..., rot // 2:rot])
    x0, x1 = x[a].astype(np.float64), x[b].astype(np.float64)
    y[a], y[b] = x0 * c - x1 * s, x1 * c + x0 * s
    tol = np.zeros_like(y)
    # the part of a turn to half a step of 1/2 (2 pi EPS / 2 of the angle) and 64-bit roundings of the
    # product (2^-53 of the angle, twice), cosine and sine to a few half steps, three roundings
    turn = 2 * np.pi * EPS / 2 + 2.0 ** -52 * np.abs(angle)[:, None]
    size = np.abs(x0) + np.abs(x1)
    tol[a] = tol[b] = size * (turn + 8 * EPS) + 1e-45
    return y, tol


def axis_of_pairs(sections, interleaved):
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    return [a for _, a in sorted((turn, a) for a, n in enumerate(sections) for turn in range(n))]


def adjust(x, history=None, history_len=None, penalties=None, bias_ids=None, bias_values=None,
           bias_len=None, allowed=None):
    """Rows of logits in 64 bits, and how far an f32 result may be off."""
    rows, vocab = x.shape
    y = x.astype(np.float64).copy()
    tol = np.zeros_like(y)
    with np.errstate(all="ignore"):
        for r in range(rows):
            if history is not None:
                ids = history[r, :min(int(history_len[r]), history.shape[1])]
                ids, count = np.unique(ids[ids < vocab], return_counts=True)
                rep, presence, frequency = (float(v) for v in penalties[r])
                z = y[r, ids]
                z = np.where(z > 0, z / rep, z * rep)
                cut = presence + frequency * count
                # a quotient or product, a product and a sum, a difference
                tol[r, ids] = EPS * (2 * np.abs(z) + 3 * (np.abs(presence) + np.abs(frequency) * count))
                y[r, ids] = z - cut
            if bias_ids is not None:
                last = {}
                for i in range(min(int(bias_len[r]), bias_ids.shape[1])):
                    last[int(bias_ids[r, i])] = float(bias_values[r, i])
                for i, b in last.items():
                    if i < vocab:
                        y[r, i] += b
                        tol[r, i] += EPS * (np.abs(y[r, i]) + tol[r, i]) * 1.0001
            if allowed is not None:
                on = np.unpackbits(np.ascontiguousarray(allowed[r]).view(np.uint8), bitorder="little")[:vocab]
                y[r, on == 0] = -np.inf
    return y, tol


def near(got, want, tol, what=""):
    """Every value within its tolerance; infinities and NaN where the reference has them."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN in other places"
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)]), f"{what}: infinities"
    off = np.abs(got - np.where(fine, want, 0))[fine]
    bad = off > np.broadcast_to(tol, want.shape)[fine]
    worst = float((off / np.maximum(np.broadcast_to(tol, want.shape)[fine], 1e-300)).max(initial=0))
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.size} values off, worst {worst:.3g} of the tolerance"


def u32(a):
    return np.ascontiguousarray(np.asarray(a, np.int64) & 0xffffffff, dtype=np.uint32)
