// Attention of one query per sequence over the paged cache.
#pragma once

#include "kv_common.hpp"

namespace kv {

struct DecodeArgs {
    AttnArgs a;
    float *partials;
    uint32_t *arrivals;
    uint32_t splits, head_tiles;
};

// The matrix operands of a tile of 32 positions, in either type of page. Lane l is
// column c = l % 16 (a query head) of group g = l / 16. The products run transposed,
// S^T = K q^T and O^T = V^T P, and the positions are dealt to the rows of S^T so
// that what a lane holds of it, positions 8 g + 0..7 for its head, is what it has
// to hand to the second product: the weights never leave their registers. V lies
// in the cache with a channel's positions side by side, so both operands are read
// from memory as they are used, 16 bytes a lane.
// FULL: head_dim is D; else it is less, and what lies beyond it reads as zeros.
template <typename T, int D, bool FULL> struct Tile;

template <int D, bool FULL> struct Tile<_Float16, D, FULL> {
    static constexpr int COLS = 8;        // columns 0..7 the first part of a head's q and weights, 8..15 the second
    static constexpr int KS = D / 32;     // operand pieces of a row of K
    static constexpr int DT = D / 16;     // channel tiles
    typedef f16x8 K[2][KS];
    typedef f16x8 V[DT];
    f16x8 q[KS];

    // The head's q, scaled by a power of two to a largest magnitude of about 2^13, as
    // f16 parts (22 bits of that magnitude); returns the inverse scale. What is
    // not finite goes whole into the first part.
    __device__ __forceinline__ float load_q(const float *row, uint32_t c, uint32_t g, uint32_t hd, bool live) {
        float x[KS][8], top = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t d = 32u * s + 8u * g + j;
                x[s][j] = live && d < hd ? row[d] : 0.0f;
                top = fmaxf(top, fabsf(x[s][j]));
            }
        }
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const int by = scale_bits(top);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float y = ldexpf(x[s][j], by);
                const _Float16 hi = (_Float16)y;
                const float rest = fabsf((float)hi) < INFINITY ? y - (float)hi : 0.0f;
                q[s][j] = c < 8u ? hi : (_Float16)rest;
            }
        }
        return ldexpf(1.0f, -by);
    }
    // K row of lane l in half t of the tile: position 8 (r / 4) + r % 4 + 4 t for r = l % 16
    __device__ __forceinline__ void load_k(K &k, const _Float16 *row0, uint32_t g, uint32_t hd) const {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const uint32_t d = 32u * s + 8u * g;
            const bool in = FULL || d < hd;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const f16x8 x = *(const f16x8 *)(row0 + 4u * t * (FULL ? D : hd) + (in ? d : 0u));
                k[t][s] = in ? x : f16x8{};
            }
        }
    }
    // channel 16 t + c, positions 8 g + 0..7
    __device__ __forceinline__ void load_v(V &v, const _Float16 *at, uint32_t c, uint32_t shift, uint32_t hd) const {
#pragma unroll
        for (int t = 0; t < DT; ++t) {
            const uint32_t d = 16u * t + c; // (results of channels beyond the last are not used)
            v[t] = *(const f16x8 *)(at + ((FULL ? d : min(d, hd - 1u)) << shift));
        }
    }
    __device__ __forceinline__ void scores(float (&x)[8], const K &k, uint32_t c) const {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[t][s], q[s], acc, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                // both parts of the head: columns c and c + 8 of 16. Where the key is infinite the
                // first part's infinity (or NaN) is the score, whatever the second one gives.
                const float part = c < 8u ? acc[i] : __builtin_amdgcn_fmed3f(acc[i], -3.402823466e38f, 3.402823466e38f);
                x[4 * t + i] = part + ror8(part);
            }
        }
    }
    __device__ __forceinline__ void weigh(f32x4 (&o)[DT], const V &v, const float (&w)[8], uint32_t c) const {
        f16x8 p;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const _Float16 hi = (_Float16)w[j];
            p[j] = c < 8u ? hi : (_Float16)(w[j] - (float)hi);
        }
#pragma unroll
        for (int t = 0; t < DT; ++t) {
            o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[t], p, o[t], 0, 0, 0);
        }
    }
    // positions whose bit of `mask` is not set as zeros (0 x infinity would be NaN)
    __device__ __forceinline__ void clear(V &v, uint32_t mask) const {
#pragma unroll
        for (int t = 0; t < DT; ++t) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[t][j] = (mask >> j) & 1u ? v[t][j] : (_Float16)0.0f;
            }
        }
    }
    __device__ __forceinline__ float whole(float x) const { return x + ror8(x); }
};

template <int D, bool FULL> struct Tile<float, D, FULL> {
    static constexpr int COLS = 16;
    static constexpr int KS = D / 16;
    static constexpr int DT = D / 16;
    typedef f32x4 K[2][KS];
    typedef f32x4 V[DT][2];
    f32x4 q[KS];

    __device__ __forceinline__ float load_q(const float *row, uint32_t, uint32_t g, uint32_t hd, bool live) {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t d = 16u * s + 4u * g + j;
                q[s][j] = live && d < hd ? row[d] : 0.0f;
            }
        }
        return 1.0f;
    }
    __device__ __forceinline__ void load_k(K &k, const float *row0, uint32_t g, uint32_t hd) const {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const uint32_t d = 16u * s + 4u * g;
            const bool in = FULL || d < hd;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const f32x4 x = *(const f32x4 *)(row0 + 4u * t * (FULL ? D : hd) + (in ? d : 0u));
                k[t][s] = in ? x : f32x4{};
            }
        }
    }
    __device__ __forceinline__ void load_v(V &v, const float *at, uint32_t c, uint32_t shift, uint32_t hd) const {
#pragma unroll
        for (int t = 0; t < DT; ++t) {
            const uint32_t d = 16u * t + c;
            const float *p = at + ((FULL ? d : min(d, hd - 1u)) << shift);
            v[t][0] = *(const f32x4 *)p;
            v[t][1] = *(const f32x4 *)(p + 4);
        }
    }
    __device__ __forceinline__ void scores(float (&x)[8], const K &k, uint32_t) const {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 0; s < KS; ++s) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(k[t][s][j], q[s][j], acc, 0, 0, 0);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[4 * t + i] = acc[i];
            }
        }
    }
    __device__ __forceinline__ void weigh(f32x4 (&o)[DT], const V &v, const float (&w)[8], uint32_t) const {
#pragma unroll
        for (int t = 0; t < DT; ++t) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                o[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[t][j / 4][j % 4], w[j], o[t], 0, 0, 0);
            }
        }
    }
    __device__ __forceinline__ void clear(V &v, uint32_t mask) const {
#pragma unroll
        for (int t = 0; t < DT; ++t) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[t][j / 4][j % 4] = (mask >> j) & 1u ? v[t][j / 4][j % 4] : 0.0f;
            }
        }
    }
    __device__ __forceinline__ float whole(float x) const { return x; }
};

// Partial results of the workgroups that share a sequence travel in 8-byte
// device-scope pieces, past this die's L2.
__device__ __forceinline__ void put2(float *at, float x, float y) {
    const uint64_t v = (uint64_t)__float_as_uint(x) | (uint64_t)__float_as_uint(y) << 32;
    __hip_atomic_store((uint64_t *)at, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void get2(const float *at, float &x, float &y) {
    const uint64_t v = __hip_atomic_load((const uint64_t *)at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    x = __uint_as_float((uint32_t)v);
    y = __uint_as_float((uint32_t)(v >> 32));
}

// A workgroup of four waves per key-value head, tile of its query heads, sequence
// and share of the positions; a wave takes every fourth tile of 32 positions
// straight from memory into the matrix operands. The softmax runs over one pass:
// weights are 2^(x - m + 6) with a reference m per head that follows the maximum
// only when that has moved by more than 8 (so weights stay below 2^14, exact in two
// f16 parts, and most tiles need no exchange between lanes); l and o are
// their f32 sums. The waves join in LDS, the workgroups of a sequence through
// memory: the last to arrive adds the parts up in the order of their positions.
template <typename T, int D, bool FULL, int WAVES_PER_SIMD>
__global__ __launch_bounds__(256, WAVES_PER_SIMD) void attn_decode_kernel(DecodeArgs args) {
    typedef Tile<T, D, FULL> M;
    constexpr int COLS = M::COLS, DT = M::DT, PITCH = D + 4;
    __shared__ __align__(16) float merged[4 * COLS * PITCH];
    __shared__ float stats[4][2][COLS];
    __shared__ uint32_t arrived;
    const AttnArgs &a = args.a;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t c = lane & 15u, g = lane >> 4;
    const uint32_t units = a.cache.kv_heads * args.head_tiles;
    const uint32_t seq = blockIdx.y, split = blockIdx.x / units, unit = blockIdx.x % units;
    const uint32_t kvh = unit % a.cache.kv_heads, head_tile = unit / a.cache.kv_heads;
    const uint32_t hd = FULL ? (uint32_t)D : a.cache.head_dim, shift = a.cache.page_shift;
    const uint32_t heads = min((uint32_t)COLS, a.group - head_tile * COLS); // of this tile
    const uint32_t head0 = kvh * a.group + head_tile * COLS;

    const int len = seq_len(a, seq), p = len - 1;
    int lo, hi;
    visible(a, len, seq, seq, p, lo, hi);
    const int start = lo & ~31;
    const uint32_t tiles = hi > lo ? (uint32_t)(hi - start + 31) >> 5 : 0u;
    const uint32_t per = (((tiles + args.splits - 1u) / args.splits) + 3u) & ~3u;
    const uint32_t parts = tiles > per ? (tiles + per - 1u) / per : 1u;
    if (split >= parts) {
        return;
    }
    const uint32_t t1 = min(tiles, (split + 1u) * per);

    M m;
    const uint32_t col = COLS == 8 ? c & 7u : c;
    const bool live = col < heads;
    const float unscale = m.load_q(a.q + (size_t)seq * a.q_stride + (size_t)(head0 + (live ? col : 0u)) * hd, c, g, hd, live);
    const float slope = a.slopes != nullptr && live ? a.slopes[head0 + col] * LOG2E : 0.0f;
    const float to_log2 = a.softcap > 0.0f ? a.scale * unscale / a.softcap : a.scale * unscale * LOG2E;
    const float cap_log2 = a.softcap * LOG2E;

    f32x4 o[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) {
        o[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    float top = -3.402823466e38f, l = 0.0f;

    const uint32_t *table = a.table + (size_t)seq * a.table_stride;
    const uint32_t last_entry = a.table_stride - 1u, in_page = (1u << shift) - 1u;
    const uint32_t page_elements = hd << shift;
    auto head_page = [&](uint32_t page) { return ((size_t)page * a.cache.kv_heads + kvh) * page_elements; };
    const uint32_t row = 8u * (c >> 2) + (c & 3u); // of K in the tile's first half
    for (uint32_t t = split * per + wave; t < t1; t += 4u) {
        const uint32_t base = (uint32_t)start + 32u * t;
        const uint32_t k_page = table[min((base + row) >> shift, last_entry)];
        const uint32_t v_page = table[min((base + 8u * g) >> shift, last_entry)];
        const bool known = v_page < a.cache.pages;
        typename M::K k;
        typename M::V v;
        const size_t k_at = head_page(k_page < a.cache.pages ? k_page : 0u);
        const size_t v_at = head_page(known ? v_page : 0u);
        m.load_k(k, (const T *)a.cache.k + k_at + ((base + row) & in_page) * hd, g, hd);
        m.load_v(v, (const T *)a.cache.v + v_at + ((base + 8u * g) & in_page), c, shift, hd);
        float x[8];
        m.scores(x, k, c);
        if (a.softcap > 0.0f) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[j] = cap_log2 * tanh_of(x[j] * to_log2);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[j] *= to_log2;
            }
        }
        const int at = (int)(base + 8u * g);
        if (a.slopes != nullptr) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[j] -= slope * fabsf((float)(p - at - j));
            }
        }
        if (!__all((int)base >= lo && (int)base + 32 <= hi && known)) {
            uint32_t mask = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const bool seen = known && at + j >= lo && at + j < hi;
                mask |= (seen ? 1u : 0u) << j;
                x[j] = seen ? x[j] : -INFINITY;
            }
            m.clear(v, mask);
        }
        float most = x[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) {
            most = fmaxf(most, x[j]);
        }
        if (__any(most > top + 8.0f)) {
            most = fmaxf(most, __shfl_xor(most, 16));
            most = fmaxf(most, __shfl_xor(most, 32));
            most = fmaxf(most, top);
            const float keep = exp2_of(top - most);
            top = most;
            l *= keep;
#pragma unroll
            for (int i = 0; i < DT; ++i) {
                o[i] *= keep;
            }
        }
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            w[j] = exp2_of(x[j] - top + 6.0f);
            l += w[j];
        }
        m.weigh(o, v, w, c);
    }

    // the waves' results
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
#pragma unroll
    for (int t = 0; t < DT; ++t) {
        f32x4 whole;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            whole[i] = m.whole(o[t][i]);
        }
        if (c < (uint32_t)COLS) {
            *(f32x4 *)&merged[(wave * COLS + c) * PITCH + 16u * t + 4u * g] = whole;
        }
    }
    if (g == 0u && c < (uint32_t)COLS) {
        stats[wave][0][c] = top;
        stats[wave][1][c] = l;
    }
    __syncthreads();
    const uint32_t pairs = hd / 2u; // channel pairs of a head
    const size_t part_floats = (size_t)COLS * (hd + 2u);
    const size_t slot = (size_t)seq * units + unit;
    float *mine = args.partials + (slot * args.splits + split) * part_floats;
    for (uint32_t i = threadIdx.x; i < heads * pairs; i += 256u) {
        const uint32_t h = i / pairs, d = 2u * (i % pairs);
        float best = stats[0][0][h];
#pragma unroll
        for (int w = 1; w < 4; ++w) {
            best = fmaxf(best, stats[w][0][h]);
        }
        float sum = 0.0f, y0 = 0.0f, y1 = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = exp2_of(stats[w][0][h] - best);
            sum += f * stats[w][1][h];
            y0 += f * merged[(w * COLS + h) * PITCH + d];
            y1 += f * merged[(w * COLS + h) * PITCH + d + 1u];
        }
        if (parts == 1u) {
            float *out = a.out + (size_t)seq * a.out_stride + (size_t)(head0 + h) * hd + d;
            out[0] = sum == 0.0f ? 0.0f : y0 / sum;
            out[1] = sum == 0.0f ? 0.0f : y1 / sum;
        } else {
            put2(mine + h * hd + d, y0, y1);
            if (d == 0u) {
                put2(mine + COLS * hd + 2u * h, best, sum);
            }
        }
    }
    if (parts == 1u) {
        return;
    }
    // Every wave waits until its stores are acknowledged, then the arrival is counted;
    // the loads of the last workgroup to arrive follow the count. The empty asm
    // statements keep the compiler from moving the relaxed accesses across.
    __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8)); // vmcnt(0)
    asm volatile("" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0u) {
        arrived = __hip_atomic_fetch_add(&args.arrivals[slot], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (arrived != parts - 1u) {
        return;
    }
    asm volatile("" ::: "memory");
    if (threadIdx.x == 0u) { // (zero between launches)
        __hip_atomic_store(&args.arrivals[slot], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    const float *first = args.partials + slot * args.splits * part_floats;
    float *factor = merged; // [head][part], then the sums
    float *sums = &stats[0][0][0];
    for (uint32_t h = wave; h < heads; h += 4u) {
        float best = -3.402823466e38f, sum = 0.0f;
        for (uint32_t s = lane; s < parts; s += 64u) {
            float t, n;
            get2(first + s * part_floats + COLS * hd + 2u * h, t, n);
            best = fmaxf(best, t);
        }
        for (int x = 32; x > 0; x >>= 1) {
            best = fmaxf(best, __shfl_xor(best, x));
        }
        for (uint32_t s = lane; s < parts; s += 64u) {
            float t, n;
            get2(first + s * part_floats + COLS * hd + 2u * h, t, n);
            const float f = exp2_of(t - best);
            factor[h * DECODE_MAX_SPLITS + s] = f;
            sum += f * n;
        }
        for (int x = 32; x > 0; x >>= 1) {
            sum += __shfl_xor(sum, x);
        }
        if (lane == 0u) {
            sums[h] = sum;
        }
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < heads * pairs; i += 256u) {
        const uint32_t h = i / pairs, d = 2u * (i % pairs);
        float y0 = 0.0f, y1 = 0.0f;
#pragma unroll 8
        for (uint32_t s = 0; s < parts; ++s) {
            float u0, u1;
            get2(first + s * part_floats + h * hd + d, u0, u1);
            const float f = factor[h * DECODE_MAX_SPLITS + s];
            y0 += f * u0;
            y1 += f * u1;
        }
        const float sum = sums[h];
        float *out = a.out + (size_t)seq * a.out_stride + (size_t)(head0 + h) * hd + d;
        out[0] = sum == 0.0f ? 0.0f : y0 / sum;
        out[1] = sum == 0.0f ? 0.0f : y1 / sum;
    }
}

} // namespace kv
