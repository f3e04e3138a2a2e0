// What the kernels over the paged key-value cache share (gfx950, wave64): the
// cache's layout, the visible range of a query and the arguments of the two
// attention kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <hip/hip_ext.h>
#include <stdint.h>

#include "kv_plan.hpp"
#include "q8_common.hpp"

namespace kv {

constexpr float LOG2E = 1.4426950408889634f;

typedef q8::f32x4 f32x4;
typedef f32x4 f32x4_unaligned __attribute__((aligned(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// x = cap * tanh(x) for a lane's scores (x = score / cap; cap in units of log2 e), tanh
// to a few half steps relative to its value: its series below 1/2 (the first term left
// out is 9.7e-9 of tanh there, a sixth of a half step) and below 1/4 (8.6e-9, five terms);
// above, (1 - t) / (1 + t) with t = exp(-2 |x|). The ways are chosen for the wave: scores are mostly well below their cap.
template <int N> __device__ __forceinline__ void cap_of(float (&x)[N], float cap) {
    float most = 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        most = fmaxf(most, fabsf(x[j]));
    }
    if (__all(most < 0.25f)) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float z = x[j] * x[j];
            float s = 0.0218694885f;
            s = fmaf(s, z, -0.0539682540f);
            s = fmaf(s, z, 0.1333333333f);
            s = fmaf(s, z, -0.3333333333f);
            x[j] = cap * fmaf(x[j] * z, s, x[j]);
        }
        return;
    }
    const bool small = __all(most < 0.5f);
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const float z = x[j] * x[j];
        float s = -0.0014558344f;
        s = fmaf(s, z, 0.0035921280f);
        s = fmaf(s, z, -0.0088632355f);
        s = fmaf(s, z, 0.0218694885f);
        s = fmaf(s, z, -0.0539682540f);
        s = fmaf(s, z, 0.1333333333f);
        s = fmaf(s, z, -0.3333333333f);
        const float series = fmaf(x[j] * z, s, x[j]);
        if (!small) {
            const float t = exp2_of(-2.0f * LOG2E * fabsf(x[j]));
            const float u = copysignf((1.0f - t) * __builtin_amdgcn_rcpf(1.0f + t), x[j]);
            x[j] = cap * (fabsf(x[j]) < 0.5f ? series : u);
        } else {
            x[j] = cap * series;
        }
    }
}

// What a dot product is multiplied by: to a score in units of the cap, or of log2 e. (Finite for
// a cap of next to nothing too, or a dot product of zero would become NaN.)
__device__ __forceinline__ float score_factor(float scale, float cap) {
    const float by = cap > 0.0f ? scale / cap : scale * LOG2E;
    return __builtin_amdgcn_fmed3f(by, -3.402823466e38f, 3.402823466e38f);
}

// The power of two that brings a largest magnitude to about 2^13 (none where it is not
// finite), at which two f16 parts hold 22 bits of it without overflow.
__device__ __forceinline__ int scale_bits(float top) {
    const int by = top < INFINITY ? 13 - (int)((__float_as_uint(top) >> 23) & 0xffu) + 127 : 0;
    return by < 100 ? by : 100;
}

// The value of the lane eight columns on, of sixteen.
__device__ __forceinline__ float ror8(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x128, 0xf, 0xf, false));
}

// The cache: k [page][kv_head][place][channel], v [page][kv_head][channel][place].
struct Cache {
    const void *k, *v;
    uint32_t pages, page_shift, kv_heads, head_dim;
    // elements of one page of one head
    __device__ __forceinline__ size_t head_page() const { return (size_t)head_dim << page_shift; }
    // first element of a page of a head, in either buffer
    __device__ __forceinline__ size_t base(uint32_t page, uint32_t head) const {
        return ((size_t)page * kv_heads + head) * head_page();
    }
};

struct AttnArgs {
    Cache cache;
    const float *q; // rows from their offset
    float *out;
    const uint32_t *table, *lens, *starts; // starts: null, one row per sequence
    const float *slopes;
    const uint32_t *first, *prefix;
    uint32_t tokens, seqs, q_heads, group, table_stride, q_stride, out_stride, window;
    float scale, softcap;
};

// Cached tokens of a sequence, cut at what its table can name.
__device__ __forceinline__ int seq_len(const AttnArgs &a, uint32_t seq) {
    const uint32_t most = a.table_stride << a.cache.page_shift;
    const uint32_t len = a.lens[seq];
    return (int)(len < most ? len : most);
}

// The positions lo <= j < hi that the query at position p sees.
__device__ __forceinline__ void visible(const AttnArgs &a, int len, uint32_t seq, uint32_t row, int p,
                                        int &lo, int &hi) {
    const uint32_t first = a.first != nullptr ? a.first[row] : 0u;
    lo = first < (uint32_t)len ? (int)first : len;
    if (a.window != 0u && p >= 0 && a.window <= (uint32_t)p) {
        const int from = p - (int)a.window + 1;
        lo = from > lo ? from : lo;
    }
    hi = p + 1;
    if (a.prefix != nullptr) {
        const uint32_t prefix = a.prefix[seq];
        const int both = prefix < (uint32_t)len ? (int)prefix : len;
        hi = both > hi ? both : hi;
    }
    hi = hi < len ? hi : len;
}

// The smallest and the largest of a row of 16 lanes, in all of them; and of the wave, as a scalar.
template <int N> __device__ __forceinline__ int ror(int x) {
    return __builtin_amdgcn_update_dpp(0, x, 0x120 + N, 0xf, 0xf, false);
}
__device__ __forceinline__ int least16(int x) {
    x = min(x, ror<8>(x));
    x = min(x, ror<4>(x));
    x = min(x, ror<2>(x));
    return min(x, ror<1>(x));
}
__device__ __forceinline__ int most16(int x) {
    x = max(x, ror<8>(x));
    x = max(x, ror<4>(x));
    x = max(x, ror<2>(x));
    return max(x, ror<1>(x));
}
__device__ __forceinline__ int least64(int x) {
    x = least16(x);
    return min(min(__builtin_amdgcn_readlane(x, 0), __builtin_amdgcn_readlane(x, 16)),
               min(__builtin_amdgcn_readlane(x, 32), __builtin_amdgcn_readlane(x, 48)));
}
__device__ __forceinline__ int most64(int x) {
    x = most16(x);
    return max(max(__builtin_amdgcn_readlane(x, 0), __builtin_amdgcn_readlane(x, 16)),
               max(__builtin_amdgcn_readlane(x, 32), __builtin_amdgcn_readlane(x, 48)));
}

// Sums and maxima over the lanes up to each, within rows of 16 and then from row to row.
template <int CONTROL, int ROWS> __device__ __forceinline__ uint32_t moved(uint32_t x) { // 0 where nothing comes from
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CONTROL, ROWS, 0xf, false);
}
template <int CONTROL, int ROWS> __device__ __forceinline__ uint64_t moved(uint64_t x) {
    return (uint64_t)moved<CONTROL, ROWS>((uint32_t)(x >> 32)) << 32 | moved<CONTROL, ROWS>((uint32_t)x);
}
template <typename U, typename OP> __device__ __forceinline__ U over_lanes(U x, OP op) {
    x = op(x, moved<0x111, 0xf>(x)); // from 1, 2, 4 and 8 lanes before
    x = op(x, moved<0x112, 0xf>(x));
    x = op(x, moved<0x114, 0xf>(x));
    x = op(x, moved<0x118, 0xf>(x));
    x = op(x, moved<0x142, 0xa>(x)); // from the end of the row before, to the second and fourth
    return op(x, moved<0x143, 0xc>(x)); // from the end of the second, to the third and fourth
}
template <typename U> __device__ __forceinline__ U sum_over_lanes(U x) {
    return over_lanes(x, [](U a, U b) { return a + b; });
}
__device__ __forceinline__ uint32_t last_of(uint32_t x) { return (uint32_t)__builtin_amdgcn_readlane((int)x, 63); }
__device__ __forceinline__ uint64_t last_of(uint64_t x) {
    return (uint64_t)last_of((uint32_t)(x >> 32)) << 32 | last_of((uint32_t)x);
}

// Rows of sequence s0 + lane of a ragged batch, for a wave that goes through the sequences 64
// at a time, and the first of them (`highest`: of the bounds before). A sequence has rows where its bounds ascend
// within the batch and no earlier bound is above its first, so that no two sequences share
// one.
__device__ __forceinline__ uint32_t rows_of(const AttnArgs &a, uint32_t s0, uint32_t &highest, uint32_t &first) {
    const uint32_t lane = threadIdx.x & 63u, s = min(s0 + lane, a.seqs - 1u);
    const uint32_t r0 = a.starts[s], r1 = a.starts[s + 1u];
    first = r0;
    const uint32_t above = max(over_lanes(r0, [](uint32_t x, uint32_t y) { return max(x, y); }), highest);
    highest = last_of(above);
    return s0 + lane < a.seqs && r0 == above && r0 <= r1 && r1 <= a.tokens ? r1 - r0 : 0u;
}

// The index-th tile of the batch's rows (a query and a head of the key-value head's
// group each), the sequences' tiles one after the other and taken from the last (which
// has the most positions to see) to the first. Returns the tile's number, or 0xffffffff. Every
// wave looks for itself, 64 sequences a step.
__device__ __forceinline__ uint32_t find_tile(const AttnArgs &a, uint32_t tile_rows, uint32_t index, uint32_t &seq,
                                              uint32_t &tile, uint32_t &row0, uint32_t &rows) {
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t want = 0;
    seq = tile = row0 = rows = 0;
    uint32_t first = 0, n = 0, mine = 0, upto = 0;
    for (int pass = 0; pass < 2; ++pass) {
        uint32_t before = 0, highest = 0;
        bool here = false;
        for (uint32_t s0 = 0; s0 < a.seqs && !here; s0 += 64u) {
            if (pass == 0 || a.seqs > 64u) {
                n = rows_of(a, s0, highest, first) * a.group;
                mine = (n + tile_rows - 1u) / tile_rows;
                upto = sum_over_lanes(mine);
            }
            if (pass == 1) {
                const uint64_t found = __ballot(want < before + upto);
                if (found != 0ull) {
                    const int at = __builtin_ctzll(found);
                    seq = s0 + (uint32_t)at;
                    tile = want - before - (__shfl(upto, at) - __shfl(mine, at));
                    row0 = __shfl(first, at);
                    rows = __shfl(n, at);
                    here = true;
                }
            }
            before += last_of(upto);
        }
        if (pass == 0) {
            if (index >= before) {
                return 0xffffffffu;
            }
            want = before - 1u - index;
        }
    }
    seq = __builtin_amdgcn_readfirstlane(seq);
    tile = __builtin_amdgcn_readfirstlane(tile);
    row0 = __builtin_amdgcn_readfirstlane(row0);
    rows = __builtin_amdgcn_readfirstlane(rows);
    return want;
}

} // namespace kv
