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
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// tanh to a few half steps relative to its value: below 1/2 its series (the first term
// left out is 5e-9 of it there), above it 1 - 2 t / (1 + t) with t = exp(-2 |y|),
// which no wave computes whose values are all small (scores well below their cap).
__device__ __forceinline__ float tanh_of(float y) {
    const float z = y * y;
    float s = -0.0014558344f;
    s = fmaf(s, z, 0.0035921280f);
    s = fmaf(s, z, -0.0088632355f);
    s = fmaf(s, z, 0.0218694885f);
    s = fmaf(s, z, -0.0539682540f);
    s = fmaf(s, z, 0.1333333333f);
    s = fmaf(s, z, -0.3333333333f);
    float r = fmaf(y * z, s, y);
    const bool large = !(fabsf(y) < 0.5f);
    if (__any(large)) {
        const float t = exp2_of(-2.0f * LOG2E * fabsf(y));
        const float u = (1.0f - t) * __builtin_amdgcn_rcpf(1.0f + t);
        r = large ? copysignf(u, y) : r;
    }
    return r;
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

} // namespace kv
