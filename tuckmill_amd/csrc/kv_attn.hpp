// Attention over the paged cache, a wave per query row and head.
#pragma once

#include "kv_common.hpp"

namespace kv {

__device__ __forceinline__ float wave_max(float x) {
    for (int m = 32; m > 0; m >>= 1) {
        x = fmaxf(x, __shfl_xor(x, m));
    }
    return x;
}
__device__ __forceinline__ float wave_sum(float x) {
    for (int m = 32; m > 0; m >>= 1) {
        x += __shfl_xor(x, m);
    }
    return x;
}

// 64 positions a step, one per lane: their scores, then the running maximum and
// sum of the softmax, then every lane's four channels of the weighted values.
template <typename T> __global__ __launch_bounds__(64) void attn_rows_kernel(AttnArgs a) {
    const uint32_t row = blockIdx.x, head = blockIdx.y, lane = threadIdx.x;
    uint32_t seq = row;
    int p, len;
    if (a.starts != nullptr) {
        seq = a.seqs;
        uint32_t r0 = 0, r1 = 0;
        for (uint32_t s = 0; s < a.seqs; ++s) {
            r0 = a.starts[s];
            r1 = a.starts[s + 1u];
            if (r0 <= row && row < r1 && r1 <= a.tokens) {
                seq = s;
                break;
            }
        }
        if (seq == a.seqs) {
            return;
        }
        len = seq_len(a, seq);
        p = len - (int)(r1 - row);
    } else {
        len = seq_len(a, seq);
        p = len - 1;
    }
    int lo, hi;
    visible(a, len, seq, row, p, lo, hi);
    const uint32_t D = a.cache.head_dim, kvh = head / a.group, shift = a.cache.page_shift;
    __shared__ float qs[256];
    __shared__ float ps[64];
    const float *q = a.q + (size_t)row * a.q_stride + head * D;
    for (uint32_t d = lane; d < D; d += 64u) {
        qs[d] = q[d];
    }
    __syncthreads();
    float m = -INFINITY, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const uint32_t *table = a.table + (size_t)seq * a.table_stride;
    for (int j0 = lo; j0 < hi; j0 += 64) {
        const int j = j0 + (int)lane;
        const uint32_t page = j < hi ? table[j >> shift] : 0xffffffffu;
        const uint32_t place = (uint32_t)j & ((1u << shift) - 1u);
        float x = -INFINITY;
        if (page < a.cache.pages) {
            const T *k = (const T *)a.cache.k + a.cache.base(page, kvh) + (size_t)place * D;
            float dot = 0.0f;
            for (uint32_t d = 0; d < D; ++d) {
                dot += qs[d] * (float)k[d];
            }
            x = dot * a.scale;
            if (a.softcap > 0.0f) {
                x = a.softcap * tanhf(x / a.softcap);
            }
            if (a.slopes != nullptr) {
                x -= a.slopes[head] * fabsf((float)(p - j));
            }
        }
        const float top = fmaxf(m, wave_max(x));
        const float base = top == -INFINITY ? 0.0f : top;
        const float w = page < a.cache.pages ? expf(x - base) : 0.0f;
        const float keep = expf(m - base);
        m = top;
        l = l * keep + wave_sum(w);
        __syncthreads();
        ps[lane] = w;
        __syncthreads();
        for (int c = 0; c < 4; ++c) {
            const uint32_t d = lane + 64u * c;
            o[c] *= keep;
            for (int i = 0; d < D && i < 64 && j0 + i < hi; ++i) {
                const uint32_t at = (uint32_t)(j0 + i), pg = table[at >> shift];
                if (pg < a.cache.pages) {
                    const T *v = (const T *)a.cache.v + a.cache.base(pg, kvh);
                    o[c] += ps[i] * (float)v[((size_t)d << shift) + (at & ((1u << shift) - 1u))];
                }
            }
        }
    }
    float *out = a.out + (size_t)row * a.out_stride + head * D;
    for (int c = 0; c < 4; ++c) {
        const uint32_t d = lane + 64u * c;
        if (d < D) {
            out[d] = l == 0.0f ? 0.0f : o[c] / l;
        }
    }
}

} // namespace kv
