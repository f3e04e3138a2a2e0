// Penalties for repeated tokens, biases and grammar masks on rows of logits.
#pragma once

#include "kv_common.hpp"

namespace kv {

struct LogitsArgs {
    const float *x;
    float *y;
    const uint32_t *history, *history_len;
    const float *penalties;
    const uint32_t *bias_ids;
    const float *bias_values;
    const uint32_t *bias_len, *allowed;
    uint32_t vocab, history_stride, bias_stride, allowed_stride;
};

// A workgroup per row and tile of ids. It reads the row's history and bias list
// whole and keeps what falls into its tile in LDS: how often an id is in the
// history, and the last bias entry that names it (an integer maximum: the
// order of the atomics does not show). One pass over the logits, nothing in memory;
// a thread's logits are on their way while the lists are read. Bound by the
// stream of logits where there are many rows: every tile reads the lists again, so
// tiles are large there; a single row is a matter of latency, and small tiles
// spread it over the card. 64 rows of 151936 with histories of 4096, biases and allowed ids: 80 MB,
// 20.2 us = 4.0 TB/s; one row 3.2 us, which is the launch.
// SHORT: lists of fewer than 2^16 entries, whose counts and indices share a word: four workgroups of
// a large tile on a CU instead of two.
template <int TILE, int THREADS, bool SHORT>
__global__ __launch_bounds__(THREADS) void logits_adjust_kernel(LogitsArgs a) {
    constexpr int PER = TILE / THREADS; // logits of a thread, in pieces of four
    __shared__ __align__(16) uint32_t count[TILE];
    __shared__ __align__(16) uint32_t entries[SHORT ? 4 : TILE];
    uint32_t *entry = SHORT ? count : entries; // 1 + its index, 0: none (SHORT: in the upper half)
    const uint32_t row = blockIdx.y, id0 = blockIdx.x * TILE;
    const uint32_t here = min((uint32_t)TILE, a.vocab - id0);
    const float *x = a.x + (size_t)row * a.vocab + id0;
    float *y = a.y + (size_t)row * a.vocab + id0;
    // (a vocabulary that is no multiple of four leaves rows that are not aligned)
    const bool wide = here == (uint32_t)TILE && (((uintptr_t)x | (uintptr_t)y) & 15u) == 0u;
    float v[PER];
#pragma unroll
    for (int j = 0; j < PER / 4; ++j) {
        const uint32_t at = 4u * (threadIdx.x + (uint32_t)(j * THREADS));
        if (wide) {
            const f32x4 u = *(const f32x4 *)(x + at);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v[4 * j + k] = u[k];
            }
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v[4 * j + k] = at + k < here ? x[at + k] : 0.0f;
            }
        }
    }
    const bool listed = a.history != nullptr || a.bias_ids != nullptr;
    float rep = 1.0f, presence = 0.0f, frequency = 0.0f;
    if (listed) {
#pragma unroll
        for (int j = 0; j < PER / 4; ++j) {
            const uint32_t at = threadIdx.x + (uint32_t)(j * THREADS);
            ((q8::u32x4 *)count)[at] = q8::u32x4{0u, 0u, 0u, 0u};
            if constexpr (!SHORT) {
                ((q8::u32x4 *)entries)[at] = q8::u32x4{0u, 0u, 0u, 0u};
            }
        }
        __syncthreads();
        if (a.bias_ids != nullptr) { // (first: the largest index is found while the counts are zero)
            const uint32_t n = min(a.bias_len[row], a.bias_stride);
            const uint32_t *ids = a.bias_ids + (size_t)row * a.bias_stride;
            for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
                const uint32_t at = ids[i] - id0; // (below id0 wraps to a large value)
                if (at < (uint32_t)TILE) {
                    atomicMax(&entry[at], SHORT ? (i + 1u) << 16 : i + 1u);
                }
            }
            if (SHORT && a.history != nullptr) {
                __syncthreads();
            }
        }
        if (a.history != nullptr) {
            const uint32_t n = min(a.history_len[row], a.history_stride);
            const uint32_t *ids = a.history + (size_t)row * a.history_stride;
#pragma unroll 4
            for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
                const uint32_t at = ids[i] - id0;
                if (at < (uint32_t)TILE) {
                    atomicAdd(&count[at], 1u);
                }
            }
            rep = a.penalties[(size_t)row * 3u];
            presence = a.penalties[(size_t)row * 3u + 1u];
            frequency = a.penalties[(size_t)row * 3u + 2u];
        }
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < PER / 4; ++j) {
        const uint32_t at = 4u * (threadIdx.x + (uint32_t)(j * THREADS));
        uint32_t allowed = 0xfu; // (four ids of one word: id0 and `at` are multiples of four)
        if (a.allowed != nullptr && at < here) {
            const uint32_t id = id0 + at;
            allowed = a.allowed[(size_t)row * a.allowed_stride + (id >> 5)] >> (id & 31u);
        }
        if (listed) {
            q8::u32x4 c = ((const q8::u32x4 *)count)[at / 4u], e = ((const q8::u32x4 *)entry)[at / 4u];
            if constexpr (SHORT) {
                c &= 0xffffu;
                e >>= 16;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float z = v[4 * j + k];
                if (c[k] != 0u) {
                    z = z > 0.0f ? z / rep : z * rep;
                    z -= presence + frequency * (float)c[k];
                }
                if (e[k] != 0u) {
                    z += a.bias_values[(size_t)row * a.bias_stride + e[k] - 1u];
                }
                v[4 * j + k] = z;
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            v[4 * j + k] = (allowed >> k) & 1u ? v[4 * j + k] : -INFINITY;
        }
        if (wide) {
            f32x4 u;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                u[k] = v[4 * j + k];
            }
            *(f32x4 *)(y + at) = u;
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (at + k < here) {
                    y[at + k] = v[4 * j + k];
                }
            }
        }
    }
}

} // namespace kv
