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

constexpr uint32_t LOGITS_TILE = 4096; // ids a workgroup adjusts

// A workgroup per row and tile of ids. It reads the row's history and bias list
// whole and keeps what falls into its tile in LDS: how often an id is in the
// history, and the last bias entry that names it (an integer maximum: the
// order of the atomics does not show). One pass over the logits, nothing in memory.
__global__ __launch_bounds__(256) void logits_adjust_kernel(LogitsArgs a) {
    __shared__ uint32_t count[LOGITS_TILE];
    __shared__ uint32_t entry[LOGITS_TILE]; // 1 + its index, 0: none
    const uint32_t row = blockIdx.y, id0 = blockIdx.x * LOGITS_TILE;
    for (uint32_t i = threadIdx.x; i < LOGITS_TILE; i += 256u) {
        count[i] = 0u;
        entry[i] = 0u;
    }
    __syncthreads();
    float rep = 1.0f, presence = 0.0f, frequency = 0.0f;
    if (a.history != nullptr) {
        const uint32_t n = min(a.history_len[row], a.history_stride);
        const uint32_t *ids = a.history + (size_t)row * a.history_stride;
        for (uint32_t i = threadIdx.x; i < n; i += 256u) {
            const uint32_t at = ids[i] - id0; // (below id0 wraps to a large value)
            if (at < LOGITS_TILE) {
                atomicAdd(&count[at], 1u);
            }
        }
        rep = a.penalties[(size_t)row * 3u];
        presence = a.penalties[(size_t)row * 3u + 1u];
        frequency = a.penalties[(size_t)row * 3u + 2u];
    }
    if (a.bias_ids != nullptr) {
        const uint32_t n = min(a.bias_len[row], a.bias_stride);
        const uint32_t *ids = a.bias_ids + (size_t)row * a.bias_stride;
        for (uint32_t i = threadIdx.x; i < n; i += 256u) {
            const uint32_t at = ids[i] - id0;
            if (at < LOGITS_TILE) {
                atomicMax(&entry[at], i + 1u);
            }
        }
    }
    __syncthreads();
    const size_t base = (size_t)row * a.vocab;
    for (uint32_t i = threadIdx.x; i < LOGITS_TILE && i < a.vocab - id0; i += 256u) {
        const uint32_t id = id0 + i;
        float x = a.x[base + id];
        const uint32_t c = count[i], e = entry[i];
        if (c != 0u) {
            x = x > 0.0f ? x / rep : x * rep;
            x -= presence + frequency * (float)c;
        }
        if (e != 0u) {
            x += a.bias_values[(size_t)row * a.bias_stride + e - 1u];
        }
        if (a.allowed != nullptr &&
            ((a.allowed[(size_t)row * a.allowed_stride + (id >> 5)] >> (id & 31u)) & 1u) == 0u) {
            x = -INFINITY;
        }
        a.y[base + id] = x;
    }
}

} // namespace kv
