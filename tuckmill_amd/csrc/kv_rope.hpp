// Rotary positions on q and k, and k, v into the paged cache.
#pragma once

#include "kv_common.hpp"

namespace kv {

struct RopeArgs {
    const float *q, *k, *v; // rows from their offsets
    float *q_out;
    void *k_cache, *v_cache;
    const uint32_t *positions, *slots;
    const float *freqs;
    uint32_t tokens, q_heads, kv_heads, head_dim, pages, page_shift;
    uint32_t q_stride, k_stride, v_stride, out_stride;
    uint32_t rot_dim, adjacent;
    uint8_t axis[128];
};

// cos and sin of position * freq: the product of a 32-bit integer and a float and
// its reduction to one turn are taken in f64 (at position 10^6 an f32 product is
// off by up to 0.06 radians), what is left of a turn is turned in f32.
__device__ __forceinline__ void turn_of(uint32_t position, float freq, float &c, float &s) {
    const double turns = (double)position * (double)freq * 0.15915494309189535;
    const float part = (float)(turns - rint(turns)); // -0.5 .. 0.5
    sincospif(2.0f * part, &s, &c);
}

template <typename T> __device__ __forceinline__ T to_page(float x);
template <> __device__ __forceinline__ float to_page<float>(float x) { return x; }
template <> __device__ __forceinline__ _Float16 to_page<_Float16>(float x) { return (_Float16)x; }

// A workgroup per row.
template <typename T> __global__ __launch_bounds__(256) void rope_store_kernel(RopeArgs a) {
    const uint32_t t = blockIdx.x;
    const uint32_t half = a.rot_dim / 2u, D = a.head_dim;
    // of several rows that name one slot the last stores
    const uint32_t slot = a.slots[t];
    bool named_later = false;
    for (uint32_t u = t + 1u + threadIdx.x; u < a.tokens; u += 256u) {
        named_later = named_later || a.slots[u] == slot;
    }
    const bool store = (slot >> a.page_shift) < a.pages && __syncthreads_or(named_later) == 0;
    T *kc = (T *)a.k_cache, *vc = (T *)a.v_cache;
    const uint32_t place = slot & ((1u << a.page_shift) - 1u);
    const size_t page = (size_t)(slot >> a.page_shift) * a.kv_heads * ((size_t)D << a.page_shift);
    auto k_at = [&](uint32_t h, uint32_t d) { return page + (((size_t)h << a.page_shift) + place) * D + d; };
    const float *q = a.q + (size_t)t * a.q_stride, *k = a.k + (size_t)t * a.k_stride;
    const float *v = a.v + (size_t)t * a.v_stride;
    float *out = a.q_out + (size_t)t * a.out_stride;
    for (uint32_t at = threadIdx.x; at < half * (a.q_heads + a.kv_heads); at += 256u) {
        const uint32_t h = at / half, i = at % half;
        const uint32_t d0 = a.adjacent ? 2u * i : i, d1 = a.adjacent ? 2u * i + 1u : i + half;
        float c, s;
        turn_of(a.positions[(size_t)a.axis[i] * a.tokens + t], a.freqs[i], c, s);
        const float *x = h < a.q_heads ? q + h * D : k + (h - a.q_heads) * D;
        const float x0 = x[d0], x1 = x[d1];
        const float y0 = x0 * c - x1 * s, y1 = x1 * c + x0 * s;
        if (h < a.q_heads) {
            out[h * D + d0] = y0;
            out[h * D + d1] = y1;
        } else if (store) {
            kc[k_at(h - a.q_heads, d0)] = to_page<T>(y0);
            kc[k_at(h - a.q_heads, d1)] = to_page<T>(y1);
        }
    }
    const uint32_t rest = D - a.rot_dim;
    for (uint32_t at = threadIdx.x; at < rest * (a.q_heads + a.kv_heads); at += 256u) {
        const uint32_t h = at / rest, d = a.rot_dim + at % rest;
        if (h < a.q_heads) {
            out[h * D + d] = q[h * D + d];
        } else if (store) {
            kc[k_at(h - a.q_heads, d)] = to_page<T>(k[(h - a.q_heads) * D + d]);
        }
    }
    for (uint32_t at = threadIdx.x; store && at < a.kv_heads * D; at += 256u) {
        vc[page + ((size_t)at << a.page_shift) + place] = to_page<T>(v[at]);
    }
}

} // namespace kv
