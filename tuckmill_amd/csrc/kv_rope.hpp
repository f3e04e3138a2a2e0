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

constexpr uint32_t ROPE_ROWS = 16;    // rows of a workgroup
constexpr uint32_t ROPE_HEADS = 16;   // heads of q and k it turns (4, 8, 16: 49.3, 48.5, 47.0 us below)
constexpr uint32_t ROPE_CHANNELS = 256; // channels of v it stores

// Four f32 as the page's type, in one piece.
__device__ __forceinline__ void store4(float *at, f32x4 x) { *(f32x4 *)at = x; }
__device__ __forceinline__ void store4(_Float16 *at, f32x4 x) {
    typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
    *(f16x4 *)at = f16x4{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
}

// Workgroups of 16 rows: blockIdx.y names sixteen heads of q and k, or behind those 256
// channels of v. The angles of the rows are taken once per workgroup, into LDS; heads
// go four pairs a thread (WIDE: everything is aligned for 16-byte pieces). v is
// stored with a channel's places side by side, so there the lanes of a wave are rows:
// rows that follow each other in the cache make up a line between them. Bound by the
// stream of q, k and v: 4093 rows of 32 and 8 heads of 128 channels, 184 MB, 47 us = 3.9 TB/s.
template <typename T, bool WIDE> __global__ __launch_bounds__(256) void rope_store_kernel(RopeArgs a) {
    constexpr int W = WIDE ? 4 : 1;
    __shared__ float angle[2][ROPE_ROWS][128];
    __shared__ uint32_t slot_of[ROPE_ROWS]; // 0xffffffff: not stored
    const uint32_t t0 = blockIdx.x * ROPE_ROWS, rows = min(ROPE_ROWS, a.tokens - t0);
    const uint32_t half = a.rot_dim / 2u, D = a.head_dim, heads = a.q_heads + a.kv_heads;
    const uint32_t parts = (heads + ROPE_HEADS - 1u) / ROPE_HEADS;
    const uint32_t part = blockIdx.y, h0 = part * ROPE_HEADS;
    if (part >= parts || h0 + ROPE_HEADS > a.q_heads) { // (keys or values among its work)
        // of several rows that name one slot the last stores
        if (threadIdx.x < ROPE_ROWS) {
            const uint32_t slot = threadIdx.x < rows ? a.slots[t0 + threadIdx.x] : 0xffffffffu;
            slot_of[threadIdx.x] = (slot >> a.page_shift) < a.pages ? slot : 0xffffffffu;
        }
        __syncthreads();
        // (each later row is compared with all of these only if it lies between them)
        uint32_t mine[ROPE_ROWS], lowest = 0xffffffffu, highest = 0, again = 0;
#pragma unroll
        for (uint32_t r = 0; r < ROPE_ROWS; ++r) {
            mine[r] = slot_of[r];
            lowest = min(lowest, mine[r]);
            highest = mine[r] != 0xffffffffu ? max(highest, mine[r]) : highest;
        }
        for (uint32_t u0 = t0 + 1u + threadIdx.x; u0 < a.tokens; u0 += 4u * 256u) {
            uint32_t other[4];
#pragma unroll
            for (uint32_t k = 0; k < 4u; ++k) {
                other[k] = a.slots[min(u0 + 256u * k, a.tokens - 1u)];
            }
#pragma unroll
            for (uint32_t k = 0; k < 4u; ++k) {
                const uint32_t u = min(u0 + 256u * k, a.tokens - 1u);
                if (other[k] >= lowest && other[k] <= highest) {
#pragma unroll
                    for (uint32_t r = 0; r < ROPE_ROWS; ++r) {
                        again |= other[k] == mine[r] && u > t0 + r ? 1u << r : 0u;
                    }
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (uint32_t r = 0; r < ROPE_ROWS; ++r) {
            if ((again >> r) & 1u) {
                slot_of[r] = 0xffffffffu; // (whoever finds it writes the same)
            }
        }
    }
    const uint32_t in_page = (1u << a.page_shift) - 1u;
    const size_t head_page = (size_t)D << a.page_shift;
    if (part >= parts) {
        __syncthreads();
        const uint32_t r = threadIdx.x & (ROPE_ROWS - 1u), c0 = (part - parts) * ROPE_CHANNELS;
        const uint32_t slot = slot_of[r];
        if (r >= rows || slot == 0xffffffffu) {
            return;
        }
        T *to = (T *)a.v_cache + (size_t)(slot >> a.page_shift) * a.kv_heads * head_page + (slot & in_page);
        const float *v = a.v + (size_t)(t0 + r) * a.v_stride;
        const uint32_t upto = min(c0 + ROPE_CHANNELS, a.kv_heads * D);
        for (uint32_t c = c0 + W * (threadIdx.x / ROPE_ROWS); c < upto; c += W * (256u / ROPE_ROWS)) {
            float x[W];
            if constexpr (WIDE) {
                const f32x4 u = *(const f32x4 *)(v + c);
                x[0] = u[0], x[1] = u[1], x[2] = u[2], x[3] = u[3];
            } else {
                x[0] = v[c];
            }
#pragma unroll
            for (int k = 0; k < W; ++k) {
                to[(size_t)(c + k) << a.page_shift] = to_page<T>(x[k]);
            }
        }
        return;
    }
    for (uint32_t i = threadIdx.x; i < rows * half; i += 256u) {
        const uint32_t r = i / half, pair = i % half;
        turn_of(a.positions[(size_t)a.axis[pair] * a.tokens + t0 + r], a.freqs[pair], angle[0][r][pair], angle[1][r][pair]);
    }
    __syncthreads();
    const uint32_t here = min(ROPE_HEADS, heads - h0);
    const uint32_t turned = half / W, copied = (D - a.rot_dim) / W, pieces = turned + copied;
    for (uint32_t i = threadIdx.x; i < rows * here * pieces; i += 256u) {
        const uint32_t piece = i % pieces, h = h0 + i / pieces % here, r = i / pieces / here;
        const bool is_q = h < a.q_heads;
        const uint32_t kh = h - a.q_heads, slot = is_q ? 0u : slot_of[r];
        if (!is_q && slot == 0xffffffffu) {
            continue;
        }
        const float *x = is_q ? a.q + (size_t)(t0 + r) * a.q_stride + h * D : a.k + (size_t)(t0 + r) * a.k_stride + kh * D;
        float *out = a.q_out + (size_t)(t0 + r) * a.out_stride + h * D;
        T *kc = (T *)a.k_cache + ((size_t)(slot >> a.page_shift) * a.kv_heads + kh) * head_page + (size_t)(slot & in_page) * D;
        auto put = [&](uint32_t d, const float (&y)[W]) {
            if constexpr (WIDE) {
                const f32x4 u = {y[0], y[1], y[2], y[3]};
                if (is_q) {
                    *(f32x4 *)(out + d) = u;
                } else {
                    store4(kc + d, u);
                }
            } else if (is_q) {
                out[d] = y[0];
            } else {
                kc[d] = to_page<T>(y[0]);
            }
        };
        auto get = [&](uint32_t d, float (&y)[W]) {
            if constexpr (WIDE) {
                const f32x4 u = *(const f32x4 *)(x + d);
                y[0] = u[0], y[1] = u[1], y[2] = u[2], y[3] = u[3];
            } else {
                y[0] = x[d];
            }
        };
        if (piece >= turned) {
            const uint32_t d = a.rot_dim + (piece - turned) * W;
            float y[W];
            get(d, y);
            put(d, y);
            continue;
        }
        const uint32_t p0 = piece * W;
        float x0[W], x1[W], y0[W], y1[W];
        const uint32_t d0 = a.adjacent ? 2u * p0 : p0, d1 = a.adjacent ? 2u * p0 + W : p0 + half;
        get(d0, x0);
        get(d1, x1);
        if (WIDE && a.adjacent) { // eight channels in a row are four pairs
            const float u0[4] = {x0[0], x0[2 % W], x1[0], x1[2 % W]}, u1[4] = {x0[1 % W], x0[3 % W], x1[1 % W], x1[3 % W]};
#pragma unroll
            for (int k = 0; k < W; ++k) {
                x0[k] = u0[k];
                x1[k] = u1[k];
            }
        }
#pragma unroll
        for (int k = 0; k < W; ++k) {
            const float c = angle[0][r][p0 + k], s = angle[1][r][p0 + k];
            y0[k] = x0[k] * c - x1[k] * s;
            y1[k] = x1[k] * c + x0[k] * s;
        }
        if (WIDE && a.adjacent) {
            const float u0[4] = {y0[0], y1[0], y0[1 % W], y1[1 % W]}, u1[4] = {y0[2 % W], y1[2 % W], y0[3 % W], y1[3 % W]};
#pragma unroll
            for (int k = 0; k < W; ++k) {
                y0[k] = u0[k];
                y1[k] = u1[k];
            }
        }
        put(d0, y0);
        put(d1, y1);
    }
}

} // namespace kv
