// Attention of ragged batches of many query rows over a paged cache of f16.
#pragma once

#include "kv_attn_decode.hpp"

namespace kv {

struct PrefillArgs {
    AttnArgs a;
    float *partials;
    uint32_t *arrivals;
    uint32_t splits, tile_bound;
};

// Sizes of the kernel for heads of up to D channels. A row is a query and a head; heads of one
// key-value head that belong to the same query are neighbours, so a tile of rows reads its
// keys and values once for all of them.
template <int D> struct PrefillShape {
    static constexpr int E = 8;                  // elements of a 16-byte unit
    static constexpr int N = 64;                 // positions of a step
    static constexpr int SUB = N / 32;           // tiles of scores
    static constexpr int UK = D / E;             // units of a key
    static constexpr int KS = UK / 2;            // operand pieces of a key
    static constexpr int DT = D / 32;            // channel tiles
    static constexpr int BYTES = N * D * 2;      // of a step's keys, and of its values
    static constexpr int FETCHES = BYTES / 1024 / 4; // a wave's, of either
    static constexpr int SWIZZLE = UK < 16 ? UK - 1 : 15;
};

constexpr uint32_t ASIDE = 32; // steps that a wave puts aside; where there are more it goes through all again

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// How a row's q is held, the products and how weights enter the second one.
template <int D, bool FULL> struct Rows {
    typedef PrefillShape<D> S;
    typedef f16x8 Unit;
    Unit hi[S::KS], lo[S::KS]; // q in two parts (22 bits of the row's largest magnitude)

    // (a lane without a row is given one that is there: its results are not used)
    __device__ __forceinline__ float load_q(const float *row, uint32_t h, uint32_t hd, float minus) {
        float top = 0.0f;
        auto read = [&](float (&x)[8], int s) {
            const uint32_t d = 8u * (2u * s + h);
            const float *from = row + (FULL || d < hd ? d : 0u);
            const f32x4 y[2] = {*(const f32x4_unaligned *)from, *(const f32x4_unaligned *)(from + 4)};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[j] = FULL || d < hd ? y[j / 4][j % 4] : 0.0f;
            }
        };
#pragma unroll
        for (int s = 0; s < S::KS; ++s) {
            float x[8];
            read(x, s);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                top = fmaxf(top, fabsf(x[j]));
            }
        }
        top = fmaxf(top, __shfl_xor(top, 32));
        const int by = scale_bits(top);
        const float scale = ldexpf(1.0f, by);
        const bool finite = top < INFINITY; // (what is not goes whole into the first part)
#pragma unroll
        for (int s = 0; s < S::KS; ++s) {
            float x[8];
            read(x, s);
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const f32x2 y = {x[j] * scale, x[j + 1] * scale};
                const f16x2 first = __builtin_convertvector(y, f16x2);
                const f32x2 rest = {finite ? fmaf((float)first[0], minus, y[0]) : 0.0f,
                                    finite ? fmaf((float)first[1], minus, y[1]) : 0.0f};
                const f16x2 second = __builtin_convertvector(rest, f16x2);
                hi[s][j] = first[0];
                hi[s][j + 1] = first[1];
                lo[s][j] = second[0];
                lo[s][j + 1] = second[1];
            }
        }
        return ldexpf(1.0f, -by);
    }
    __device__ __forceinline__ f32x16 score(f32x16 acc, const Unit &k, int s) const {
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, hi[s], acc, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(k, lo[s], acc, 0, 0, 0);
    }
    static constexpr int PIECES = S::N / 16; // of the weights: 16 positions each
    struct Weights {
        Unit hi, lo;
    };
    static __device__ __forceinline__ Weights pack(const float (&x)[S::SUB][16], int i, float minus) {
        Weights w;
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const float *y = &x[i / 2][(i % 2) * 8 + j];
            const f16x2 hi = __builtin_convertvector((f32x2{y[0], y[1]}), f16x2);
            // (y - hi, which is exact: one instruction that takes the f16 where it is, if the
            // compiler does not know that `minus` is -1)
            const f32x2 rest = {fmaf((float)hi[0], minus, y[0]), fmaf((float)hi[1], minus, y[1])};
            const f16x2 lo = __builtin_convertvector(rest, f16x2);
            w.hi[j] = hi[0];
            w.hi[j + 1] = hi[1];
            w.lo[j] = lo[0];
            w.lo[j + 1] = lo[1];
        }
        return w;
    }
    static __device__ __forceinline__ f32x16 weigh(f32x16 acc, const Unit &v, const Weights &w) {
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, w.hi, acc, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(v, w.lo, acc, 0, 0, 0);
    }
};

// A workgroup of four waves per key-value head, tile of 128 rows and share of the
// positions; each wave has 32 rows and reads the step's keys and values from LDS,
// where the four fetch them straight from the pages, a step ahead. The products run
// transposed like the decode kernel's, S^T = K q^T in 32 x 32 tiles whose rows the
// positions are dealt to (row 8 a + 4 h + b of a tile is position
// 16 (a / 2) + 8 h + 4 (a % 2) + b) such that a lane holds of S^T what it hands to O^T = V^T P.
// In LDS the 16-byte units of a row are swapped by exclusive or with the row's number,
// which spreads a column of units over the banks.
// Bound by the matrix cores where rows are many: a prompt of 8192, 32 heads of 128 channels,
// 960 us = 575 TFLOP/s (1150 with both parts of q and of the weights counted). 4001 rows of packed
// documents of 64 channels with bias and cap 55 us: vector instructions, 18 a score, keep a SIMD busy for
// 42% of it; the rest is that tiles have 1 to 13 steps, six on average, and are all there at once, so
// that some CUs end early, and how each begins and ends.
template <int D, bool FULL, int WAVES_PER_SIMD>
__global__ __launch_bounds__(256, WAVES_PER_SIMD) void attn_prefill_kernel(PrefillArgs args) {
    typedef _Float16 T;
    typedef PrefillShape<D> S;
    typedef Rows<D, FULL> R;
    typedef typename R::Unit Unit;
    extern __shared__ __align__(1024) uint8_t lds[]; // two stages of keys and values
    __shared__ int range[4][2];
    __shared__ uint32_t arrived, cleaned, aside[4][ASIDE];
    __shared__ float factor[PREFILL_MAX_SPLITS][128];
    const AttnArgs &a = args.a;
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t c = lane & 31u, h = lane >> 5;
    const uint32_t stages = lds_address(lds); // (a multiple of a row of units)
    const uint32_t kvh = blockIdx.x % a.cache.kv_heads, rest = blockIdx.x / a.cache.kv_heads;
    const uint32_t split = rest % args.splits, index = rest / args.splits;
    const uint32_t hd = FULL ? (uint32_t)D : a.cache.head_dim, shift = a.cache.page_shift;

    uint32_t seq, tile, row0, rows;
    const uint32_t want = find_tile(a, PREFILL_ROWS, index, seq, tile, row0, rows);
    if (want == 0xffffffffu) {
        return;
    }

    // this lane's row
    const int len = seq_len(a, seq), n = (int)(rows / a.group);
    const uint32_t r = tile * 128u + wave * 32u + c;
    const bool live = r < rows;
    const uint32_t query = live ? r / a.group : 0u, head = kvh * a.group + (live ? r % a.group : 0u);
    const uint32_t row = row0 + query;
    const int p = len - n + (int)query;
    int lo = 0, hi = 0;
    if (live) {
        visible(a, len, seq, row, p, lo, hi);
    }
    // What any row of the wave sees, and what all of them see. (Rows that are not
    // there may be given anything.)
    const bool sees = live && lo < hi;
    int any_lo = sees ? lo : 0x7fffffff, any_hi = sees ? hi : 0, all_lo = live ? lo : 0, all_hi = live ? hi : 0x7fffffff;
    any_lo = least64(any_lo);
    any_hi = most64(any_hi);
    all_lo = most64(all_lo);
    all_hi = least64(all_hi);
    if (threadIdx.x == 0u) {
        cleaned = 0u;
    }
    if (lane == 0u) {
        range[wave][0] = any_lo;
        range[wave][1] = any_hi;
    }
    __syncthreads();
    const int from = min(min(range[0][0], range[1][0]), min(range[2][0], range[3][0]));
    const int upto = max(max(range[0][1], range[1][1]), max(range[2][1], range[3][1]));
    const uint32_t start = __builtin_amdgcn_readfirstlane(from < upto ? (uint32_t)from & ~(uint32_t)(S::N - 1) : 0u);
    const uint32_t steps = __builtin_amdgcn_readfirstlane(from < upto ? ((uint32_t)upto - start + S::N - 1u) / S::N : 0u);
    const uint32_t shares = max(min(args.splits, steps / PREFILL_MIN_STEPS), 1u), per = (steps + shares - 1u) / shares;
    const uint32_t parts = steps != 0u ? (steps + per - 1u) / per : 1u;
    if (split >= parts) {
        return;
    }
    const uint32_t s_begin = split * per, s_end = min(steps, s_begin + per);

    // Pages of a step: one for every 16 positions.
    constexpr int PAGES = S::N / 16;
    const __attribute__((address_space(4))) uint32_t *table =
        (const __attribute__((address_space(4))) uint32_t *)(a.table + (size_t)seq * a.table_stride);
    const uint32_t last_entry = a.table_stride - 1u, in_page = (1u << shift) - 1u;
    const uint32_t page_elements = hd << shift;
    uint32_t pages[PAGES], next_pages[PAGES];
    auto look_up = [&](uint32_t step) {
        const uint32_t base = start + step * S::N;
#pragma unroll
        for (int i = 0; i < PAGES; ++i) {
            next_pages[i] = table[min((base + 16u * i) >> shift, last_entry)];
        }
    };
    // Fetch a step: a wave's keys lie within 16 positions, a lane's values within one unit.
    const uint32_t v_at = ((lane & 7u) ^ (lane >> 3)) * S::E;
    auto fetch = [&](uint32_t step, uint32_t stage) {
        const uint32_t base = start + step * S::N;
        uint8_t *k_lds = lds + stage * (2u * S::BYTES) + wave * (S::FETCHES * 1024u);
        uint8_t *v_lds = k_lds + S::BYTES;
        uint32_t k_page = next_pages[0], v_page = next_pages[0];
#pragma unroll
        for (int i = 1; i < PAGES; ++i) {
            k_page = (wave * (S::N / 4u)) >> 4 == (uint32_t)i ? next_pages[i] : k_page;
            v_page = v_at >> 4 == (uint32_t)i ? next_pages[i] : v_page;
        }
        k_page = k_page < a.cache.pages ? k_page : 0u; // (not seen by any row; somewhere to read from)
        v_page = v_page < a.cache.pages ? v_page : 0u;
        const T *k = (const T *)a.cache.k + ((size_t)k_page * a.cache.kv_heads + kvh) * page_elements;
        const T *v = (const T *)a.cache.v + ((size_t)v_page * a.cache.kv_heads + kvh) * page_elements +
                     ((base + v_at) & in_page);
#pragma unroll
        for (int f = 0; f < S::FETCHES; ++f) {
            const uint32_t i = wave * S::FETCHES + f;
            const uint32_t at = i * (64u / S::UK) + lane / S::UK; // row of the stage
            const uint32_t unit = (lane % S::UK) ^ (at & S::SWIZZLE);
            const uint32_t position = (at & ~12u) | (at & 4u) << 1 | (at & 8u) >> 1;
            const uint32_t d = unit * S::E;
            fetch16(k + ((base + position) & in_page) * hd + (FULL || d < hd ? d : 0u), lds_address(k_lds) + f * 1024);
        }
#pragma unroll
        for (int f = 0; f < S::FETCHES; ++f) {
            const uint32_t d = (wave * S::FETCHES + f) * 8u + (lane >> 3);
            fetch16(v + ((FULL ? d : min(d, hd - 1u)) << shift), lds_address(v_lds) + f * 1024);
        }
    };

    if (s_begin < s_end) { // (on its way while the rows' q are taken apart)
        look_up(s_begin);
        fetch(s_begin, 0u);
    }
    float minus = -1.0f;
    asm("" : "+s"(minus));
    R q;
    const float unscale = q.load_q(a.q + (size_t)row * a.q_stride + (size_t)head * hd, h, hd, minus);
    const float slope = a.slopes != nullptr ? a.slopes[head] * LOG2E : 0.0f;
    const float to_log2 = score_factor(a.scale * unscale, a.softcap);
    const float cap_log2 = a.softcap * LOG2E;

    f32x16 o[S::DT];
#pragma unroll
    for (int t = 0; t < S::DT; ++t) {
#pragma unroll
        for (int v = 0; v < 16; ++v) {
            o[t][v] = 0.0f;
        }
    }
    float top = -3.402823466e38f, l = 0.0f;
    uint32_t asides = 0; // steps put aside
    for (uint32_t step = s_begin; step < s_end; ++step) {
#pragma unroll
        for (int i = 0; i < PAGES; ++i) {
            pages[i] = next_pages[i];
        }
        if (step + 1u < s_end) {
            look_up(step + 1u);
        }
        // This wave's fetches have landed and its reads of the other stage are done;
        // behind the barrier everybody's.
        __builtin_amdgcn_s_waitcnt(7 << 4); // vmcnt(0) lgkmcnt(0)
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const uint32_t stage = (step - s_begin) & 1u;
        if (step + 1u < s_end) {
            fetch(step + 1u, stage ^ 1u);
        }
        const int base = (int)(start + step * S::N);
        if (base >= any_hi || base + S::N <= any_lo) {
            continue; // nothing for this wave's rows
        }
        f32x16 acc[S::SUB];
#pragma unroll
        for (int b = 0; b < S::SUB; ++b) {
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                acc[b][v] = 0.0f;
            }
        }
        // (each piece's reads stand before the products of the one in front of it and no
        // earlier: left alone, the compiler reads everything first and spills)
        // A unit's address is its row's, with the bits of the unit that the lane and the piece
        // give exchanged for one another's exclusive or: one instruction each, where addresses kept
        // from step to step would take the registers of 16 bytes a lane for every piece.
        typedef const __attribute__((address_space(3))) Unit *Lds;
        const uint32_t k_at = stages + stage * (2u * S::BYTES) + (c * S::UK + (h ^ (c & S::SWIZZLE))) * 16u;
        const uint32_t v_row = stages + stage * (2u * S::BYTES) + S::BYTES + (c * 8u + (h ^ (c & 7u))) * 16u;
        Unit k_next[S::SUB];
        auto read_k = [&](int s) {
#pragma unroll
            for (int b = 0; b < S::SUB; ++b) {
                const Unit k = *(Lds)((k_at ^ (32u * s)) + b * (32u * S::UK * 16u));
                k_next[b] = !FULL && (2u * s + h) * S::E >= hd ? Unit{} : k;
            }
        };
        // (the matrix cores first: the other wave of the SIMD has its scores to see to; a prompt of 8192
        // 965 -> 942 us)
        __builtin_amdgcn_s_setprio(1);
        read_k(0);
#pragma unroll
        for (int s = 0; s < S::KS; ++s) {
            Unit k[S::SUB];
#pragma unroll
            for (int b = 0; b < S::SUB; ++b) {
                k[b] = k_next[b];
            }
            asm volatile("" ::: "memory");
            if (s + 1 < S::KS) {
                read_k(s + 1);
            }
#pragma unroll
            for (int b = 0; b < S::SUB; ++b) {
                acc[b] = q.score(acc[b], k[b], s);
            }
        }
        __builtin_amdgcn_s_setprio(0);
        float x[S::SUB][16];
        const int mine = base + 8 * (int)h; // position of value v of tile b: mine + 32 b + 16 (v / 8) + v % 8
#pragma unroll
        for (int b = 0; b < S::SUB; ++b) {
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                x[b][v] = acc[b][v] * to_log2;
            }
            if (a.softcap > 0.0f) {
                cap_of(x[b], cap_log2);
            }
        }
        if (a.slopes != nullptr) {
            const float from = (float)(mine - p);
#pragma unroll
            for (int b = 0; b < S::SUB; ++b) {
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    x[b][v] = fmaf(-slope, fabsf(from + (float)(32 * b + 16 * (v / 8) + v % 8)), x[b][v]);
                }
            }
        }
        bool known = true;
#pragma unroll
        for (int i = 0; i < PAGES; ++i) {
            known = known && pages[i] < a.cache.pages;
        }
        const bool whole = known && base >= all_lo && base + S::N <= all_hi;
        if (!whole) {
            const uint32_t first = (uint32_t)(lo - mine), count = lo < hi ? (uint32_t)(hi - lo) : 0u;
#pragma unroll
            for (int i = 0; i < PAGES; ++i) {
                const uint32_t some = pages[i] < a.cache.pages ? count : 0u;
#pragma unroll
                for (int v = 0; v < 8; ++v) {
                    float &y = x[i / 2][8 * (i % 2) + v];
                    y = 16u * i + v - first < some ? y : -INFINITY;
                }
            }
        }
        float most = x[0][0]; // or NaN, which any of them hands on
#pragma unroll
        for (int b = 0; b < S::SUB; ++b) {
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                most = __builtin_elementwise_maximum(most, x[b][v]);
            }
        }
        if (__any(!(most <= top + 14.0f))) {
            if (__any(most != most)) {
                // A score may be NaN that should be an infinity: the two parts of q share a sum, and an infinite
                // key meets each with a sign of its own, or as a zero. The step is put aside for the wave, to
                // be gone through in f32 after the loop, unless only rows have it that are NaN anyway: of a q
                // that is not finite, or a score of infinity.
                Unit odd = {};
#pragma unroll
                for (int i = 0; i < S::KS; ++i) {
                    odd = __builtin_elementwise_fma(q.hi[i], Unit{}, odd);
                }
                bool lost = l != l || !(top < INFINITY);
#pragma unroll
                for (int j = 0; j < S::E; ++j) {
                    lost = lost || odd[j] != (T)0.0f;
                }
                lost = __shfl_xor((int)lost, 32) != 0 || lost;
                if (__any(most != most && !lost)) {
                    if (lane == 0u) {
                        aside[wave][asides % ASIDE] = step;
                    }
                    ++asides;
                    l = lost ? NAN : l;
                    most = -INFINITY;
#pragma unroll
                    for (int b = 0; b < S::SUB; ++b) {
#pragma unroll
                        for (int v = 0; v < 16; ++v) {
                            x[b][v] = -INFINITY;
                        }
                    }
                }
            }
            most = fmaxf(most, __shfl_xor(most, 32));
            most = fmaxf(most - 6.0f, top);
            const float keep = exp2_of(top - most);
            top = most;
            l *= keep;
#pragma unroll
            for (int t = 0; t < S::DT; ++t) {
                o[t] *= keep;
            }
        }
#pragma unroll
        for (int b = 0; b < S::SUB; ++b) {
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                x[b][v] = exp2_of(x[b][v] - top);
                l += x[b][v];
            }
        }
        auto v_of = [&](int t, int i) { return (v_row ^ (32u * i)) + t * (32u * 128u); };
        if (!whole) {
            // A value that is not finite must not reach a row that does not see it through
            // a weight of zero: it becomes zero in the stage (where the other waves may have
            // read it before or not), and after the loop the rows that see it are told.
            Unit bad = {};
#pragma unroll
            for (int t = 0; t < S::DT; ++t) {
#pragma unroll
                for (int i = 0; i < R::PIECES; ++i) {
                    asm volatile("" ::: "memory");
                    bad = __builtin_elementwise_fma(*(Lds)v_of(t, i), Unit{}, bad);
                }
            }
            bool any = false;
#pragma unroll
            for (int j = 0; j < S::E; ++j) {
                any = any || bad[j] != (T)0.0f;
            }
            if (__any(any)) {
                // (only what some row of the workgroup sees is worth telling: places behind the
                // sequence or in a page that is not there hold anything)
                const int seen_lo = min(min(range[0][0], range[1][0]), min(range[2][0], range[3][0])) - mine;
                const int seen_hi = max(max(range[0][1], range[1][1]), max(range[2][1], range[3][1])) - mine;
                uint32_t there = 0;
#pragma unroll
                for (int i = 0; i < PAGES; ++i) {
                    there |= pages[i] < a.cache.pages ? 1u << i : 0u;
                }
                uint32_t tell = 0;
#pragma unroll 1
                for (int t = 0; t < S::DT; ++t) {
#pragma unroll 1
                    for (int i = 0; i < R::PIECES; ++i) {
                        Unit v = *(Lds)v_of(t, i);
                        uint32_t wrong = 0;
#pragma unroll
                        for (int j = 0; j < S::E; ++j) {
                            const bool finite = fabsf((float)v[j]) < INFINITY;
                            wrong |= finite ? 0u : 1u << j;
                            v[j] = finite ? v[j] : (T)0.0f;
                        }
                        *(__attribute__((address_space(3))) Unit *)v_of(t, i) = v;
                        const int first = min(max(seen_lo - 16 * i, 0), S::E), last = min(max(seen_hi - 16 * i, first), S::E);
                        tell |= (there >> i & 1u) != 0u ? wrong & ((1u << last) - (1u << first)) : 0u;
                    }
                }
                if (__any(tell != 0u) && lane == 0u) {
                    cleaned = 1u;
                }
            }
        }
        __builtin_amdgcn_s_setprio(1);
        Unit v_next = *(Lds)v_of(0, 0);
#pragma unroll
        for (int i = 0; i < R::PIECES; ++i) {
            const typename R::Weights w = R::pack(x, i, minus);
#pragma unroll
            for (int t = 0; t < S::DT; ++t) {
                const Unit v = v_next;
                asm volatile("" ::: "memory");
                if (i * S::DT + t + 1 < R::PIECES * S::DT) {
                    v_next = *(Lds)v_of((t + 1) % S::DT, i + (t + 1) / S::DT);
                }
                o[t] = R::weigh(o[t], v, w);
            }
        }
        __builtin_amdgcn_s_setprio(0);
    }
    l += __shfl_xor(l, 32);
    __syncthreads();
    if (cleaned != 0u) {
        // Rare, and as slow as it looks: every value that a row of the wave sees.
        for (uint32_t step = s_begin; step < s_end; ++step) {
            const int base = (int)(start + step * S::N);
            bool finite = true;
            for (uint32_t i = lane; i < hd * S::N; i += 64u) {
                const uint32_t at = (uint32_t)base + i % S::N, page = table[min(at >> shift, last_entry)];
                const T *v = (const T *)a.cache.v + ((size_t)(page < a.cache.pages ? page : 0u) * a.cache.kv_heads + kvh) * page_elements;
                finite = finite && fabsf((float)v[((i / S::N) << shift) + (at & in_page)]) < INFINITY;
            }
            if (__all(finite)) {
                continue;
            }
#pragma unroll 1
            for (int at = max(base, any_lo); at < min(base + S::N, any_hi); ++at) {
                const uint32_t page = table[min((uint32_t)at >> shift, last_entry)];
                const bool seen = live && at >= lo && at < hi && page < a.cache.pages;
                const T *v = (const T *)a.cache.v + ((size_t)(page < a.cache.pages ? page : 0u) * a.cache.kv_heads + kvh) * page_elements +
                             ((uint32_t)at & in_page);
#pragma unroll
                for (int t = 0; t < S::DT; ++t) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const uint32_t d = 32u * t + 8u * (j / 4) + 4u * h + (j % 4);
                        const float x = (float)v[(FULL ? d : min(d, hd - 1u)) << shift];
                        o[t][j] = seen && !(fabsf(x) < INFINITY) ? NAN : o[t][j];
                    }
                }
            }
        }
    }

    // channel of value v of tile t: 32 t + 8 (v / 4) + 4 h + v % 4
    float *out = a.out + (size_t)row * a.out_stride + (size_t)head * hd;
    // (shared positions: by way of LDS, so that a wave's stores lie side by side; units swapped as in a stage)
    float *all = (float *)lds;
    static_assert(4 * S::BYTES == 128 * D * 4, "results");
    auto unit_of = [&](uint32_t unit) { return (f32x4 *)(all + (wave * 32u + c) * D + (unit ^ (c & 15u)) * 4u); };
    if (parts == 1u && asides == 0u) {
        if (live) {
            const float by = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
            for (int t = 0; t < S::DT; ++t) {
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    const uint32_t d = 32u * t + 8u * (v / 4) + 4u * h + (v % 4);
                    if (FULL || d < hd) {
                        out[d] = l == 0.0f ? 0.0f : o[t][v] * by;
                    }
                }
            }
        }
    } else {
#pragma unroll
        for (int t = 0; t < S::DT; ++t) {
#pragma unroll
            for (int v = 0; v < 16; v += 4) {
                *unit_of(8u * t + v / 2u + h) = f32x4{o[t][v], o[t][v + 1], o[t][v + 2], o[t][v + 3]};
            }
        }
    }
    // The steps put aside, or, of more than there is room for, all: in f32, with the rows' results in LDS. Rare, and slow.
    if (asides != 0u) {
        // (what this needs is taken again from the lane's number and the kernel's arguments, or it
        // would stay in registers over the loop)
        uint32_t lane_here = lane;
        auto kernel_args = (const __attribute__((address_space(4))) PrefillArgs *)__builtin_amdgcn_kernarg_segment_ptr();
        asm volatile("" : "+v"(lane_here), "+s"(kernel_args));
        const AttnArgs a = *(const AttnArgs *)&kernel_args->a;
        const uint32_t c = lane_here & 31u, h = lane_here >> 5, r = tile * 128u + wave * 32u + c;
        const bool live = r < rows, all_steps = asides > ASIDE;
        const uint32_t query = live ? r / a.group : 0u, head = kvh * a.group + (live ? r % a.group : 0u);
        const float *q_row = a.q + (size_t)(row0 + query) * a.q_stride + (size_t)head * hd;
        float *out = a.out + (size_t)(row0 + query) * a.out_stride + (size_t)head * hd;
        const int p = len - n + (int)query;
        const float slope = a.slopes != nullptr ? a.slopes[head] * LOG2E : 0.0f;
        int lo, hi;
        visible(a, len, seq, row0 + query, p, lo, hi);
        auto unit_of = [&](uint32_t unit) { return (f32x4 *)(all + (wave * 32u + c) * D + (unit ^ (c & 15u)) * 4u); };
        const float by = score_factor(a.scale, a.softcap);
        if (all_steps) {
            l = l == l ? 0.0f : l;
            top = -3.402823466e38f;
            for (uint32_t d = 4u * h; d < hd; d += 8u) {
                *unit_of(d / 4u) = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            }
        }
        const uint32_t some = all_steps ? s_end - s_begin : asides;
        for (uint32_t i = 0; i < some; ++i) {
            const int base = (int)(start + (all_steps ? s_begin + i : aside[wave][i]) * S::N);
            const int last = min(base + S::N, any_hi);
            // (as long as there is a row that is not NaN)
            for (int at = max(base, any_lo); at < last && __any(live && l == l); ++at) {
                const uint32_t page = table[min((uint32_t)at >> shift, last_entry)];
                const size_t place = ((size_t)(page < a.cache.pages ? page : 0u) * a.cache.kv_heads + kvh) * page_elements;
                const T *k = (const T *)a.cache.k + place + ((uint32_t)at & in_page) * hd;
                const T *v = (const T *)a.cache.v + place + ((uint32_t)at & in_page);
                float x[1] = {0.0f};
                for (uint32_t d = 4u * h; d < hd; d += 8u) {
#pragma unroll
                    for (uint32_t j = 0; j < 4u; ++j) {
                        x[0] = fmaf(q_row[d + j], (float)k[d + j], x[0]);
                    }
                }
                x[0] = (x[0] + __shfl_xor(x[0], 32)) * by;
                if (a.softcap > 0.0f) {
                    cap_of(x, cap_log2);
                }
                if (a.slopes != nullptr) {
                    x[0] = fmaf(-slope, fabsf((float)(at - p)), x[0]);
                }
                if (live && at >= lo && at < hi && page < a.cache.pages) {
                    const float most = fmaxf(top, x[0]), keep = exp2_of(top - most), w = exp2_of(x[0] - most);
                    top = most;
                    l = fmaf(l, keep, w);
                    for (uint32_t d = 4u * h; d < hd; d += 8u) {
                        f32x4 y = *unit_of(d / 4u);
#pragma unroll
                        for (uint32_t j = 0; j < 4u; ++j) {
                            y[j] = fmaf(y[j], keep, w * (float)v[(d + j) << shift]);
                        }
                        *unit_of(d / 4u) = y;
                    }
                }
            }
        }
        for (uint32_t d = 4u * h; parts == 1u && live && d < hd; d += 8u) {
            const f32x4 y = *unit_of(d / 4u);
#pragma unroll
            for (uint32_t j = 0; j < 4u; ++j) {
                out[d + j] = l == 0.0f ? 0.0f : y[j] / l;
            }
        }
    }
    if (parts == 1u) {
        return;
    }
    // Shared positions: the parts go to memory, and the last workgroup of the tile to
    // arrive adds them up in the order of their positions (as the decode kernel does).
    const size_t part_floats = 128u * (size_t)(hd + 2u);
    const size_t slot = (size_t)want * a.cache.kv_heads + kvh;
    const float *first = args.partials + slot * args.splits * part_floats;
    const uint32_t here = min(128u, rows - tile * 128u), pairs = hd / 2u;
    __syncthreads();
    {
        float *to = (float *)first + split * part_floats;
        for (uint32_t i = threadIdx.x; i < here * pairs; i += 256u) {
            const uint32_t at = i / pairs, d = 2u * (i % pairs);
            const float *from = all + at * D + ((d >> 2) ^ (at & 15u)) * 4u + (d & 2u);
            put2(to + 2u * i, from[0], from[1]);
        }
        if (live && h == 0u) {
            put2(to + 128u * hd + 2u * (wave * 32u + c), top, l);
        }
    }
    __builtin_amdgcn_s_waitcnt(7 << 4);
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
    if (threadIdx.x == 0u) {
        __hip_atomic_store(&args.arrivals[slot], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    // Weights of the parts, then as many rows at a time as LDS holds of all parts: every load is
    // a trip past the L2, so all of a turn's are on their way at once.
    if (threadIdx.x < here) {
        const float *stats = first + 128u * hd + 2u * threadIdx.x;
        float t[PREFILL_MAX_SPLITS], y[PREFILL_MAX_SPLITS];
#pragma unroll
        for (uint32_t s = 0; s < PREFILL_MAX_SPLITS; ++s) {
            t[s] = -INFINITY;
            y[s] = 0.0f;
            if (s < parts) {
                get2(stats + s * part_floats, t[s], y[s]);
            }
        }
        float best = t[0], sum = 0.0f;
#pragma unroll
        for (uint32_t s = 1; s < PREFILL_MAX_SPLITS; ++s) {
            best = fmaxf(best, t[s]);
        }
#pragma unroll
        for (uint32_t s = 0; s < PREFILL_MAX_SPLITS; ++s) {
            t[s] = exp2_of(t[s] - best);
            sum += t[s] * y[s];
        }
#pragma unroll
        for (uint32_t s = 0; s < PREFILL_MAX_SPLITS; ++s) {
            factor[s][threadIdx.x] = sum == 0.0f ? -1.0f : t[s] / sum; // (-1: the row's result is zero)
        }
    }
    const uint32_t row_bytes = hd * 4u;
    const uint32_t at_once = 4u * S::BYTES / 1024u / parts * 1024u / row_bytes; // (pieces of 1 KiB of each part)
    for (uint32_t r0 = 0; r0 < here; r0 += at_once) {
        const uint32_t some = min(at_once, here - r0), bytes = some * row_bytes, pieces = (bytes + 1023u) / 1024u;
        __syncthreads(); // (what lay there has been read, the factors have been written)
        for (uint32_t f = wave; f < parts * pieces; f += 4u) {
            const uint8_t *part = (const uint8_t *)(first + (f / pieces) * part_floats + r0 * hd);
            fetch16_past(part + min((f % pieces) * 1024u + lane * 16u, bytes - 16u), stages + f * 1024u);
        }
        wait_fetches<0>();
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < some * pairs; i += 256u) {
            const uint32_t at = r0 + i / pairs, d = 2u * (i % pairs);
            float y0 = 0.0f, y1 = 0.0f;
            for (uint32_t s = 0; s < parts; ++s) {
                const float *u = (const float *)(lds + s * pieces * 1024u) + 2u * i;
                const float f = factor[s][at];
                y0 += f * u[0];
                y1 += f * u[1];
            }
            const uint32_t rr = tile * 128u + at;
            float *to = a.out + (size_t)(row0 + rr / a.group) * a.out_stride + (size_t)(kvh * a.group + rr % a.group) * hd + d;
            const bool none = factor[0][at] < 0.0f; // (whatever the values: a part of no weight may hold NaN)
            to[0] = none ? 0.0f : y0;
            to[1] = none ? 0.0f : y1;
        }
    }
}

} // namespace kv
