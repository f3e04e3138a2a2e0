// Attention over the paged cache of one query per sequence, of few ragged rows, and of all rows over f32 pages.
#pragma once

#include "kv_common.hpp"

namespace kv {

struct DecodeArgs {
    AttnArgs a;
    float *partials;
    uint32_t *arrivals;
    uint32_t shares, head_tiles; // shares: to make of the positions, 0: one of each unit
};

// The matrix operands of a tile of positions, in either type of page. Lane l is
// column c = l % 16 (a row of the call) of group g = l / 16. The products run transposed,
// S^T = K q^T and O^T = V^T P, and the positions are dealt to the rows of S^T so
// that what a lane holds of it, positions VALUES g + 0.. for its row, is what it has
// to hand to the second product: the weights never leave their registers. V lies
// in the cache with a channel's positions side by side, so both operands are read
// as they lie there, 16 bytes a lane. In LDS the 16-byte units of a row are swapped by
// exclusive or with (part of) the row's number, which spreads a column of units over
// the banks.
// FULL: head_dim is D; else it is less, and what lies beyond it reads as zeros.
template <typename T, int D, bool FULL> struct Tile;

template <int D, bool FULL> struct Tile<_Float16, D, FULL> {
    static constexpr int COLS = 8;        // columns 0..7 the first part of a row's q and weights, 8..15 the second
    static constexpr int VALUES = 8;      // of a tile of 32 positions that a lane holds
    static constexpr int E = 8, UK = D / 8, SWIZZLE = UK < 16 ? UK - 1 : 15; // 16-byte units: elements, of a key
    static constexpr int KS = D / 32;     // operand pieces of a key
    static constexpr int DT = D / 16;     // channel tiles
    static constexpr int HALVES = 2;      // of 16 keys each in a tile's stage
    static constexpr bool PARTS = true;
    typedef f16x8 Unit;
    typedef Unit K[2]; // of a piece
    typedef f32x4 S[2];
    Unit q[KS];

    // The row's q, scaled by a power of two to a largest magnitude of about 2^13, as
    // f16 parts (22 bits of that magnitude); returns the inverse scale. What is
    // not finite goes whole into the first part.
    __device__ __forceinline__ float load_q(const float *row, uint32_t c, uint32_t g, uint32_t hd, bool live, float sign) {
        float x[KS][8], top = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const uint32_t d = 32u * s + 8u * g;
            const bool there = live && (FULL || d < hd);
            const float *from = row + (FULL || d < hd ? d : 0u);
            const f32x4 y[2] = {*(const f32x4_unaligned *)from, *(const f32x4_unaligned *)(from + 4)};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[s][j] = there ? y[j / 4][j % 4] : 0.0f;
                top = fmaxf(top, fabsf(x[s][j]));
            }
        }
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const int by = scale_bits(top);
        const float scale = ldexpf(sign, by);
        float minus = -1.0f; // (for one instruction that takes the f16 where it is)
        asm("" : "+s"(minus));
#pragma unroll
        for (int s = 0; s < KS; ++s) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float y = x[s][j] * scale;
                const float rest = fmaf((float)(_Float16)y, minus, y);
                q[s][j] = (_Float16)(c < 8u ? y : rest);
            }
        }
        if (__any(!(top < INFINITY))) {
            const bool none = c >= 8u && !(top < INFINITY);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                q[s] = none ? Unit{} : q[s];
            }
        }
        return ldexpf(1.0f, -by);
    }
    // row `at` of a stage of keys (16 a half) is this position of the tile
    static constexpr __device__ __forceinline__ uint32_t k_position(uint32_t at) {
        return 8u * ((at & 15u) >> 2) + (at & 3u) + 4u * (at >> 4);
    }
    static __device__ __forceinline__ void read_k(K &k, const uint8_t *stage, uint32_t c, uint32_t g, uint32_t hd, int s) {
        const uint32_t unit = 4u * s + g;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const uint32_t at = 16u * t + c;
            const Unit x = *(const Unit *)(stage + (at * UK + (unit ^ (at & SWIZZLE))) * 16u);
            k[t] = FULL || 8u * unit < hd ? x : Unit{};
        }
    }
    __device__ __forceinline__ void product(S &acc, const K &k, int s) const {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[t], q[s], acc[t], 0, 0, 0);
        }
    }
    // Both parts of the row: columns c and c + 8 of 16. Where a key is infinite the first
    // part's infinity (or NaN) is the score, whatever the second one gives: `careful`.
    static __device__ __forceinline__ void scores(float (&x)[VALUES], const S &acc, uint32_t c, bool careful) {
#pragma unroll
        for (int j = 0; j < VALUES; ++j) {
            const float y = acc[j / 4][j % 4];
            const float part = careful && c >= 8u ? __builtin_amdgcn_fmed3f(y, -3.402823466e38f, 3.402823466e38f) : y;
            x[j] = part + ror8(part);
        }
    }
    // the part of the weights that the column stands for
    typedef Unit Weights;
    static __device__ __forceinline__ Weights pack(const float (&w)[VALUES], uint32_t c) {
        const float second = c < 8u ? 0.0f : -1.0f;
        Weights p;
#pragma unroll
        for (int j = 0; j < VALUES; ++j) {
            p[j] = (_Float16)fmaf((float)(_Float16)w[j], second, w[j]);
        }
        return p;
    }
    static __device__ __forceinline__ f32x4 weigh(f32x4 o, const Unit &v, const Weights &w) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(v, w, o, 0, 0, 0);
    }
    static __device__ __forceinline__ float whole(float x) { return x + ror8(x); }
};

template <int D, bool FULL> struct Tile<float, D, FULL> {
    static constexpr int COLS = 16;
    static constexpr int VALUES = 4; // of a tile of 16 positions
    static constexpr int E = 4, UK = D / 4, SWIZZLE = 15;
    static constexpr int KS = D / 16;
    static constexpr int DT = D / 16;
    static constexpr int HALVES = 1;
    static constexpr bool PARTS = false;
    typedef f32x4 Unit;
    typedef Unit K;
    typedef f32x4 S[2]; // two sums: a product waits for the one before it in its sum
    Unit q[KS];

    __device__ __forceinline__ float load_q(const float *row, uint32_t, uint32_t g, uint32_t hd, bool live, float sign) {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const uint32_t d = 16u * s + 4u * g;
            const f32x4 x = *(const f32x4_unaligned *)(row + (FULL || d < hd ? d : 0u)) * sign;
            q[s] = live && (FULL || d < hd) ? x : f32x4{};
        }
        return 1.0f;
    }
    static constexpr __device__ __forceinline__ uint32_t k_position(uint32_t at) { return at; }
    static __device__ __forceinline__ void read_k(K &k, const uint8_t *stage, uint32_t c, uint32_t g, uint32_t hd, int s) {
        const uint32_t unit = 4u * s + g;
        const Unit x = *(const Unit *)(stage + (c * UK + (unit ^ (c & SWIZZLE))) * 16u);
        k = FULL || 4u * unit < hd ? x : Unit{};
    }
    __device__ __forceinline__ void product(S &acc, const K &k, int s) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            acc[j % 2] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[j], q[s][j], acc[j % 2], 0, 0, 0);
        }
    }
    static __device__ __forceinline__ void scores(float (&x)[VALUES], const S &acc, uint32_t, bool) {
#pragma unroll
        for (int j = 0; j < VALUES; ++j) {
            x[j] = acc[0][j] + acc[1][j];
        }
    }
    typedef Unit Weights;
    static __device__ __forceinline__ Weights pack(const float (&w)[VALUES], uint32_t) { return Unit{w[0], w[1], w[2], w[3]}; }
    static __device__ __forceinline__ f32x4 weigh(f32x4 o, const Unit &v, const Weights &w) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            o = __builtin_amdgcn_mfma_f32_16x16x4f32(v[j], w[j], o, 0, 0, 0);
        }
        return o;
    }
    static __device__ __forceinline__ float whole(float x) { return x; }
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

// 64 x 16 bytes from memory into 1 KiB of LDS: from the lanes' addresses, or from 32-bit
// offsets beyond a common one. From inline assembly, and waited for by hand: the
// compiler's own bookkeeping would order every LDS read behind all such loads in flight.
__device__ __forceinline__ void fetch16(const void *from, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(lds), "v"(from) : "memory", "m0");
}
__device__ __forceinline__ void fetch16(const void *base, uint32_t offset, uint32_t lds) {
    const uint64_t at = (uint64_t)(uintptr_t)base; // (the same in every lane; said, not left to be found out)
    const uint32_t low = __builtin_amdgcn_readfirstlane((uint32_t)at); // (an int until it is an unsigned one)
    const uint32_t high = __builtin_amdgcn_readfirstlane((uint32_t)(at >> 32));
    const uint64_t uniform = (uint64_t)high << 32 | low;
    // (five wait states between a vector instruction that writes a scalar register and the
    // memory instruction that reads it: here the compiler does not see the latter)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "s"(lds), "v"(offset), "s"(uniform)
                 : "memory", "m0");
}
// past this die's L2, as get2
__device__ __forceinline__ void fetch16_past(const void *from, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off sc1" : : "s"(lds), "v"(from) : "memory", "m0");
}
__device__ __forceinline__ uint32_t lds_address(const uint8_t *p) {
    return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t *)p);
}

// Waits until at most N of the wave's fetches are in flight; its reads of LDS are done.
template <int N> __device__ __forceinline__ void wait_fetches() {
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4));
    asm volatile("" ::: "memory");
}

// Stages of a wave in LDS: two, where one query per sequence waits for memory (48 ragged sequences
// of 128 channels 155 us, with one 162), or one for keys and values in turn, which leaves room for
// more workgroups, where several rows share them (2000 f32 rows of 128 channels 115 us, with two
// 139; 1500 of 256 channels 69, with two 95) or a stage is large: one query per sequence of 256 f32
// channels takes as long with two (16 sequences with a window 30.3 and 30.3, 64 of 2000 67.2 and 67.7, one
// of 600 12.8 and 13.0, one of 100000 101 and 97) until a CU has several workgroups (200 of 700 76 and 85).
template <typename T, int D, bool RAGGED> struct DecodeShape {
    static constexpr int RING = RAGGED || D > 128 ? 1 : 2;
    static constexpr int COLS = sizeof(T) == 2 ? 8 : 16, PITCH = D + 4;
    static constexpr int BYTES = 64 * D;          // keys or values of a tile
    static constexpr int RESULTS = COLS * PITCH * 4;
    static constexpr int LDS = DECODE_WAVES * (RING * BYTES > RESULTS ? RING * BYTES : RESULTS);
};

// A unit of work is a key-value head and a tile of rows; a row is a query and a head of
// the key-value head's group (RAGGED: the rows of tm_hip_attn_prefill where a sequence
// has few, else one query a sequence). The positions of all units, in steps of a tile for
// each of the four waves, are cut into shares of nearly one size, as many as keep the card
// busy: sequences of any lengths end together. A share lies in one unit (one that ran
// on into the next unit would save 1% of the steps and cost a second prologue and join).
// The keys and values of a tile of positions come straight from the pages into the wave's
// own LDS; a stage is fetched again as soon as it has been read, so that keys or values
// are always on their way, the waves never wait for each other before the end, and
// registers do not bound what is in flight. A fetch
// costs no vector instruction: the lanes' offsets stay the same from tile to
// tile, pages and places move the scalar base.
// The softmax runs over one pass: weights are 2^(x - m + 6) with a reference m
// per row that follows the maximum only when that has moved by more than 8 (so weights
// stay below 2^14, and most tiles need no exchange between lanes); two f16 parts hold 22 bits
// of a weight, or where it is below 2^-3 (the row's largest is 2^6 and more) 2^-25; l and o are
// f32 sums. The waves join in LDS, the workgroups of a
// unit through memory: the last to arrive adds the parts up in the order of
// their positions.
// Bound by memory where queries are few: one sequence of 131071 tokens, 8 heads of 128
// channels in f16, 100 us = 5.4 TB/s. Short calls (777 tokens 9 us, where a kernel that does next to nothing
// takes 3) are bound by a chain of waits (lengths, share, table, first pages, parts, join) and the
// way through the code, every line of which is fetched once: loads of q in
// wide pieces and a rolled join (20 KB of code for 30) took 16 sequences in f32 from 57 to 30 us.
// Bound by the f32 matrix cores where f32 rows are many: two sequences of 2000 rows, 16 heads of 128
// channels, 347 us.
template <typename T, int D, bool FULL, bool RAGGED>
__global__ __launch_bounds__(64 * DECODE_WAVES, 2) void attn_decode_kernel(DecodeArgs args) {
    typedef Tile<T, D, FULL> M;
    typedef DecodeShape<T, D, RAGGED> Shape;
    typedef typename M::Unit Unit;
    constexpr int COLS = M::COLS, DT = M::DT, KS = M::KS, PITCH = Shape::PITCH, VALUES = M::VALUES, TOKENS = 4 * VALUES;
    constexpr int NW = DECODE_WAVES, RING = Shape::RING, THREADS = 64 * NW;
    constexpr int PIECES = RING == 2 ? 64 : 4; // of keys and values on their way from LDS at a time
    constexpr int BYTES = Shape::BYTES, FETCHES = BYTES / 1024; // keys or values of a tile
    constexpr int PAGES = TOKENS / 16, KINDS = FETCHES / M::HALVES; // of lane offsets of keys
    // that a join takes at a time, of 8 bytes for each thread
    constexpr int PARTS = Shape::LDS / (8 * THREADS) < 32 ? Shape::LDS / (8 * THREADS) : 32;
    extern __shared__ __align__(1024) uint8_t lds[]; // keys and values of each wave; at the end the waves' results
    static_assert(TOKENS * D * (int)sizeof(T) == BYTES && COLS == Shape::COLS, "results");
    float *merged = (float *)lds;
    __shared__ float stats[NW][2][COLS];
    __shared__ float joins[PARTS][COLS][2];
    __shared__ uint32_t arrived;
    const AttnArgs &a = args.a;
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t c = lane & 15u, g = lane >> 4;
    const uint32_t hd = FULL ? (uint32_t)D : a.cache.head_dim, shift = a.cache.page_shift;
    const size_t part_floats = (size_t)COLS * (hd + 2u);
    const uint32_t last_entry = a.table_stride - 1u, in_page = (1u << shift) - 1u;
    const uint32_t page_elements = hd << shift;
    uint8_t *stage = lds + wave * (RING * BYTES), *v_stage = stage + (RING - 1) * BYTES;
    const uint32_t k_lds = lds_address(stage), v_lds = lds_address(v_stage);
    // A fetch of keys is rows 64 / UK of the stage, all within 16 positions of the tile.
    constexpr uint32_t ROWS = 64u / M::UK;
    uint32_t k_offset[KINDS];
#pragma unroll
    for (int f = 0; f < KINDS; ++f) {
        const uint32_t at = f * ROWS + lane / M::UK, d = ((lane % M::UK) ^ (at & M::SWIZZLE)) * M::E;
        k_offset[f] = ((M::k_position(at) & 15u) * hd + (FULL || d < hd ? d : 0u)) * (uint32_t)sizeof(T);
    }
    // A fetch of values is 16 channels' units of the tile.
    const uint32_t v_row = lane >> 2, v_position = ((lane & 3u) ^ ((v_row >> 2) & 3u)) * M::E;

    // What there is to do, and this workgroup's share of it.
    auto units_of = [&](uint32_t n) { // of a sequence of n rows
        return RAGGED ? (n * a.group + COLS - 1u) / COLS * a.cache.kv_heads : a.cache.kv_heads * args.head_tiles;
    };
    // Steps of a unit: of the positions that the sequence's query sees, or (RAGGED, where
    // every row sees its own) all that any could.
    auto steps_of = [&](uint32_t s, uint32_t n) {
        const int len = seq_len(a, s);
        int lo = 0, hi = len;
        if constexpr (!RAGGED) {
            visible(a, len, s, s, len - 1, lo, hi);
        } else if (a.window != 0u && a.prefix == nullptr) {
            hi = (int)min((uint64_t)len, (uint64_t)a.window + n + TOKENS);
        }
        const uint32_t tiles = lo < hi ? ((uint32_t)hi - ((uint32_t)lo & ~(uint32_t)(TOKENS - 1)) + TOKENS - 1u) / TOKENS : 0u;
        return max(1u, (tiles + NW - 1u) / NW); // (a unit that sees nothing has zeros to write)
    };
    uint32_t seq = blockIdx.y, tile = blockIdx.x / a.cache.kv_heads, kvh = blockIdx.x % a.cache.kv_heads;
    uint32_t row0 = seq, rows = a.group, part = 0, parts = 1, slot = 0;
    if (RAGGED || args.shares != 0u) {
        // 64 sequences, one a lane: its rows, a unit's steps, and the sum up to its end: of steps, or
        // (once the size of a share is known) of shares, and in the high half of those that
        // are not all of their unit
        uint32_t s0 = 0, highest = 0, rows_up_to = 0, first_here = 0, rows_here = 0, steps_here = 0, size = 0;
        uint64_t before = 0, upto = 0; // `before`: of the sequences before s0
        auto add_up = [&]() {
            const uint64_t shares = size != 0u ? (steps_here + size - 1u) / size : 0u;
            upto = sum_over_lanes((uint64_t)units_of(rows_here) *
                                  (size == 0u ? steps_here : shares > 1u ? shares | shares << 32 : shares));
        };
        auto look = [&]() {
            rows_up_to = highest;
            const uint32_t s = min(s0 + lane, a.seqs - 1u);
            first_here = s;
            rows_here = RAGGED ? rows_of(a, s0, rows_up_to, first_here) : s0 + lane < a.seqs ? 1u : 0u;
            steps_here = steps_of(s, rows_here);
            steps_here = rows_here != 0u ? steps_here : 0u;
            add_up();
        };
        auto look_on = [&]() {
            before += last_of(upto);
            highest = rows_up_to;
            s0 += 64u;
            look();
        };
        look();
        while (s0 + 64u < a.seqs) {
            look_on();
        }
        size = (uint32_t)((before + last_of(upto) + args.shares - 1u) / args.shares);
        size = __builtin_amdgcn_readfirstlane(max(size, 1u));
        before = 0;
        if (s0 == 0u) {
            add_up();
        } else {
            s0 = highest = 0;
            look();
        }
        uint64_t found;
        while ((found = __ballot(blockIdx.x < (uint32_t)(before + upto))) == 0ull) {
            if (s0 + 64u >= a.seqs) {
                return;
            }
            look_on();
        }
        const int at = __builtin_ctzll(found);
        seq = s0 + (uint32_t)at;
        parts = (__shfl(steps_here, at) + size - 1u) / size;
        rows = __shfl(rows_here, at) * a.group;
        row0 = __shfl(first_here, at);
        before += at > 0 ? __shfl(upto, at - 1) : 0u;
        const uint32_t index = blockIdx.x - (uint32_t)before, unit = index / parts;
        part = index % parts;
        slot = (uint32_t)(before >> 32) + unit * parts; // (at most two for each full share)
        kvh = unit % a.cache.kv_heads;
        tile = unit / a.cache.kv_heads;
        seq = __builtin_amdgcn_readfirstlane(seq);
        parts = __builtin_amdgcn_readfirstlane(parts);
        part = __builtin_amdgcn_readfirstlane(part);
        tile = __builtin_amdgcn_readfirstlane(tile);
        kvh = __builtin_amdgcn_readfirstlane(kvh);
        row0 = __builtin_amdgcn_readfirstlane(row0);
        rows = __builtin_amdgcn_readfirstlane(rows);
        slot = __builtin_amdgcn_readfirstlane(slot); // of the unit's first part
    }
    const uint32_t first_row = tile * COLS, here = min((uint32_t)COLS, rows - first_row); // of this tile

    // this lane's row, what it sees, what any row of the tile sees and what all see
    const uint32_t col = COLS == 8 ? c & 7u : c;
    const bool live = col < here;
    const uint32_t r = first_row + (live ? col : 0u);
    const uint32_t query = RAGGED ? r / a.group : 0u, head = kvh * a.group + (RAGGED ? r % a.group : r);
    const int len = seq_len(a, seq);
    const int p = RAGGED ? len - (int)(rows / a.group) + (int)query : len - 1;
    int lo, hi;
    visible(a, len, seq, row0 + query, p, lo, hi);
    int any_lo = lo < hi ? lo : 0x7fffffff, any_hi = lo < hi ? hi : 0, all_lo = lo, all_hi = hi;
    if constexpr (RAGGED) {
        any_lo = least16(any_lo);
        any_hi = most16(any_hi);
        all_lo = most16(all_lo);
        all_hi = least16(all_hi);
    }
    any_lo = __builtin_amdgcn_readfirstlane(any_lo);
    any_hi = __builtin_amdgcn_readfirstlane(any_hi);
    all_lo = __builtin_amdgcn_readfirstlane(all_lo);
    all_hi = __builtin_amdgcn_readfirstlane(all_hi);
    const uint32_t start = any_lo < any_hi ? (uint32_t)any_lo & ~(uint32_t)(TOKENS - 1) : 0u;
    const uint32_t tiles = any_lo < any_hi ? ((uint32_t)any_hi - start + TOKENS - 1u) / TOKENS : 0u;
    const uint32_t each = (tiles + parts * NW - 1u) / (parts * NW); // of a wave
    const uint32_t t0 = min(tiles, (part * NW + wave) * each), n = min(tiles, t0 + each) - t0;

    // Pages of a tile, one for every 16 positions, looked up ahead.
    const __attribute__((address_space(4))) uint32_t *table =
        (const __attribute__((address_space(4))) uint32_t *)(a.table + (size_t)seq * a.table_stride);
    struct Pages {
        uint32_t id[PAGES];
    };
    auto look_up = [&](uint32_t i) {
        Pages p;
        const uint32_t base = start + TOKENS * (t0 + i);
#pragma unroll
        for (int b = 0; b < PAGES; ++b) {
            p.id[b] = table[min((base + 16u * b) >> shift, last_entry)];
        }
        return p;
    };
    auto head_page = [&](uint32_t page) { // (a page that is not there is not seen: somewhere to read from)
        return ((size_t)(page < a.cache.pages ? page : 0u) * a.cache.kv_heads + kvh) * page_elements;
    };
    auto fetch_k = [&](uint32_t i, const Pages &p) {
        const uint32_t base = start + TOKENS * (t0 + i);
#pragma unroll
        for (int b = 0; b < PAGES; ++b) {
            const uint8_t *page = (const uint8_t *)((const T *)a.cache.k + head_page(p.id[b]) + ((base + 16u * b) & in_page) * hd);
#pragma unroll
            for (int f = 0; f < FETCHES; ++f) {
                if ((int)(M::k_position(f * ROWS) >> 4) == b) {
                    // (the second half of a stage lies four positions on)
                    fetch16(page + (f / KINDS) * (4u * hd * sizeof(T)), k_offset[f % KINDS], k_lds + f * 1024);
                }
            }
        }
    };
    auto fetch_v = [&](uint32_t i, const Pages &p) {
        const uint32_t base = start + TOKENS * (t0 + i);
        const T *v = (const T *)a.cache.v + head_page(p.id[0]) + (base & in_page);
        if (PAGES == 1 || in_page >= (uint32_t)TOKENS - 1u) {
#pragma unroll
            for (int f = 0; f < FETCHES; ++f) { // (channels beyond the last: results that are not used)
                const uint32_t d = FULL ? v_row : min(16u * f + v_row, hd - 1u);
                fetch16(v + (FULL ? (16u * f) << shift : 0u), ((d << shift) + v_position) * (uint32_t)sizeof(T), v_lds + f * 1024);
            }
        } else { // pages of 16 positions
            const T *second = (const T *)a.cache.v + head_page(p.id[PAGES - 1]);
            const T *mine = (v_position < 16u ? v : second) + (v_position & 15u);
#pragma unroll
            for (int f = 0; f < FETCHES; ++f) {
                fetch16(mine + ((FULL ? 16u * f + v_row : min(16u * f + v_row, hd - 1u)) << shift), v_lds + f * 1024);
            }
        }
    };
    Pages now = {}, next = {};
    if (n > 0u) {
        now = look_up(0u);
        fetch_k(0u, now);
        if constexpr (RING == 2) {
            fetch_v(0u, now);
        }
        next = look_up(1u);
    }

    M m;
    const float unscale = m.load_q(a.q + (size_t)(row0 + query) * a.q_stride + (size_t)head * hd, c, g, hd, live,
                                   a.scale < 0.0f ? -1.0f : 1.0f);
    const float slope = a.slopes != nullptr ? a.slopes[head] * LOG2E : 0.0f;
    const float scale = fabsf(a.scale) * unscale; // (its sign is with q)
    const float to_log2 = score_factor(scale, a.softcap);
    const float cap_log2 = a.softcap * LOG2E;

    f32x4 o[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) {
        o[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    float top = -3.402823466e38f, l = 0.0f;
    bool cleaned = false;

    for (uint32_t i = 0; i < n; ++i) {
        const uint32_t base = start + TOKENS * (t0 + i);
        const Pages after = look_up(i + 2u);
        typename M::S acc = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}, f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
        wait_fetches<(RING - 1) * FETCHES>(); // all but this tile's values
        {
            // (where registers are short: a few pieces are read while those before them are
            // multiplied, and no earlier)
            constexpr int AT_ONCE = PIECES < KS ? PIECES : KS;
            typename M::K k[AT_ONCE], ahead[AT_ONCE];
#pragma unroll
            for (int s = 0; s < AT_ONCE; ++s) {
                M::read_k(ahead[s], stage, c, g, hd, s);
            }
#pragma unroll
            for (int s0 = 0; s0 < KS; s0 += AT_ONCE) {
#pragma unroll
                for (int s = 0; s < AT_ONCE; ++s) {
                    __builtin_memcpy(&k[s], &ahead[s], sizeof(k[s]));
                }
                if (s0 + AT_ONCE < KS) {
                    asm volatile("" ::: "memory");
#pragma unroll
                    for (int s = 0; s < AT_ONCE; ++s) {
                        M::read_k(ahead[s], stage, c, g, hd, s0 + AT_ONCE + s);
                    }
                } else if constexpr (RING == 1) {
                    wait_fetches<0>(); // (the reads of the keys)
                    fetch_v(i, now);
                }
#pragma unroll
                for (int s = 0; s < AT_ONCE; ++s) {
                    m.product(acc, k[s], s0 + s);
                }
            }
        }
        if (RING == 2 && i + 1u < n) {
            wait_fetches<FETCHES>(); // (the reads of the keys)
            fetch_k(i + 1u, next);
        }
        const bool known = (PAGES == 1 || g < 2u ? now.id[0] : now.id[PAGES - 1]) < a.cache.pages;
        const int at = (int)(base + VALUES * g);
        const bool whole = __all((int)base >= all_lo && (int)base + TOKENS <= all_hi && known);
        float w[VALUES];
        float keep = 1.0f, sum = l;
        for (bool careful = false;; careful = true) {
            float x[VALUES];
            M::scores(x, acc, c, careful);
            // (rounded before the reference is taken from it: a fused difference would leave
            // a huge score's rounding in the exponent)
#pragma unroll
            for (int j = 0; j < VALUES; ++j) {
                x[j] *= to_log2;
            }
            if (a.softcap > 0.0f) {
                cap_of(x, cap_log2);
            }
            if (a.slopes != nullptr) {
#pragma unroll
                for (int j = 0; j < VALUES; ++j) {
                    x[j] = fmaf(-slope, fabsf((float)(at - p) + (float)j), x[j]);
                }
            }
            if (!whole) {
#pragma unroll
                for (int j = 0; j < VALUES; ++j) {
                    x[j] = known && at + j >= lo && at + j < hi ? x[j] : -INFINITY;
                }
            }
            float most = x[0];
#pragma unroll
            for (int j = 1; j < VALUES; ++j) {
                most = fmaxf(most, x[j]);
            }
            if (__any(most > top + 8.0f)) {
                most = fmaxf(most, __shfl_xor(most, 16));
                most = fmaxf(most, __shfl_xor(most, 32));
                most = fmaxf(most, top);
                keep *= exp2_of(top - most);
                top = most;
            }
            l = sum * keep;
#pragma unroll
            for (int j = 0; j < VALUES; ++j) {
                w[j] = exp2_of(x[j] - top + 6.0f);
                l += w[j];
            }
            if (!M::PARTS || careful || !__any(l != l)) {
                break;
            }
        }
        if (__any(keep != 1.0f)) {
#pragma unroll
            for (int j = 0; j < DT; ++j) {
                o[j] *= keep;
            }
        }
        if (RING == 2 && i + 1u < n) {
            wait_fetches<FETCHES>(); // all but the next tile's keys
        } else {
            wait_fetches<0>();
        }
        if (!whole) {
            // What a row does not see must not reach it through a weight of zero: positions that
            // no row sees become zeros (0 x infinity would be NaN), and so do values that are
            // not finite where rows see different positions; those that see them are told
            // after the loop.
            const bool there = (PAGES == 1 || v_position < 16u ? now.id[0] : now.id[PAGES - 1]) < a.cache.pages;
            const int from = there ? any_lo - (int)(base + v_position) : 0x7fffffff, upto = any_hi - (int)(base + v_position);
            bool wrong = false;
#pragma unroll 4
            for (int f = 0; f < FETCHES; ++f) {
                Unit *unit = (Unit *)(v_stage + f * 1024 + lane * 16u);
                Unit v = *unit;
#pragma unroll
                for (int j = 0; j < VALUES; ++j) {
                    const bool by_any = j >= from && j < upto, finite = !RAGGED || fabsf((float)v[j]) < INFINITY;
                    wrong = wrong || (by_any && !finite);
                    v[j] = by_any && finite ? v[j] : (T)0.0f;
                }
                *unit = v;
            }
            cleaned = cleaned || (RAGGED && __any(wrong));
        }
        {
            const typename M::Weights p = M::pack(w, c);
            auto read_v = [&](int t) { // channel 16 t + c, positions VALUES g and on
                const uint32_t d = 16u * t + c;
                return *(const Unit *)(v_stage + (d * 4u + (g ^ ((d >> 2) & 3u))) * 16u);
            };
            constexpr int AT_ONCE = PIECES < DT ? PIECES : DT;
            Unit v[AT_ONCE], ahead[AT_ONCE];
#pragma unroll
            for (int t = 0; t < AT_ONCE; ++t) {
                ahead[t] = read_v(t);
            }
#pragma unroll
            for (int t0 = 0; t0 < DT; t0 += AT_ONCE) {
#pragma unroll
                for (int t = 0; t < AT_ONCE; ++t) {
                    v[t] = ahead[t];
                }
                if (t0 + AT_ONCE < DT) {
                    asm volatile("" ::: "memory");
#pragma unroll
                    for (int t = 0; t < AT_ONCE; ++t) {
                        ahead[t] = read_v(t0 + AT_ONCE + t);
                    }
                } else if (RING == 1 && i + 1u < n) {
                    wait_fetches<0>(); // (the reads of the values)
                    fetch_k(i + 1u, next);
                }
#pragma unroll
                for (int t = 0; t < AT_ONCE; ++t) {
                    o[t0 + t] = M::weigh(o[t0 + t], v[t], p);
                }
            }
        }
        if (RING == 2 && i + 1u < n) {
            wait_fetches<FETCHES>(); // (the reads of the values)
            fetch_v(i + 1u, next);
        }
        now = next;
        next = after;
    }

    if (RAGGED && cleaned) {
        // Rare, and as slow as it looks: every value of the wave's tiles that a row sees.
        const int first = max(any_lo, (int)(start + TOKENS * t0)), last = min(any_hi, (int)(start + TOKENS * (t0 + n)));
#pragma unroll 1
        for (int at = first; at < last; ++at) {
            const uint32_t page = table[min((uint32_t)at >> shift, last_entry)];
            const bool seen = live && at >= lo && at < hi && page < a.cache.pages;
            const T *v = (const T *)a.cache.v + head_page(page) + ((uint32_t)at & in_page);
#pragma unroll
            for (int t = 0; t < DT; ++t) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t d = 16u * t + 4u * g + j;
                    const float x = (float)v[(FULL ? d : min(d, hd - 1u)) << shift];
                    o[t][j] = seen && !(fabsf(x) < INFINITY) ? NAN : o[t][j];
                }
            }
        }
    }

    // the waves' results
    __syncthreads(); // (in the place of their rings)
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
    auto write_out = [&](uint32_t of, uint32_t d, float sum, float y0, float y1) {
        const uint32_t r = first_row + of, query = RAGGED ? r / a.group : 0u;
        float *out = a.out + (size_t)(row0 + query) * a.out_stride + (size_t)(kvh * a.group + (RAGGED ? r % a.group : r)) * hd + d;
        out[0] = sum == 0.0f ? 0.0f : y0 / sum;
        out[1] = sum == 0.0f ? 0.0f : y1 / sum;
    };
    auto part_of = [&](uint32_t of) { return args.partials + (slot + of) * part_floats; };
    for (uint32_t i = threadIdx.x; i < here * pairs; i += THREADS) {
        const uint32_t h = i / pairs, d = 2u * (i % pairs);
        float best = stats[0][0][h];
#pragma unroll
        for (int w = 1; w < NW; ++w) {
            best = fmaxf(best, stats[w][0][h]);
        }
        float sum = 0.0f, y0 = 0.0f, y1 = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float f = exp2_of(stats[w][0][h] - best);
            sum += f * stats[w][1][h];
            y0 += f * merged[(w * COLS + h) * PITCH + d];
            y1 += f * merged[(w * COLS + h) * PITCH + d + 1u];
        }
        if (parts == 1u) {
            write_out(h, d, sum, y0, y1);
        } else {
            float *to = part_of(part);
            put2(to + h * hd + d, y0, y1);
            if (d == 0u) {
                put2(to + COLS * hd + 2u * h, best, sum);
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
    // As many rows at a time as there are threads for, a batch of their parts at a time in LDS:
    // every load is a trip past the L2, so all of a batch's are on their way at once.
    const uint32_t at_once = THREADS / pairs;
    for (uint32_t h0 = 0; h0 < here; h0 += at_once) {
        const uint32_t some_rows = min(at_once, here - h0), bytes = some_rows * hd * 4u, pieces = (bytes + 1023u) / 1024u;
        const bool mine = threadIdx.x < some_rows * pairs;
        const uint32_t row = mine ? threadIdx.x / pairs : 0u, d = 2u * (threadIdx.x % pairs);
        float best = -3.402823466e38f, sum = 0.0f, y0 = 0.0f, y1 = 0.0f;
        for (uint32_t s0 = 0; s0 < parts; s0 += PARTS) {
            const uint32_t some = min((uint32_t)PARTS, parts - s0);
            __syncthreads(); // (what lay there has been read)
            for (uint32_t f = wave; f < some * pieces; f += NW) {
                const uint8_t *from = (const uint8_t *)(part_of(s0 + f / pieces) + h0 * hd);
                fetch16_past(from + min((f % pieces) * 1024u + lane * 16u, bytes - 16u), lds_address(lds) + f * 1024u);
            }
            for (uint32_t i = threadIdx.x; i < some * some_rows; i += THREADS) {
                float t, of;
                get2(part_of(s0 + i / some_rows) + COLS * hd + 2u * (h0 + i % some_rows), t, of);
                joins[i / some_rows][i % some_rows][0] = t;
                joins[i / some_rows][i % some_rows][1] = of;
            }
            wait_fetches<0>();
            __syncthreads();
            const float before = best;
            for (uint32_t k = 0; k < some; ++k) {
                best = fmaxf(best, joins[k][row][0]);
            }
            const float keep = exp2_of(before - best);
            sum *= keep;
            y0 *= keep;
            y1 *= keep;
#pragma unroll 4
            for (uint32_t k = 0; k < some; ++k) {
                const float *of = (const float *)(lds + k * pieces * 1024u) + row * hd + d;
                const float f = exp2_of(joins[k][row][0] - best);
                sum += f * joins[k][row][1];
                y0 += f * of[0];
                y1 += f * of[1];
            }
        }
        if (mine) {
            write_out(h0 + row, d, sum, y0, y1);
        }
    }
}

} // namespace kv
