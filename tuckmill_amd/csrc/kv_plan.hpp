// Host-only rules of the operators over the paged cache: how an attention call is cut
// into workgroups and what it needs of the context's workspace. Plain C++.
#pragma once

#include <cstdint>

namespace kv {

// Query heads of one key-value head that a workgroup of the decode kernel takes: the
// 16 columns of its matrix operand hold 8 heads in two f16 parts, or 16 in f32.
inline uint32_t decode_cols(uint32_t type_id) { return type_id == 1u ? 8u : 16u; }

// Shares of the positions: one for each CU. (In us, with 256, 320 and 512 of them: a sequence
// of 131071 tokens and 8 heads 101, 126, 111; 48 ragged ones up to 8192 156, 159, 157; 1500 f32
// rows over a window 69, 69, 90; 256 f32 rows 17, 20, 20: the second workgroup of a CU
// starts late, and every share is a part to join.)
constexpr uint32_t DECODE_SHARES = 256;
constexpr uint64_t DECODE_MAX_GRID = 1u << 23; // (a dimension of a grid is below 2^32 threads)
constexpr uint32_t DECODE_WAVES = 4; // of a workgroup
// Sequences whose work is shared out. Every workgroup then goes through all of them, which their number
// makes dearer and a long one among them makes worth it. (In us, 16 heads of 128 channels on 8, f16, shared and
// not: 513 sequences of 200 135 and 106, one of them of 100000 189 and 1200; 1024 308 and 195, with one 352 and
// 1240; 2048 882 and 362, with one 847 and 1326.)
constexpr uint32_t DECODE_MAX_SEQS = 512;

struct AttnPlan {
    bool tiled = false;      // ragged rows: with the prefill kernel (else the decode kernel's)
    uint32_t shares = 0;     // decode kernel: to make of the positions, 0: one of each unit
    uint64_t grid = 0;       // workgroups for them, at most
    uint32_t splits = 1;     // prefill kernel: workgroups that share a tile's positions, at most
    uint32_t head_tiles = 1; // tiles of a key-value head's query heads
    uint64_t tile_bound = 0; // prefill kernel: tiles of rows, at most
    uint64_t partial_floats = 0, arrivals = 0; // of the workspace
};

// The decode kernel's workgroups: a share each, and what rounding up adds in each unit. How the
// rows and positions fall to units is known on the device only.
inline void share_work(AttnPlan &p, uint64_t units, uint32_t cols, uint32_t head_dim, uint64_t positions) {
    const uint64_t steps = (positions + 63u) / 64u; // (of 64 or 128 positions)
    const uint64_t most = DECODE_SHARES + units, all = units > most / steps ? most : units * steps;
    p.shares = DECODE_SHARES;
    p.grid = all < most ? all : most;
    // (a unit that is cut has more steps than a share: two workgroups for each full share in it)
    p.arrivals = 2u * DECODE_SHARES;
    p.partial_floats = p.arrivals * cols * (head_dim + 2u);
}

// One row per sequence.
inline AttnPlan decode_plan(uint32_t type_id, uint32_t seqs, uint32_t q_heads, uint32_t kv_heads,
                            uint32_t head_dim, uint64_t positions) {
    AttnPlan p;
    const uint32_t cols = decode_cols(type_id);
    p.head_tiles = (q_heads / kv_heads + cols - 1u) / cols;
    if (seqs <= DECODE_MAX_SEQS) {
        share_work(p, (uint64_t)seqs * kv_heads * p.head_tiles, cols, head_dim, positions);
    }
    return p;
}

constexpr uint32_t PREFILL_ROWS = 128; // query rows x heads of a workgroup
constexpr uint32_t PREFILL_MAX_SPLITS = 8;
// Where tiles leave CUs without one their positions are shared, eight steps of 64 at least (in us,
// with 2, 4 and 8: 512 rows of 128 channels on 64 cached 43, 42, 30, on 16000 154 each).
constexpr uint32_t PREFILL_MIN_STEPS = 8;
constexpr uint32_t PREFILL_SHARES = 256; // (512: 256 rows on 16000 cached 118 for 92)
constexpr uint64_t PREFILL_MAX_GROUPS = 1u << 23;
// Up to this many units the decode kernel takes ragged rows. (In us, it and the prefill kernel, on up
// to 64, 2000 and 16000 cached positions: of 128 channels at 1032 units 20, 39, 127 and 21, 53, 92, at
// 2056 38, 66, 281 and 30, 57, 153; of 64 channels at 776 11, 15, 33 and 14, 22, 36, at 1544 21, 35, 88
// and 20, 32, 58; of 256 channels at 516 26, 43, 152 and 52, 105, 190, at 1028 58, 92, 490 and 91, 120,
// 333: near the limit long caches would be better off with the prefill kernel, short ones not, and which they
// are only the device knows; here there is the room in the table.) Pages of f32 it takes always: their products go at
// a sixteenth of f16's rate, and its waves of 16 rows fill the card better than tiles of
// 128 did (1500 rows of 256 channels 69 and 138, 4000 926 and 1216, 4000 of 128 347 and 509).
constexpr uint64_t DECODE_MAX_UNITS = 1056;

// Ragged rows. How they fall to sequences is known on the device only: every
// sequence may have one tile that is not full. Where that leaves few workgroups the
// positions are shared between several (the parts then go through memory).
inline AttnPlan prefill_plan(uint32_t type_id, uint32_t seqs, uint32_t tokens, uint32_t q_heads, uint32_t kv_heads,
                             uint32_t head_dim, uint64_t positions) {
    AttnPlan p;
    const uint64_t rows = (uint64_t)tokens * (q_heads / kv_heads);
    auto tiles_of = [&](uint32_t size) { // (a tile has a row)
        const uint64_t tiles = rows / size + seqs;
        return tiles < rows ? tiles : rows;
    };
    const uint32_t cols = decode_cols(type_id);
    const uint64_t few = tiles_of(cols) * kv_heads;
    if (type_id != 1u || few <= DECODE_MAX_UNITS) {
        share_work(p, few, cols, head_dim, positions);
        return p;
    }
    p.tiled = true;
    p.tile_bound = tiles_of(PREFILL_ROWS);
    const uint64_t units = p.tile_bound * kv_heads;
    uint64_t splits = units < PREFILL_SHARES ? (PREFILL_SHARES + units - 1u) / units : 1u;
    const uint64_t most = positions / (64u * PREFILL_MIN_STEPS);
    splits = splits < most ? splits : most;
    p.splits = (uint32_t)(splits < 1u ? 1u : splits > PREFILL_MAX_SPLITS ? PREFILL_MAX_SPLITS : splits);
    if (p.splits > 1u) {
        p.partial_floats = units * p.splits * PREFILL_ROWS * (head_dim + 2u);
        p.arrivals = units;
    }
    return p;
}

// Ids of a workgroup that adjusts logits: large tiles where they still give every CU one. (In us, large
// and small, rows of 151936: one 7.8 and 7.8, 16 7.9 and 7.6, 64 with histories of 4096 20 and 30; the shortest
// of a call's times 6.6 and 6.4, 7.2 and 7.0.)
constexpr uint32_t LOGITS_LARGE = 8192, LOGITS_SMALL = 1024, LOGITS_MIN_GROUPS = 256;

} // namespace kv
