// Host-only rules of the operators over the paged cache: how an attention call is cut
// into workgroups and what it needs of the context's workspace. Plain C++.
#pragma once

#include <cstdint>

namespace kv {

// Query heads of one key-value head that a workgroup of the decode kernel takes: the
// 16 columns of its matrix operand hold 8 heads in two f16 parts, or 16 in f32.
inline uint32_t decode_cols(uint32_t type_id) { return type_id == 1u ? 8u : 16u; }

constexpr uint32_t DECODE_MAX_SPLITS = 256;

struct AttnPlan {
    uint32_t splits = 1;     // workgroups that share a sequence's positions
    uint32_t head_tiles = 1; // workgroups that share a key-value head's query heads
    uint64_t tile_bound = 0; // tiles of rows, at most
    uint64_t partial_floats = 0, arrivals = 0; // of the workspace
};

// One row per sequence. The number of positions is known on the device only: the
// table's width bounds it, and every workgroup takes an equal share of what there
// really is (of shares that would be empty the workgroup ends at once).
inline AttnPlan decode_plan(uint32_t type_id, uint32_t seqs, uint32_t q_heads, uint32_t kv_heads,
                            uint32_t head_dim, uint64_t positions) {
    AttnPlan p;
    const uint32_t cols = decode_cols(type_id);
    p.head_tiles = (q_heads / kv_heads + cols - 1u) / cols;
    const uint64_t units = (uint64_t)seqs * kv_heads * p.head_tiles;
    uint64_t splits = (2048u + units - 1u) / units;
    const uint64_t most = (positions + 127u) / 128u; // a step of the four waves each
    splits = splits < most ? splits : most;
    p.splits = (uint32_t)(splits < 1u ? 1u : splits > DECODE_MAX_SPLITS ? DECODE_MAX_SPLITS : splits);
    if (p.splits > 1u) {
        p.partial_floats = units * p.splits * cols * (head_dim + 2u);
        p.arrivals = units;
    }
    return p;
}

constexpr uint32_t PREFILL_ROWS = 128; // query rows x heads of a workgroup
constexpr uint32_t PREFILL_MAX_SPLITS = 32;
constexpr uint64_t PREFILL_MAX_GROUPS = 1u << 23;

// Ragged rows. How they fall to sequences is known on the device only: every
// sequence may have one tile that is not full. Where that leaves few workgroups the
// positions are shared between several (the parts then go through memory).
inline AttnPlan prefill_plan(uint32_t seqs, uint32_t tokens, uint32_t q_heads, uint32_t kv_heads,
                             uint32_t head_dim, uint64_t positions) {
    AttnPlan p;
    const uint64_t rows = (uint64_t)tokens * (q_heads / kv_heads);
    const uint64_t per_tile = rows / PREFILL_ROWS + seqs;
    p.tile_bound = per_tile < rows ? per_tile : rows; // (a tile has a row)
    const uint64_t units = p.tile_bound * kv_heads;
    uint64_t splits = units < 256u ? (512u + units - 1u) / units : 1u;
    const uint64_t most = (positions + 255u) / 256u;
    splits = splits < most ? splits : most;
    p.splits = (uint32_t)(splits < 1u ? 1u : splits > PREFILL_MAX_SPLITS ? PREFILL_MAX_SPLITS : splits);
    if (p.splits > 1u) {
        p.partial_floats = units * p.splits * PREFILL_ROWS * (head_dim + 2u);
        p.arrivals = units;
    }
    return p;
}

// Ids of a workgroup that adjusts logits: large tiles where they still give every CU one.
constexpr uint32_t LOGITS_LARGE = 8192, LOGITS_SMALL = 1024, LOGITS_MIN_GROUPS = 256;

} // namespace kv
