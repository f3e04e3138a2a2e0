// tm_kv.cpp — the operators between a step's products: rotary positions with the
// store into the paged cache, attention over it, logits. Turns an operation with
// KvParams (tm_plan.hpp) into kernel arguments, an instantiation and a grid.
#include "tm_launch.hpp"

#include "kv_attn_decode.hpp"
#include "kv_attn_prefill.hpp"
#include "kv_logits.hpp"
#include "kv_rope.hpp"

using namespace tmh;

namespace {

template <typename T> T *ptr_of(const Alloc *a) { return a != nullptr ? (T *)a->ptr : nullptr; }

kv::AttnArgs attn_args(const Op &op) {
    const KvParams &p = *op.kv;
    kv::AttnArgs a;
    a.cache = kv::Cache{op.a[1]->ptr, op.a[2]->ptr, p.pages, p.page_shift, p.kv_heads, p.head_dim};
    a.q = ptr_of<const float>(op.a[0]) + p.q_off;
    a.out = ptr_of<float>(op.a[3]) + p.out_off;
    a.table = ptr_of<const uint32_t>(p.more[0]);
    a.lens = ptr_of<const uint32_t>(p.more[1]);
    a.starts = ptr_of<const uint32_t>(p.more[2]);
    a.slopes = ptr_of<const float>(p.more[3]);
    a.first = ptr_of<const uint32_t>(p.more[4]);
    a.prefix = ptr_of<const uint32_t>(p.more[5]);
    a.tokens = p.tokens;
    a.seqs = p.seqs;
    a.q_heads = p.q_heads;
    a.group = p.q_heads / p.kv_heads;
    a.table_stride = p.table_stride;
    a.q_stride = p.q_stride;
    a.out_stride = p.out_stride;
    a.window = p.window;
    a.scale = p.scale;
    a.softcap = p.softcap;
    return a;
}

// A launch with LDS bytes of dynamic LDS: beyond 64 KiB (the few static words counted in)
// a kernel has to be told once that it may.
template <uint32_t LDS, auto KERNEL, typename Args>
hipError_t launch_lds(hipStream_t stream, hipEvent_t stop, dim3 grid, dim3 block, const Args &args) {
    if (LDS + 1024u > 65536u) {
        static const hipError_t told =
            hipFuncSetAttribute((const void *)KERNEL, hipFuncAttributeMaxDynamicSharedMemorySize, (int)LDS);
        if (told != hipSuccess) {
            return told;
        }
    }
    Q8_LAUNCH(KERNEL, grid, block, LDS, stream, stop, args);
    return hipGetLastError();
}

template <typename T, int D, bool RAGGED>
hipError_t launch_decode_as(hipStream_t stream, hipEvent_t stop, const kv::DecodeArgs &args, uint64_t grid_x) {
    const dim3 grid = args.shares != 0u ? dim3((uint32_t)grid_x) : dim3(args.a.cache.kv_heads * args.head_tiles, args.a.seqs);
    constexpr uint32_t LDS = kv::DecodeShape<T, D, RAGGED>::LDS;
    const dim3 block(64u * kv::DECODE_WAVES);
    return args.a.cache.head_dim == (uint32_t)D
               ? launch_lds<LDS, kv::attn_decode_kernel<T, D, true, RAGGED>>(stream, stop, grid, block, args)
               : launch_lds<LDS, kv::attn_decode_kernel<T, D, false, RAGGED>>(stream, stop, grid, block, args);
}

// A row per sequence, or (RAGGED) sequences of few rows.
template <bool RAGGED> hipError_t launch_decode(hipStream_t stream, hipEvent_t stop, const Op &op) {
    const KvParams &p = *op.kv;
    const kv::AttnPlan plan = attn_plan_of(p, op.kind);
    if (plan.shares != 0u && (p.partials == nullptr || p.arrivals == nullptr || plan.grid > kv::DECODE_MAX_GRID)) {
        return hipErrorInvalidValue;
    }
    const kv::DecodeArgs args{attn_args(op), p.partials, p.arrivals, plan.shares, plan.head_tiles};
    const uint32_t d = p.head_dim;
    if (p.type_id == 1u) {
        return d <= 64u    ? launch_decode_as<_Float16, 64, RAGGED>(stream, stop, args, plan.grid)
               : d <= 128u ? launch_decode_as<_Float16, 128, RAGGED>(stream, stop, args, plan.grid)
                           : launch_decode_as<_Float16, 256, RAGGED>(stream, stop, args, plan.grid);
    }
    return d <= 64u    ? launch_decode_as<float, 64, RAGGED>(stream, stop, args, plan.grid)
           : d <= 128u ? launch_decode_as<float, 128, RAGGED>(stream, stop, args, plan.grid)
                       : launch_decode_as<float, 256, RAGGED>(stream, stop, args, plan.grid);
}

template <int D, int W> hipError_t launch_prefill_as(hipStream_t stream, hipEvent_t stop, const kv::PrefillArgs &args) {
    constexpr uint32_t LDS = 4u * kv::PrefillShape<D>::BYTES;
    const dim3 grid(args.a.cache.kv_heads * args.splits * args.tile_bound);
    return args.a.cache.head_dim == (uint32_t)D
               ? launch_lds<LDS, kv::attn_prefill_kernel<D, true, W>>(stream, stop, grid, dim3(256), args)
               : launch_lds<LDS, kv::attn_prefill_kernel<D, false, W>>(stream, stop, grid, dim3(256), args);
}

hipError_t launch_prefill(hipStream_t stream, hipEvent_t stop, const Op &op) {
    const KvParams &p = *op.kv;
    const kv::AttnPlan plan = attn_plan_of(p, op.kind);
    if (!plan.tiled) {
        return launch_decode<true>(stream, stop, op);
    }
    if (plan.splits > 1u && (p.partials == nullptr || p.arrivals == nullptr)) {
        return hipErrorInvalidValue;
    }
    const kv::PrefillArgs args{attn_args(op), p.partials, p.arrivals, plan.splits, (uint32_t)plan.tile_bound};
    const uint32_t d = p.head_dim;
    return d <= 64u    ? launch_prefill_as<64, 2>(stream, stop, args)
           : d <= 128u ? launch_prefill_as<128, 2>(stream, stop, args)
                       : launch_prefill_as<256, 1>(stream, stop, args);
}

hipError_t launch_rope(hipStream_t stream, hipEvent_t stop, const Op &op) {
    const KvParams &p = *op.kv;
    kv::RopeArgs a;
    a.q = ptr_of<const float>(op.a[0]) + p.q_off;
    a.k = ptr_of<const float>(op.a[1]) + p.k_off;
    a.v = ptr_of<const float>(op.a[2]) + p.v_off;
    a.q_out = ptr_of<float>(op.a[3]) + p.out_off;
    a.k_cache = p.more[0]->ptr;
    a.v_cache = p.more[1]->ptr;
    a.positions = ptr_of<const uint32_t>(p.more[2]);
    a.slots = ptr_of<const uint32_t>(p.more[3]);
    a.freqs = ptr_of<const float>(p.more[4]);
    a.tokens = p.tokens;
    a.q_heads = p.q_heads;
    a.kv_heads = p.kv_heads;
    a.head_dim = p.head_dim;
    a.pages = p.pages;
    a.page_shift = p.page_shift;
    a.q_stride = p.q_stride;
    a.k_stride = p.k_stride;
    a.v_stride = p.v_stride;
    a.out_stride = p.out_stride;
    a.rot_dim = p.rot_dim;
    a.adjacent = p.adjacent;
    memcpy(a.axis, p.axis, sizeof a.axis);
    const dim3 grid((p.tokens + kv::ROPE_ROWS - 1u) / kv::ROPE_ROWS,
                    (p.q_heads + p.kv_heads + kv::ROPE_HEADS - 1u) / kv::ROPE_HEADS +
                        (p.kv_heads * p.head_dim + kv::ROPE_CHANNELS - 1u) / kv::ROPE_CHANNELS);
    // rows and both halves of a head in 16-byte pieces (head_dim is a multiple of eight)
    const bool wide = (((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.q_out) & 15u) == 0u &&
                      ((p.q_stride | p.k_stride | p.v_stride | p.out_stride) & 3u) == 0u && p.rot_dim % 8u == 0u;
    if (p.type_id == 1u) {
        if (wide) {
            Q8_LAUNCH((kv::rope_store_kernel<_Float16, true>), grid, dim3(256), 0, stream, stop, a);
        } else {
            Q8_LAUNCH((kv::rope_store_kernel<_Float16, false>), grid, dim3(256), 0, stream, stop, a);
        }
    } else if (wide) {
        Q8_LAUNCH((kv::rope_store_kernel<float, true>), grid, dim3(256), 0, stream, stop, a);
    } else {
        Q8_LAUNCH((kv::rope_store_kernel<float, false>), grid, dim3(256), 0, stream, stop, a);
    }
    return hipGetLastError();
}

hipError_t launch_logits(hipStream_t stream, hipEvent_t stop, const Op &op) {
    const KvParams &p = *op.kv;
    kv::LogitsArgs a;
    a.x = ptr_of<const float>(op.a[0]) + p.q_off;
    a.y = ptr_of<float>(op.a[1]) + p.out_off;
    a.history = ptr_of<const uint32_t>(op.a[2]);
    a.history_len = ptr_of<const uint32_t>(p.more[0]);
    a.penalties = ptr_of<const float>(p.more[1]);
    a.bias_ids = ptr_of<const uint32_t>(p.more[2]);
    a.bias_values = ptr_of<const float>(p.more[3]);
    a.bias_len = ptr_of<const uint32_t>(p.more[4]);
    a.allowed = ptr_of<const uint32_t>(p.more[5]);
    a.vocab = op.cols;
    a.history_stride = p.history_stride;
    a.bias_stride = p.bias_stride;
    a.allowed_stride = p.allowed_stride;
    auto tiles = [&](uint64_t tile) { return (uint32_t)((op.cols + tile - 1u) / tile); };
    const bool is_short = p.history_stride < 65536u && p.bias_stride < 65535u;
    if ((uint64_t)tiles(kv::LOGITS_LARGE) * op.rows >= kv::LOGITS_MIN_GROUPS) {
        const dim3 grid(tiles(kv::LOGITS_LARGE), op.rows);
        if (is_short) {
            Q8_LAUNCH((kv::logits_adjust_kernel<kv::LOGITS_LARGE, 512, true>), grid, dim3(512), 0, stream, stop, a);
        } else {
            Q8_LAUNCH((kv::logits_adjust_kernel<kv::LOGITS_LARGE, 512, false>), grid, dim3(512), 0, stream, stop, a);
        }
    } else {
        const dim3 grid(tiles(kv::LOGITS_SMALL), op.rows);
        if (is_short) {
            Q8_LAUNCH((kv::logits_adjust_kernel<kv::LOGITS_SMALL, 256, true>), grid, dim3(256), 0, stream, stop, a);
        } else {
            Q8_LAUNCH((kv::logits_adjust_kernel<kv::LOGITS_SMALL, 256, false>), grid, dim3(256), 0, stream, stop, a);
        }
    }
    return hipGetLastError();
}

} // namespace

hipError_t tmdev::launch_kv(hipStream_t stream, hipEvent_t stop, const Op &op) {
    switch (op.kind) {
    case OP_ROPE_STORE:
        return launch_rope(stream, stop, op);
    case OP_ATTN_DECODE:
        return launch_decode<false>(stream, stop, op);
    case OP_ATTN_PREFILL:
        return launch_prefill(stream, stop, op);
    case OP_LOGITS:
        return launch_logits(stream, stop, op);
    default:
        return hipErrorInvalidValue;
    }
}
