// Lifetimes of the operators between a step's products in the CPU build of
// libtm_hip's host logic, meant for the address sanitizer: the parameters and the
// buffers that a recorded operation holds beyond an ordinary operation's, through
// groups that are committed, recorded, aborted, or open when their context goes.
// Prints what is left alive at the end as one JSON object.
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <initializer_list>

#include <hip/hip_runtime.h>

#include "tm_hip.h"

namespace {

char err[512];

void ok(int rc, const char *what) {
    if (rc != TM_HIP_OK) {
        fprintf(stderr, "%s failed (%d): %s\n", what, rc, err);
        exit(2);
    }
}

struct Set {
    tm_hip_ctx *ctx;
    tm_hip_buffer *k, *v, *q, *x, *out, *small, *logits, *ids, *values, *words;
    explicit Set(tm_hip_ctx *c) : ctx(c) {
        auto make = [&](size_t n) {
            tm_hip_buffer *b = tm_hip_buffer_new(ctx, n, 1, err, sizeof err);
            if (b == nullptr) {
                fprintf(stderr, "buffer: %s\n", err);
                exit(2);
            }
            return b;
        };
        k = make(4 * 16 * 64 * 2);
        v = make(4 * 16 * 64 * 2);
        q = make(2 * 128 * 4);
        x = make(2 * 128 * 4);
        out = make(2 * 128 * 4);
        small = make(1024);
        logits = make(2 * 100 * 4);
        ids = make(1024);
        values = make(1024);
        words = make(1024);
    }
    void encode() {
        const tm_hip_kv_cache cache = {k, v, 1, 4, 16, 1, 64};
        tm_hip_rope rope = {values, 64, 1, {32, 0, 0, 0}, 0, 0};
        ok(tm_hip_rope_store_f32(ctx, &rope, &cache, q, x, x, q, ids, small, 2, 2, 0, 0, 64, 0, 0, 128, 128, 0, err,
                                 sizeof err),
           "rope_store");
        const tm_hip_attn attn = {0.125f, 30.0f, 5, values, ids, small};
        ok(tm_hip_attn_decode_f32(ctx, &attn, &cache, q, words, small, out, 2, 2, 2, 0, 0, 0, 0, err, sizeof err),
           "attn_decode");
        ok(tm_hip_attn_prefill_f32(ctx, &attn, &cache, q, words, small, ids, out, 2, 2, 2, 2, 0, 0, 0, 0, err,
                                   sizeof err),
           "attn_prefill");
        const tm_hip_logits_adjust adjust = {ids, small, values, ids, values, small, words, 3, 3, 4};
        ok(tm_hip_logits_adjust_f32(ctx, &adjust, logits, logits, 2, 100, 0, 0, err, sizeof err), "logits_adjust");
    }
    void drop() {
        for (tm_hip_buffer *b : {k, v, q, x, out, small, logits, ids, values, words}) {
            tm_hip_buffer_free(ctx, b);
        }
    }
};

} // namespace

int main() {
    tm_hip_ctx *ctx = tm_hip_create(err, sizeof err);
    if (ctx == nullptr) {
        fprintf(stderr, "create: %s\n", err);
        return 2;
    }
    {
        Set s(ctx); // each on its own
        s.encode();
        s.drop();
    }
    {
        Set s(ctx); // handles freed before the group is committed
        ok(tm_hip_begin_group(ctx, err, sizeof err), "begin");
        s.encode();
        s.encode();
        s.drop();
        ok(tm_hip_end_group(ctx, err, sizeof err), "end");
    }
    tm_hip_step *step = nullptr;
    {
        Set s(ctx); // handles freed before the step runs
        ok(tm_hip_begin_group(ctx, err, sizeof err), "begin");
        s.encode();
        ok(tm_hip_end_group_recorded(ctx, &step, err, sizeof err), "record");
        s.drop();
        ok(tm_hip_step_run(ctx, step, err, sizeof err), "run");
        ok(tm_hip_step_run(ctx, step, err, sizeof err), "run");
    }
    {
        Set s(ctx); // aborted
        ok(tm_hip_begin_group(ctx, err, sizeof err), "begin");
        s.encode();
        ok(tm_hip_abort_group(ctx, err, sizeof err), "abort");
        s.drop();
    }
    ok(tm_hip_fence(ctx, err, sizeof err), "fence");
    tm_hip_step_free(ctx, step);
    const unsigned long long live = tm_hip_allocated_bytes(ctx), leased = tm_hip_in_flight_bytes(ctx);
    Set s(ctx); // still open when the context goes
    ok(tm_hip_begin_group(ctx, err, sizeof err), "begin");
    s.encode();
    s.drop();
    tm_hip_destroy(ctx);
    printf("{\"allocated\":%llu,\"leased\":%llu}\n", live, leased);
    return 0;
}
