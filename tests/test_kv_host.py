"""What the host logic refuses of the operators over the paged cache and of the logits',
and the lifetimes of what they hold, without a GPU: the library's host code built with g++
against the stand-in runtime and launchers of tests/host_cpu/, the refusals through
the Python layer, the lifetimes under the address and undefined-behaviour sanitizers."""
import ctypes
import json
import os
import shutil
import subprocess

import numpy as np
import pytest

from tuckmill_amd import hip as H

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HERE = os.path.join(ROOT, "tests", "host_cpu")
CSRC = os.path.join(ROOT, "tuckmill_amd", "csrc")


def compile_host(out, flags, more=()):
    gxx = shutil.which(os.environ.get("CXX", "g++"))
    if gxx is None:
        pytest.fail("the CPU build of the host logic needs g++")
    cmd = [gxx, "-std=c++17", "-g", *flags, "-I", HERE, "-I", os.path.join(ROOT, "include"), "-I", CSRC, "-o", str(out),
           os.path.join(CSRC, "tm_hip.cpp"), os.path.join(HERE, "fake_runtime.cpp"), os.path.join(HERE, "stub_launch.cpp"),
           *more, "-lpthread"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    assert res.returncode == 0, res.stdout + res.stderr


def test_lifetimes_under_sanitizers(tmp_path):
    out = tmp_path / "kv_lifetimes"
    compile_host(out, ["-O1", "-fsanitize=address,undefined", "-fno-sanitize-recover=undefined", "-fno-omit-frame-pointer"],
                 [os.path.join(HERE, "kv_lifetimes.cpp")])
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:verify_asan_link_order=0", UBSAN_OPTIONS="halt_on_error=1")
    res = subprocess.run([str(out)], capture_output=True, text=True, timeout=120, env=env)
    assert res.returncode == 0, res.stderr[-4000:]
    assert json.loads(res.stdout.strip().splitlines()[-1]) == {"allocated": 0, "leased": 0}


@pytest.fixture(scope="module")
def ctx(tmp_path_factory):
    out = tmp_path_factory.mktemp("kv_host") / "libtm_host_logic.so"
    compile_host(out, ["-O1", "-shared", "-fPIC", "-Wl,-Bsymbolic"])
    lib = ctypes.CDLL(str(out))
    for name, (restype, argtypes) in H._SIGS.items():
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = restype, argtypes
    real, H._lib = H._lib, lib
    try:
        c = H.HipContext.open()
        yield c
        c.close()
    finally:
        H._lib = real


class Call:
    """A valid call of each entry point, in pieces that a test changes."""

    def __init__(self, ctx):
        self.ctx = ctx
        b = self.b = {n: ctx.buffer(size) for n, size in (
            ("k", 4 * 16 * 2 * 64 * 2), ("v", 4 * 16 * 2 * 64 * 2), ("q", 3 * 4 * 64 * 4), ("kx", 3 * 2 * 64 * 4),
            ("vx", 3 * 2 * 64 * 4), ("out", 3 * 4 * 64 * 4), ("pos", 2 * 3 * 4), ("slots", 12), ("freqs", 32 * 4),
            ("table", 3 * 2 * 4), ("lens", 12), ("starts", 16), ("slopes", 16), ("first", 12), ("prefix", 12),
            ("logits", 3 * 100 * 4), ("lout", 3 * 100 * 4), ("hist", 3 * 5 * 4), ("hlen", 12), ("pen", 36), ("bid", 3 * 4 * 4),
            ("bval", 3 * 4 * 4), ("blen", 12), ("words", 3 * 4 * 4))}
        self.sealed = ctx.buffer(64 * 1088)
        ctx.q8_0_pack(self.sealed, 64, 1024)
        self.cache = dict(type_id=1, pages=4, page_tokens=16, kv_heads=2, head_dim=64, k=b["k"], v=b["v"])
        self.rope = dict(freqs=b["freqs"], rot_dim=64, sections=[16, 16])
        self.attn = dict(scale=0.125, slopes=b["slopes"], first=b["first"], prefix=b["prefix"])
        self.adjust = dict(history=b["hist"], history_len=b["hlen"], penalties=b["pen"], bias_ids=b["bid"], bias_values=b["bval"],
                           bias_len=b["blen"], allowed=b["words"], history_stride=5, bias_stride=4, allowed_stride=4)

    def rope_store(self, cache={}, rope={}, **kw):
        b = self.b
        args = dict(q=b["q"], k=b["kx"], v=b["vx"], q_out=b["out"], positions=b["pos"], slots=b["slots"], tokens=3, q_heads=4)
        self.ctx.rope_store(H.Rope(**{**self.rope, **rope}), H.KvCache(**{**self.cache, **cache}), **{**args, **kw})

    def attn_decode(self, cache={}, attn={}, **kw):
        b = self.b
        args = dict(q=b["q"], table=b["table"], lens=b["lens"], out=b["out"], seqs=3, q_heads=4, table_stride=2)
        self.ctx.attn_decode(H.Attention(**{**self.attn, **attn}), H.KvCache(**{**self.cache, **cache}), **{**args, **kw})

    def attn_prefill(self, cache={}, attn={}, **kw):
        b = self.b
        args = dict(q=b["q"], table=b["table"], lens=b["lens"], starts=b["starts"], out=b["out"], tokens=3, seqs=3, q_heads=4,
                    table_stride=2)
        self.ctx.attn_prefill(H.Attention(**{**self.attn, **attn}), H.KvCache(**{**self.cache, **cache}), **{**args, **kw})

    def logits_adjust(self, adjust={}, **kw):
        args = dict(logits=self.b["logits"], out=self.b["lout"], rows=3, vocab=100)
        self.ctx.logits_adjust(H.LogitsAdjust(**{**self.adjust, **adjust}), **{**args, **kw})


@pytest.fixture(scope="module")
def call(ctx):
    return Call(ctx)


def refused(f, *args, code=None, **kw):
    with pytest.raises(H.TuckmillError) as e:
        f(*args, **kw)
    assert e.value.code == "InvalidRequest", e.value
    if code is not None:
        assert e.value.abi_code == code, e.value


U, B = H.TM_HIP_ERR_UNSUPPORTED, H.TM_HIP_ERR_BOUNDS


def test_the_calls_as_they_stand_are_accepted(call):
    for f in (call.rope_store, call.attn_decode, call.attn_prefill, call.logits_adjust):
        f()
    call.attn_decode(attn=dict(slopes=None, first=None, prefix=None))
    call.logits_adjust(adjust=dict(history=None, history_len=None, penalties=None))
    call.logits_adjust(adjust=dict(bias_ids=None, bias_values=None, bias_len=None, allowed=None))
    call.logits_adjust(out=call.b["logits"])
    call.rope_store(q_out=call.b["q"])
    call.ctx.fence()


@pytest.mark.parametrize("name", ["rope_store", "attn_decode", "attn_prefill"])
@pytest.mark.parametrize("cache,code", [
    (dict(type_id=8), U), (dict(type_id=2), U), (dict(pages=0), U), (dict(page_tokens=0), U), (dict(page_tokens=8), U),
    (dict(page_tokens=24), U), (dict(page_tokens=512), U), (dict(kv_heads=0), U), (dict(kv_heads=3), B), (dict(head_dim=0), U),
    (dict(head_dim=60), U), (dict(head_dim=264), U), (dict(pages=5), B), (dict(pages=0xffffffff), B), (dict(type_id=0), B),
    (dict(kv_heads=2000), U)])
def test_caches_that_cannot_be(call, name, cache, code):
    refused(getattr(call, name), cache=cache, code=code)


@pytest.mark.parametrize("kw,code", [
    (dict(tokens=0), U), (dict(tokens=4), B), (dict(tokens=(1 << 20) + 1), U), (dict(q_heads=0), U), (dict(q_heads=5), U),
    (dict(q_heads=6), B), (dict(q_off=1), B), (dict(k_off=1), B), (dict(v_off=0xffffffff), B), (dict(out_off=1), B),
    (dict(q_stride=255), U), (dict(k_stride=127), U), (dict(v_stride=1), U), (dict(out_stride=0xffffffff), B),
    (dict(rope=dict(rot_dim=66, sections=[33])), U), (dict(rope=dict(rot_dim=63, sections=[31])), U),
    (dict(rope=dict(rot_dim=0, sections=[0])), U), (dict(rope=dict(sections=[16, 15])), U), (dict(rope=dict(sections=[16, 17])), U),
    (dict(rope=dict(sections=[0xffffffff, 33])), U), (dict(rope=dict(sections=[])), U),
    (dict(rope=dict(sections=[16, 8, 8])), B), (dict(rope=dict(sections=[8, 8, 8, 4, 4])), U)])
def test_rope_store_refusals(call, kw, code):
    refused(call.rope_store, code=code, **kw)


def test_rope_store_operands(call, ctx):
    b = call.b
    refused(call.rope_store, q_out=b["k"])
    refused(call.rope_store, cache=dict(v=b["k"]), code=U)
    for other in ("q", "kx", "pos", "slots", "freqs"):
        big = ctx.buffer(1 << 16)
        role = dict(kx="k", pos="positions").get(other, other)
        kw = dict(rope=dict(freqs=big)) if other == "freqs" else {role: big}
        call.rope_store(**kw)
        refused(call.rope_store, cache=dict(k=big), code=U, **kw)
        if other in ("pos", "slots", "freqs"):
            refused(call.rope_store, q_out=big, code=U, **kw)
    # one buffer for all rows: side by side is accepted, in place too, any other overlap is not
    rows = ctx.buffer(3 * 512 * 4)
    side = dict(q=rows, k=rows, v=rows, q_off=0, k_off=256, v_off=384, q_stride=512, k_stride=512, v_stride=512)
    call.rope_store(**side)
    call.rope_store(q_out=rows, out_off=0, out_stride=512, **side)
    refused(call.rope_store, q_out=rows, out_off=1, out_stride=512, code=U, **side)
    refused(call.rope_store, q_out=rows, out_off=128, out_stride=256, code=U, **side)
    refused(call.rope_store, q_out=rows, out_off=0, out_stride=256, code=U, **side)
    refused(call.rope_store, q=b["q"], k=rows, v=rows, k_off=255, v_off=384, k_stride=512, v_stride=512, q_out=rows, out_stride=512,
            code=U)
    for role in ("q", "k", "v", "q_out", "positions", "slots"):
        refused(call.rope_store, code=U, **{role: call.sealed})
    refused(call.rope_store, rope=dict(freqs=call.sealed), code=U)
    refused(call.rope_store, cache=dict(k=call.sealed), code=U)


@pytest.mark.parametrize("name", ["attn_decode", "attn_prefill"])
@pytest.mark.parametrize("kw,code", [
    (dict(seqs=0), U), (dict(seqs=4), B), (dict(seqs=32769), U), (dict(q_heads=0), U), (dict(q_heads=3), U), (dict(q_heads=8), B),
    (dict(q_heads=2048), U), (dict(table_stride=0), U), (dict(table_stride=3), B), (dict(table_stride=1 << 27), U),
    (dict(table_stride=0xffffffff), U), (dict(q_off=1), B), (dict(out_off=1), B), (dict(q_stride=255), U), (dict(out_stride=257), B),
    (dict(out_stride=3), U), (dict(attn=dict(scale=float("nan"))), U), (dict(attn=dict(scale=float("inf"))), U),
    (dict(attn=dict(softcap=-1.0)), U), (dict(attn=dict(softcap=float("nan"))), U), (dict(attn=dict(softcap=float("inf"))), U)])
def test_attention_refusals(call, name, kw, code):
    if kw.get("seqs") == 4 and name == "attn_decode":
        code = B
    refused(getattr(call, name), code=code, **kw)


def test_prefill_refusals(call):
    refused(call.attn_prefill, tokens=0, code=U)
    refused(call.attn_prefill, tokens=4, code=B)
    refused(call.attn_prefill, tokens=(1 << 20) + 1, code=U)


@pytest.mark.parametrize("name", ["attn_decode", "attn_prefill"])
def test_attention_operands(call, ctx, name):
    f, b = getattr(call, name), call.b
    big = ctx.buffer(1 << 16)
    roles = ["q", "table", "lens"] + (["starts"] if name == "attn_prefill" else [])
    for kw in [{r: big} for r in roles] + [dict(cache=dict(k=big)), dict(cache=dict(v=big))] + \
            [dict(attn={r: big}) for r in ("slopes", "first", "prefix")]:
        f(**kw)
        refused(f, out=big, code=U, **kw)
    small = ctx.buffer(8)
    for kw in [{r: small} for r in roles + ["out"]] + [dict(cache=dict(k=small)), dict(cache=dict(v=small))] + \
            [dict(attn={r: small}) for r in ("slopes", "first", "prefix")]:
        refused(f, code=B, **kw)
    for kw in [{r: call.sealed} for r in roles + ["out"]] + [dict(cache=dict(k=call.sealed))] + \
            [dict(attn={r: call.sealed}) for r in ("slopes", "first", "prefix")]:
        refused(f, code=U, **kw)
    other = H.HipContext.open()
    foreign = other.buffer(1 << 16)
    for kw in [{r: foreign} for r in roles + ["out"]] + [dict(cache=dict(v=foreign)), dict(attn=dict(first=foreign))]:
        refused(f, code=U, **kw)
    gone = ctx.buffer(1 << 16)
    spec = dict(attn=dict(slopes=gone))
    f(**spec)
    gone.free()
    refused(f, code=U, **spec)
    foreign.free()
    other.close()


@pytest.mark.parametrize("kw,code", [
    (dict(rows=0), U), (dict(rows=4), B), (dict(rows=32769), U), (dict(vocab=0), U), (dict(vocab=101), B), (dict(vocab=0xffffffff), U),
    (dict(x_off=1), B), (dict(y_off=1), B), (dict(adjust=dict(history=None)), U), (dict(adjust=dict(history_len=None)), U),
    (dict(adjust=dict(penalties=None)), U), (dict(adjust=dict(bias_ids=None)), U), (dict(adjust=dict(bias_values=None)), U),
    (dict(adjust=dict(bias_len=None)), U), (dict(adjust=dict(history_stride=0)), U), (dict(adjust=dict(history_stride=6)), B),
    (dict(adjust=dict(bias_stride=0)), U), (dict(adjust=dict(bias_stride=5)), B), (dict(adjust=dict(allowed_stride=3)), U),
    (dict(adjust=dict(allowed_stride=5)), B)])
def test_logits_refusals(call, kw, code):
    refused(call.logits_adjust, code=code, **kw)


def test_logits_operands(call, ctx):
    big = ctx.buffer(1 << 16)
    for role in ("history", "history_len", "penalties", "bias_ids", "bias_values", "bias_len", "allowed"):
        call.logits_adjust(adjust={role: big})
        refused(call.logits_adjust, adjust={role: big}, out=big, code=U)
        refused(call.logits_adjust, adjust={role: call.sealed}, code=U)
        refused(call.logits_adjust, adjust={role: ctx.buffer(4)}, code=B)
    call.logits_adjust(logits=big, out=big, x_off=0, y_off=300)
    refused(call.logits_adjust, logits=big, out=big, x_off=0, y_off=299, code=U)
    refused(call.logits_adjust, logits=call.sealed, code=U)


def test_null_context_and_descriptions(call, ctx):
    lib, err = H.load_library(), ctypes.create_string_buffer(H.ERR_CAP)
    raw = [call.b[n].raw for n in ("q", "table", "lens", "out")]
    cache = H.KvCache(**call.cache)
    assert lib.tm_hip_attn_decode_f32(None, None, None, *raw, 3, 4, 2, 0, 0, 0, 0, err, H.ERR_CAP) == U
    assert b"null context" in err.value
    assert lib.tm_hip_attn_decode_f32(ctx.raw, None, cache.desc(), *raw, 3, 4, 2, 0, 0, 0, 0, err, H.ERR_CAP) == U
    assert lib.tm_hip_attn_decode_f32(ctx.raw, H.Attention(1.0).desc(), None, *raw, 3, 4, 2, 0, 0, 0, 0, err, H.ERR_CAP) == U
    six = [call.b[n].raw for n in ("q", "kx", "vx", "out", "pos", "slots")]
    assert lib.tm_hip_rope_store_f32(ctx.raw, None, cache.desc(), *six, 3, 4, *[0] * 8, err, H.ERR_CAP) == U
    assert lib.tm_hip_rope_store_f32(None, None, None, *six, 3, 4, *[0] * 8, None, 0) == U
    assert lib.tm_hip_logits_adjust_f32(ctx.raw, None, raw[0], raw[3], 1, 10, 0, 0, err, H.ERR_CAP) == U
    assert lib.tm_hip_attn_prefill_f32(None, None, None, *[None] * 5, 1, 1, 1, 1, 0, 0, 0, 0, err, H.ERR_CAP) == U
    assert lib.tm_hip_buffer_contents(None, None) is None and lib.tm_hip_buffer_contents(ctx.raw, None) is None
    assert lib.tm_hip_buffer_contents(ctx.raw, call.sealed.raw) is None
    assert lib.tm_hip_buffer_contents(ctx.raw, raw[0]) is not None


def test_refused_calls_leave_an_open_group_as_it_was(call, ctx):
    ctx.begin_group()
    call.attn_decode()
    refused(call.attn_decode, seqs=0)
    call.rope_store()
    ctx.end_group()
    ctx.fence()
    assert np.isfinite(ctx.last_gpu_ms())


PLAN = r"""
#include "kv_plan.hpp"
#include <cstdio>
#include <random>
#include <vector>
#define CHECK(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
int main() {
    std::mt19937_64 r(5);
    auto up_to = [&](uint64_t n) { return r() % n + 1u; };
    for (int i = 0; i < 200000; ++i) {
        const uint32_t type = r() % 2u, kv = 1u << r() % 8u, group = up_to(16), d = 8u * up_to(32), cols = kv::decode_cols(type);
        const uint32_t seqs = up_to(r() % 2u ? 8u : 600u), tokens = up_to(r() % 2u ? 64u : 20000u);
        const uint64_t positions = 16u * up_to(r() % 2u ? 16u : 1u << 20);
        const kv::AttnPlan p = i % 2 ? kv::prefill_plan(type, seqs, tokens, kv * group, kv, d, positions)
                                     : kv::decode_plan(type, seqs, kv * group, kv, d, positions);
        if (p.tiled) { // every tile and part has a slot of its own
            CHECK(type == 1u && p.splits >= 1u && p.splits <= kv::PREFILL_MAX_SPLITS);
            CHECK(p.tile_bound >= ((uint64_t)tokens * group + 127u) / 128u && p.tile_bound <= (uint64_t)tokens * group);
            CHECK(p.splits == 1u || (p.arrivals == p.tile_bound * kv && p.partial_floats == p.arrivals * p.splits * 128u * (d + 2u)));
            continue;
        }
        if (p.shares == 0u) {
            CHECK(i % 2 == 0 && seqs > kv::DECODE_MAX_SEQS);
            continue;
        }
        // sequences of any rows and steps, as the kernel deals them out
        std::vector<uint64_t> units, steps;
        uint64_t total = 0, left = tokens;
        for (uint32_t s = 0; s < seqs; ++s) {
            const uint64_t rows = i % 2 ? std::min<uint64_t>(left, r() % (2u * tokens / seqs + 2u)) : 1u;
            left -= i % 2 ? rows : 0u;
            units.push_back(i % 2 ? (rows * group + cols - 1u) / cols * kv : (group + cols - 1u) / cols * kv);
            const uint64_t n = r() % 3u ? r() % 5u * r() % (positions + 1u) : positions, tile = 4u * (type ? 32u : 16u);
            steps.push_back(std::max<uint64_t>(1u, (std::min(n, positions) + tile - 1u) / tile));
            total += units.back() * steps.back();
        }
        const uint64_t size = std::max<uint64_t>(1u, (total + p.shares - 1u) / p.shares);
        uint64_t groups = 0, slots = 0;
        for (uint32_t s = 0; s < seqs; ++s) {
            const uint64_t parts = (steps[s] + size - 1u) / size;
            groups += units[s] * parts;
            slots += parts > 1u ? units[s] * parts : 0u;
        }
        CHECK(groups <= p.grid);
        CHECK(slots <= p.arrivals && p.partial_floats == p.arrivals * cols * (d + 2u));
    }
    return 0;
}
"""


def test_shares_fit_the_launch_and_the_workspace(tmp_path):
    """Any sequences a call may hold: as many workgroups as are launched have their shares, and parts
    that others have a part beside have a slot."""
    src, out = tmp_path / "plan.cpp", tmp_path / "plan"
    src.write_text(PLAN)
    gxx = shutil.which(os.environ.get("CXX", "g++"))
    res = subprocess.run([gxx, "-std=c++17", "-O2", "-I", CSRC, "-o", str(out), str(src)], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    res = subprocess.run([str(out)], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0, res.stdout
