"""Cases, plain forms and exact values of the operators between a step's matrix products: rotary positions with the
store into the paged key-value cache, attention of single tokens and of prompt chunks over that cache, and the
adjustment of logits before a token is picked.

A cache is two buffers of pages, K as [page][kv_head][place][channel] and V as [page][kv_head][channel][place]; a
sequence is a row of a page table and a length. Activations are f32, pages f16 or f32.
"""
import math
import random

import numpy as np
import torch

own = False

_F16, _F32 = 1, 0  # the cache's type ids
_DT = {_F16: torch.float16, _F32: torch.float32}


def listed():
    return [
        # one token of a decode step (a 0.6B-class model's heads): latency
        {"name": "rope-1-token", "op": "rope", "tokens": 1, "q_heads": 16, "kv_heads": 8, "head_dim": 128, "rot": 128,
         "axes": 1, "interleaved": False, "adjacent": False, "type": _F16, "page": 16, "fused": False, "far": 40000, "skip": 0},
        # a long prompt with images: three axes, rows of one fused projection, padded rows that store nothing
        {"name": "rope-4093-image", "op": "rope", "tokens": 4093, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "rot": 128,
         "axes": 3, "interleaved": True, "adjacent": False, "type": _F16, "page": 64, "fused": True, "far": 200000, "skip": 5},
        # a chat's next token: latency
        {"name": "decode-1x777", "op": "decode", "seqs": 1, "longest": 777, "ragged": False, "q_heads": 16, "kv_heads": 8,
         "head_dim": 128, "type": _F16, "page": 16, "window": 0, "cap": 0.0, "slopes": False},
        # one very long context
        {"name": "decode-1x131071", "op": "decode", "seqs": 1, "longest": 131071, "ragged": False, "q_heads": 32, "kv_heads": 8,
         "head_dim": 128, "type": _F16, "page": 64, "window": 0, "cap": 0.0, "slopes": False},
        # a serving batch of requests of all lengths
        {"name": "decode-48-ragged", "op": "decode", "seqs": 48, "longest": 8192, "ragged": True, "q_heads": 32, "kv_heads": 8,
         "head_dim": 128, "type": _F16, "page": 32, "window": 0, "cap": 0.0, "slopes": False},
        # a 1B-class model with one key head of 256 channels: f32 pages, capped scores, a sliding window
        {"name": "decode-16-f32-window", "op": "decode", "seqs": 16, "longest": 6000, "ragged": True, "q_heads": 4, "kv_heads": 1,
         "head_dim": 256, "type": _F32, "page": 128, "window": 4096, "cap": 50.0, "slopes": False},
        # the few rows of speculative verification, over long caches
        {"name": "prefill-19-on-cached", "op": "prefill", "seqs": 4, "new": 19, "cached": 5000, "pad": 0, "q_heads": 16,
         "kv_heads": 8, "head_dim": 128, "type": _F16, "page": 16, "window": 0, "cap": 0.0, "slopes": False, "docs": False,
         "prefix": False},
        # a long prompt in one call
        {"name": "prefill-8192", "op": "prefill", "seqs": 1, "new": 8192, "cached": 0, "pad": 0, "q_heads": 32, "kv_heads": 8,
         "head_dim": 128, "type": _F16, "page": 64, "window": 0, "cap": 0.0, "slopes": False, "docs": False, "prefix": False},
        # packed prompts of several documents each, distance bias, capped, a padded batch
        {"name": "prefill-4001-docs", "op": "prefill", "seqs": 6, "new": 4001, "cached": 700, "pad": 31, "q_heads": 24, "kv_heads": 8,
         "head_dim": 64, "type": _F16, "page": 32, "window": 0, "cap": 30.0, "slopes": True, "docs": True, "prefix": False},
        # prompts whose image or instruction prefix sees itself both ways: f32 pages, 256 channels
        {"name": "prefill-1500-prefix-f32", "op": "prefill", "seqs": 2, "new": 1500, "cached": 100, "pad": 0, "q_heads": 4,
         "kv_heads": 1, "head_dim": 256, "type": _F32, "page": 128, "window": 1024, "cap": 50.0, "slopes": False, "docs": False,
         "prefix": True},
        # one chat's logits over a 0.6B-class vocabulary: latency
        {"name": "logits-1", "op": "logits", "rows": 1, "vocab": 151936, "history": 700, "biases": 0, "mask": False},
        # a serving batch with grammars and biases
        {"name": "logits-64-grammar", "op": "logits", "rows": 64, "vocab": 151936, "history": 4096, "biases": 300, "mask": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_HEADS = [(16, 8, 128), (32, 8, 128), (4, 1, 256), (24, 8, 64), (12, 12, 64), (40, 8, 128), (64, 8, 128), (32, 32, 80), (9, 3, 96),
          (32, 2, 128), (20, 1, 64), (8, 4, 192)]


def draw(rng):
    op = rng.choice(["rope", "decode", "decode", "prefill", "prefill", "logits"])
    q_heads, kv_heads, head_dim = rng.choice(_HEADS)
    heads = {"q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim}
    kind, page = rng.choice([_F16, _F16, _F32]), rng.choice([16, 32, 64, 128, 256])
    if op == "rope":
        axes, rot = rng.choice([1, 2, 3, 4]), rng.choice([head_dim, head_dim // 2])
        most = min(4093, 4093 * 48 * 128 // ((q_heads + 2 * kv_heads) * head_dim))
        return {"op": op, "tokens": _log(rng, 1, most), **heads, "rot": rot, "axes": axes, "interleaved": rng.random() < 0.5,
                "adjacent": rng.random() < 0.5, "type": kind, "page": page, "fused": rng.random() < 0.5,
                "far": _log(rng, 100, 4000000), "skip": rng.choice([0, 1, 3])}
    cap, slopes = rng.choice([0.0, 0.0, 20.0, 50.0]), rng.random() < 0.3
    per = kv_heads * head_dim * (2 if kind == _F16 else 4)  # bytes of one token's keys
    if op == "decode":
        seqs = _log(rng, 1, 64)
        longest = _log(rng, 1, min(131071, int(3.0e8 / per / seqs)))
        return {"op": op, "seqs": seqs, "longest": longest, "ragged": rng.random() < 0.7, **heads, "type": kind, "page": page,
                "window": rng.choice([0, 0, _log(rng, 1, longest + 10)]), "cap": cap, "slopes": slopes}
    if op == "prefill":
        most = 8192 * 8192 * 32 * 128 / 16  # pairs x heads x channels; f32 pages go at a tenth of the rate
        budget = most / (q_heads * head_dim) / (4 if kind == _F32 else 1)
        seqs, new = _log(rng, 1, 12), _log(rng, 1, 4000)
        new = max(seqs, min(new, int(math.sqrt(budget))))
        cached = min(_log(rng, 1, 20000), max(1, int(budget / new)), int(3.0e8 / per / seqs))
        return {"op": op, "seqs": seqs, "new": new, "cached": cached, "pad": rng.choice([0, 1, 13]), **heads, "type": kind,
                "page": page, "window": rng.choice([0, 0, _log(rng, 1, new + cached)]), "cap": cap, "slopes": slopes,
                "docs": rng.random() < 0.4, "prefix": rng.random() < 0.4}
    rows = _log(rng, 1, 64)
    return {"op": op, "rows": rows, "vocab": _log(rng, 1000, min(262144, 64 * 151936 // rows)), "history": _log(rng, 1, 8192),
            "biases": rng.choice([0, _log(rng, 1, 500)]), "mask": rng.random() < 0.5}


# ---- sizes that follow from a case alone ---------------------------------------------------------------------------------

def _dice(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _decode_lengths(case):
    r = _dice(case)
    if not case["ragged"]:
        return np.full(case["seqs"], case["longest"], np.int64)
    lens = np.array([r.randint(1, case["longest"]) for _ in range(case["seqs"])], np.int64)
    lens[r.randrange(case["seqs"])] = case["longest"]
    return lens


def _prefill_rows(case):
    """Per sequence (rows, length); per row: its sequence, position and the first position it may see; per sequence: prefix."""
    r = _dice(case)
    cuts = sorted(r.sample(range(1, case["new"]), case["seqs"] - 1)) if case["new"] > case["seqs"] else list(range(1, case["seqs"]))
    news = np.diff(np.array([0] + cuts + [case["new"]], np.int64))
    lens = news + np.array([r.randint(0, case["cached"]) for _ in news], np.int64)
    prefix = np.array([r.randint(0, int(n)) if case["prefix"] else 0 for n in lens], np.int64)
    seq, pos, first = [], [], []
    for s, (n, length) in enumerate(zip(news, lens)):
        p = np.arange(length - n, length)
        starts = np.array(sorted({0} | {r.randrange(int(length)) for _ in range(3)})) if case["docs"] else np.array([0])
        seq.append(np.full(n, s))
        pos.append(p)
        first.append(starts[np.searchsorted(starts, p, side="right") - 1])
    return news, lens, np.concatenate(seq), np.concatenate(pos), np.concatenate(first), prefix


def _sections(case):
    half, axes = case["rot"] // 2, case["axes"]
    rest = half - axes * (half // (axes + 1))  # the first axis (time) has the largest share
    return [rest + half // (axes + 1)] + [half // (axes + 1)] * (axes - 1)


def work(case):
    if case["op"] == "rope":
        e = 2 if case["type"] == _F16 else 4
        q, kv = case["q_heads"] * case["head_dim"], case["kv_heads"] * case["head_dim"]
        return {"bytes": case["tokens"] * (8 * q + 2 * kv * (4 + e) + 4 * case["axes"] + 4), "flops": case["tokens"] * 3 * (q + kv)}
    if case["op"] == "logits":
        n = case["rows"] * case["vocab"]
        more = case["rows"] * (4 * case["history"] + 8 * case["biases"] + (case["vocab"] // 8 if case["mask"] else 0))
        return {"bytes": 8 * n + more, "flops": 4 * n}
    e, d = 2 if case["type"] == _F16 else 4, case["head_dim"]
    if case["op"] == "decode":
        lens = _decode_lengths(case)
        seen = np.minimum(lens, case["window"]) if case["window"] else lens
        rows, pairs, read = case["seqs"], int(seen.sum()), int(seen.sum())
    else:
        _, lens, seq, pos, first, prefix = _prefill_rows(case)
        lo = np.maximum(first, pos - case["window"] + 1) if case["window"] else first
        hi = np.minimum(lens[seq], np.maximum(pos + 1, prefix[seq]))
        rows, pairs = len(seq), int(np.maximum(hi - lo, 0).sum())
        read = int(sum(max(0, hi[seq == s].max() - lo[seq == s].min()) for s in range(case["seqs"])))
    return {"bytes": read * 2 * case["kv_heads"] * d * e + rows * case["q_heads"] * d * 8, "flops": pairs * case["q_heads"] * d * 4}


# ---- inputs ----------------------------------------------------------------------------------------------------------------

def _cache(case, lens, gen, dev):
    """Shuffled pages for sequences of `lens` tokens, a few of them in nobody's table."""
    page, dt = case["page"], _DT[case["type"]]
    need = [-(-int(n) // page) for n in lens]
    pages, stride = sum(need) + 3, max(need + [1])
    order = torch.randperm(pages, generator=gen, device=dev).cpu().numpy()
    table, at = np.zeros((len(need), stride), np.int32), 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    shape = (pages, case["kv_heads"], page, case["head_dim"])
    k = torch.randn(shape, generator=gen, device=dev).to(dt)
    v = torch.randn((shape[0], shape[1], shape[3], shape[2]), generator=gen, device=dev).to(dt)
    return k, v, torch.from_numpy(table).to(dev)


def _ints(a, dev):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(dev)


def _inputs(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    rnd = np.random.RandomState(int(seed) % (1 << 32))
    t = {}
    if case["op"] == "logits":
        rows, vocab = case["rows"], case["vocab"]
        t["logits"] = torch.randn((rows, vocab), generator=gen, device=dev) * 4
        # a text repeats itself: ids of a skewed distribution, rows of different lengths
        ids = (torch.rand((rows, case["history"]), generator=gen, device=dev) ** 4 * vocab).to(torch.int32)
        t["history"] = torch.where(torch.rand(ids.shape, generator=gen, device=dev) < 0.02, ids[:, :1], ids)
        lens = rnd.randint(0, case["history"] + 1, rows)
        lens[0] = case["history"]
        t["history_len"] = _ints(lens, dev)
        t["penalties"] = torch.from_numpy(np.stack([rnd.uniform(1.0, 1.5, rows), rnd.uniform(0, 1, rows), rnd.uniform(0, 0.5, rows)],
                                                   1).astype(np.float32)).to(dev)
        if case["biases"]:
            t["bias_ids"] = (torch.rand((rows, case["biases"]), generator=gen, device=dev) * vocab).to(torch.int32)
            t["bias_values"] = torch.randn((rows, case["biases"]), generator=gen, device=dev) * 5
            t["bias_len"] = _ints(rnd.randint(0, case["biases"] + 1, rows), dev)
        if case["mask"]:
            words = -(-vocab // 32)
            a, b = (torch.randint(-(1 << 31), 1 << 31, (rows, words), generator=gen, device=dev).to(torch.int32) for _ in range(2))
            t["allowed"] = a & b
        t["out"] = torch.zeros((rows, vocab), device=dev)
        return t
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "rope":
        n = case["tokens"]
        t["k_cache"], t["v_cache"], _ = _cache(case, [n + 5], gen, dev)
        if case["fused"]:
            t["qkv"] = torch.randn((n, (hq + 2 * hkv) * d), generator=gen, device=dev)
        else:
            for name, h in (("q", hq), ("k", hkv), ("v", hkv)):
                t[name] = torch.randn((n, h * d), generator=gen, device=dev)
        t["positions"] = torch.randint(0, case["far"], (case["axes"], n), generator=gen, device=dev).to(torch.int32)
        i = np.arange(case["rot"] // 2)
        t["freqs"] = torch.from_numpy((1e6 ** (-2.0 * i / case["rot"])).astype(np.float32)).to(dev)
        # consecutive places of pages in any order, from somewhere in the first of them
        pages = rnd.permutation(t["k_cache"].shape[0])
        slots = (pages[:, None].astype(np.int64) * case["page"] + np.arange(case["page"])).reshape(-1)
        slots = slots[rnd.randint(0, 2 * case["page"]):][:n]
        slots[rnd.randint(0, n, case["skip"] if n > 1 else 0)] = -1
        t["slots"] = _ints(slots, dev)
        t["q_out"] = torch.zeros((n, hq * d), device=dev)
        return t
    if case["op"] == "decode":
        lens, rows = _decode_lengths(case), case["seqs"]
    else:
        news, lens, seq, pos, first, prefix = _prefill_rows(case)
        rows = len(seq) + case["pad"]
        t["starts"] = _ints(np.concatenate([[0], np.cumsum(news)]), dev)
        if case["docs"]:
            t["first"] = _ints(np.concatenate([first, np.zeros(case["pad"])]), dev)
        if case["prefix"]:
            t["prefix"] = _ints(prefix, dev)
    t["k_cache"], t["v_cache"], t["table"] = _cache(case, lens, gen, dev)
    t["lens"] = _ints(lens, dev)
    t["q"] = torch.randn((rows, hq * d), generator=gen, device=dev)
    if case["slopes"]:
        t["slopes"] = torch.from_numpy((2.0 ** (-8.0 * (1 + np.arange(hq)) / hq)).astype(np.float32)).to(dev)
    t["out"] = torch.zeros((rows, hq * d), device=dev)
    return t


def prepare(case, seed):
    state = {"case": case, "t": _inputs(case, seed)}
    if own:
        _hand_over(state)
    return state


def run(state):
    if own:
        return _OWN[state["case"]["op"]](state)
    return _PLAIN[state["case"]["op"]](state["case"], state["t"])


# ---- the framework's calls -------------------------------------------------------------------------------------------------

_context = None


def _hand_over(state):
    """The same inputs in buffers of the framework's context, and the descriptors that a program makes once."""
    global _context
    from tuckmill_amd import hip
    if _context is None:
        _context = hip.HipContext.open()
    case, bufs, views = state["case"], {}, {}
    for name, x in state.pop("t").items():
        bufs[name] = _context.buffer(x.numel() * x.element_size())
        views[name] = torch.as_tensor(bufs[name], device=x.device).view(x.dtype).view(x.shape)
        _context.fence()  # the new buffer's zero fill runs on the context's stream
        views[name].copy_(x)
    torch.cuda.synchronize()
    state["b"], state["v"] = bufs, views
    if case["op"] == "logits":
        state["spec"] = hip.LogitsAdjust(**{n: bufs.get(n) for n in ("history", "history_len", "penalties", "bias_ids", "bias_values",
                                                                    "bias_len", "allowed")},
                                         history_stride=case["history"], bias_stride=case["biases"],
                                         allowed_stride=-(-case["vocab"] // 32))
        return
    state["cache"] = hip.KvCache(bufs["k_cache"], bufs["v_cache"], case["type"], views["k_cache"].shape[0], case["page"],
                                 case["kv_heads"], case["head_dim"])
    if case["op"] == "rope":
        state["spec"] = hip.Rope(bufs["freqs"], case["rot"], _sections(case), interleaved=case["interleaved"],
                                 adjacent=case["adjacent"])
    else:
        state["spec"] = hip.Attention(case["head_dim"] ** -0.5, softcap=case["cap"], window=case["window"],
                                      slopes=bufs.get("slopes"), first=bufs.get("first"), prefix=bufs.get("prefix"))


def _own_rope(state):
    case, b, v = state["case"], state["b"], state["v"]
    q, kv = case["q_heads"] * case["head_dim"], case["kv_heads"] * case["head_dim"]
    if case["fused"]:
        rows = {"k_off": q, "v_off": q + kv, "q_stride": q + 2 * kv, "k_stride": q + 2 * kv, "v_stride": q + 2 * kv}
        x = (b["qkv"], b["qkv"], b["qkv"])
    else:
        rows, x = {}, (b["q"], b["k"], b["v"])
    _context.rope_store(state["spec"], state["cache"], *x, b["q_out"], b["positions"], b["slots"], case["tokens"], case["q_heads"],
                        **rows)
    return v["q_out"], v["k_cache"], v["v_cache"]


def _own_decode(state):
    case, b = state["case"], state["b"]
    _context.attn_decode(state["spec"], state["cache"], b["q"], b["table"], b["lens"], b["out"], case["seqs"], case["q_heads"],
                         state["v"]["table"].shape[1])
    return state["v"]["out"]


def _own_prefill(state):
    case, b = state["case"], state["b"]
    _context.attn_prefill(state["spec"], state["cache"], b["q"], b["table"], b["lens"], b["starts"], b["out"],
                          state["v"]["q"].shape[0], case["seqs"], case["q_heads"], state["v"]["table"].shape[1])
    return state["v"]["out"]


def _own_logits(state):
    _context.logits_adjust(state["spec"], state["b"]["logits"], state["b"]["out"], state["case"]["rows"], state["case"]["vocab"])
    return state["v"]["out"]


_OWN = {"rope": _own_rope, "decode": _own_decode, "prefill": _own_prefill, "logits": _own_logits}


# ---- plain forms -----------------------------------------------------------------------------------------------------------

def _axis_of_pair(case):
    """Which axis turns pair i: section after section, or the axes in turn until their sections are used up."""
    sections = _sections(case)
    if not case["interleaved"]:
        return sum(([a] * n for a, n in enumerate(sections)), [])
    return [a for _, a in sorted((turn, a) for a, n in enumerate(sections) for turn in range(n))]


def _rope_rows(case, t):
    q, kv = case["q_heads"] * case["head_dim"], case["kv_heads"] * case["head_dim"]
    return torch.split(t["qkv"], [q, kv, kv], dim=1) if case["fused"] else (t["q"], t["k"], t["v"])


def _plain_rope(case, t):
    n, d, rot = case["tokens"], case["head_dim"], case["rot"]
    q, k, v = (x.reshape(n, -1, d) for x in _rope_rows(case, t))
    pos = t["positions"][torch.tensor(_axis_of_pair(case), device=q.device)]  # [pair, token]
    angle = pos.t().double() * t["freqs"].double()
    c, s = torch.cos(angle).float().unsqueeze(1), torch.sin(angle).float().unsqueeze(1)

    def turn(x):
        y = x.clone()
        a, b = (slice(0, rot, 2), slice(1, rot, 2)) if case["adjacent"] else (slice(0, rot // 2), slice(rot // 2, rot))
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., b] * c + x[..., a] * s
        return y

    slots = t["slots"].long()
    kept = slots >= 0
    page, place = slots[kept] // case["page"], slots[kept] % case["page"]
    t["k_cache"][page, :, place] = turn(k)[kept].to(t["k_cache"].dtype)
    t["v_cache"][page, :, :, place] = v[kept].to(t["v_cache"].dtype)
    return turn(q).reshape(n, -1), t["k_cache"], t["v_cache"]


def _plain_rows(case, t, q, pos, first, prefix):
    """Attention of q [seq, row, q_head, channel] at positions pos [seq, row] over each sequence's cache."""
    seqs, rows, hq, d = q.shape
    hkv, length = case["kv_heads"], int(t["table"].shape[1]) * case["page"]
    pages = t["table"].long()
    k = t["k_cache"][pages].float().permute(0, 2, 1, 3, 4).reshape(seqs, hkv, length, d)
    v = t["v_cache"][pages].float().permute(0, 2, 1, 4, 3).reshape(seqs, hkv, length, d)
    x = q.reshape(seqs, rows, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(seqs, hkv, rows * (hq // hkv), d)
    x = torch.matmul(x, k.transpose(2, 3).contiguous()) * d ** -0.5
    x = x.reshape(seqs, hkv, rows, hq // hkv, length)
    if case["cap"]:
        x = torch.tanh(x / case["cap"]) * case["cap"]
    j = torch.arange(length, device=q.device)
    if case["slopes"]:
        x = x - t["slopes"].reshape(1, hkv, 1, -1, 1) * (pos.unsqueeze(-1) - j).abs().reshape(seqs, 1, rows, 1, length)
    lo = torch.maximum(first, pos - case["window"] + 1) if case["window"] else first
    hi = torch.minimum(torch.maximum(pos + 1, prefix.unsqueeze(1)), t["lens"].long().unsqueeze(1))
    seen = ((j >= lo.unsqueeze(-1)) & (j < hi.unsqueeze(-1))).reshape(seqs, 1, rows, 1, length)
    x = x.masked_fill(~seen, -math.inf)
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(top == -math.inf, 0, top))
    total = x.sum(-1, keepdim=True)
    x = x / torch.where(total == 0, 1, total)
    y = torch.matmul(x.reshape(seqs, hkv, -1, length), v)
    return y.reshape(seqs, hkv, rows, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(seqs, rows, hq * d)


def _plain_decode(case, t):
    q = t["q"].reshape(case["seqs"], 1, case["q_heads"], case["head_dim"])
    pos = t["lens"].long().unsqueeze(1) - 1
    return _plain_rows(case, t, q, pos, torch.zeros_like(pos), torch.zeros_like(pos[:, 0])).reshape(case["seqs"], -1)


def _plain_prefill(case, t):
    starts, lens = t["starts"].long(), t["lens"].long()
    news = starts[1:] - starts[:-1]
    most = case["new"] - case["seqs"] + 1  # no sequence has more rows
    i = torch.arange(most, device=starts.device)
    row = (starts[:-1].unsqueeze(1) + i).clamp(max=t["q"].shape[0] - 1)
    pos = (lens - news).unsqueeze(1) + i
    first = t["first"].long()[row] if case["docs"] else torch.zeros_like(pos)
    prefix = t["prefix"].long() if case["prefix"] else torch.zeros_like(lens)
    q = t["q"][row].reshape(case["seqs"], most, case["q_heads"], case["head_dim"])
    y = _plain_rows(case, t, q, pos, first, prefix)
    kept = i < news.unsqueeze(1)
    out = torch.zeros_like(t["out"])
    out[row[kept]] = y[kept]
    return out


def _plain_logits(case, t):
    rows, vocab = case["rows"], case["vocab"]
    x = t["logits"]
    at = torch.arange(case["history"], device=x.device)
    seen = (at < t["history_len"].unsqueeze(1)).float()
    count = torch.zeros_like(x).scatter_add_(1, t["history"].long(), seen)
    rep, presence, frequency = t["penalties"].unsqueeze(-1).unbind(1)
    y = torch.where(x > 0, x / rep, x * rep) - (presence + frequency * count)
    y = torch.where(count > 0, y, x)
    if case["biases"]:
        at = torch.arange(1, case["biases"] + 1, device=x.device).expand(rows, -1)
        at = torch.where(at <= t["bias_len"].unsqueeze(1), at, 0)
        last = torch.zeros((rows, vocab), dtype=torch.long, device=x.device).scatter_reduce_(1, t["bias_ids"].long(), at, "amax")
        y = torch.where(last > 0, y + t["bias_values"].gather(1, (last - 1).clamp(min=0)), y)
    if case["mask"]:
        bits = (t["allowed"].unsqueeze(-1) >> torch.arange(32, device=x.device, dtype=torch.int32)) & 1
        y = y.masked_fill(bits.reshape(rows, -1)[:, :vocab] == 0, -math.inf)
    return y


_PLAIN = {"rope": _plain_rope, "decode": _plain_decode, "prefill": _plain_prefill, "logits": _plain_logits}


# ---- the definitions in 64 bits, one sequence and one head at a time -------------------------------------------------------

def exact(case, seed):
    t = _inputs(case, seed)
    return {"rope": _exact_rope, "decode": _exact_attention, "prefill": _exact_attention, "logits": _exact_logits}[case["op"]](case, t)


def _exact_rope(case, t):
    hq, hkv, d, rot = case["q_heads"], case["kv_heads"], case["head_dim"], case["rot"]
    n, half = case["tokens"], case["rot"] // 2
    left = _sections(case)
    axis, a = [], 0
    while len(axis) < half:  # deal the pairs out
        if left[a]:
            axis.append(a)
            left[a] -= 1
            a = (a + 1) % len(left) if case["interleaved"] else a
        else:
            a = (a + 1) % len(left)
    if case["fused"]:
        q, k, v = (t["qkv"][:, i:j].double() for i, j in ((0, hq * d), (hq * d, (hq + hkv) * d), ((hq + hkv) * d, (hq + 2 * hkv) * d)))
    else:
        q, k, v = t["q"].double(), t["k"].double(), t["v"].double()
    angles = [t["positions"][axis[i]].double() * float(t["freqs"][i]) for i in range(half)]
    outs = []
    for x, h in ((q, hq), (k, hkv)):
        y = x.clone().reshape(n, h, d)
        for i in range(half):
            i0, i1 = (2 * i, 2 * i + 1) if case["adjacent"] else (i, i + half)
            z = torch.complex(y[:, :, i0].clone(), y[:, :, i1].clone()) * torch.exp(1j * angles[i]).unsqueeze(1)
            y[:, :, i0], y[:, :, i1] = z.real, z.imag
        outs.append(y)
    kc, vc = t["k_cache"].double(), t["v_cache"].double()
    for row, slot in enumerate(t["slots"].tolist()):
        if slot >= 0:
            kc[slot // case["page"], :, slot % case["page"]] = outs[1][row]
            vc[slot // case["page"], :, :, slot % case["page"]] = v[row].reshape(hkv, d)
    return outs[0].reshape(n, hq * d), kc, vc


def _exact_attention(case, t):
    hq, hkv, d, page = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
    out = torch.zeros(t["out"].shape, dtype=torch.float64, device=t["out"].device)
    starts = t["starts"].tolist() if case["op"] == "prefill" else list(range(case["seqs"] + 1))
    for s, length in enumerate(t["lens"].tolist()):
        r0, r1 = starts[s], starts[s + 1]
        used = t["table"][s, :-(-length // page)].long()
        p = torch.arange(length - (r1 - r0), length, device=out.device)
        lo = t["first"][r0:r1].long() if case.get("docs") else torch.zeros_like(p)
        if case["window"]:
            lo = torch.maximum(lo, p + 1 - case["window"])
        hi = p + 1
        if case.get("prefix"):
            hi = hi.clamp(min=int(t["prefix"][s]))
        j = torch.arange(length, device=out.device)
        hidden = (j[None, :] < lo[:, None]) | (j[None, :] >= hi[:, None])
        for h in range(hkv):
            keys = t["k_cache"][used, h].double().reshape(-1, d)[:length]
            values = t["v_cache"][used, h].double().transpose(1, 2).reshape(-1, d)[:length]
            for g in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                x = t["q"][r0:r1, g * d:(g + 1) * d].double() @ keys.t().contiguous() / math.sqrt(d)
                if case["cap"]:
                    x = case["cap"] * torch.tanh(x / case["cap"])
                if case["slopes"]:
                    x = x - float(t["slopes"][g]) * (p[:, None] - j[None, :]).abs()
                x[hidden] = -math.inf
                w = torch.nan_to_num(torch.softmax(x, 1), nan=0.0)  # a row that sees nothing
                out[r0:r1, g * d:(g + 1) * d] = w @ values
    return out


def _exact_logits(case, t):
    x = t["logits"].double().cpu().numpy()
    y = x.copy()
    for r in range(case["rows"]):
        n = int(t["history_len"][r])
        ids, times = np.unique(t["history"][r, :n].cpu().numpy(), return_counts=True)
        rep, presence, frequency = (float(p) for p in t["penalties"][r])
        z = x[r, ids]
        y[r, ids] = np.where(z > 0, z / rep, z * rep) - presence - frequency * times
        if case["biases"]:
            m = int(t["bias_len"][r])
            named = dict(zip(t["bias_ids"][r, :m].tolist(), t["bias_values"][r, :m].double().tolist()))
            y[r, list(named.keys())] += np.array(list(named.values()))
        if case["mask"]:
            bits = np.unpackbits(t["allowed"][r].cpu().numpy().view(np.uint8), bitorder="little")[:case["vocab"]]
            y[r, bits == 0] = -np.inf
    return torch.from_numpy(y)
