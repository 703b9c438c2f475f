"""Attention of whole prompts and over a 4-bit KV cache, as measurable cases.

Four operators of the library beside its single-token attention layer:

    rows    query and key rows of many tokens: RMSNorm of each head, then RoPE
            (smoe_hip_qk_norm_rope)
    prompt  causal attention of packed sequences with grouped heads
            (smoe_hip_attention_prompt)
    store   key and value rows into a 4-bit cache, and back
            (smoe_hip_kv4_append, smoe_hip_kv4_read)
    kv4     attention of one token a sequence over that cache
            (smoe_hip_attention_kv4)

    listed()             the named cases
    draw(rng)            one more case of the same ranges
    prepare(case, seed)  inputs on the GPU
    run(state)           one pass, and its outputs: in plain torch, or where
                         `own` is true by the library's entry points
    work(case)           bytes and operations that a pass cannot do without
    exact(case, seed)    the same outputs in 64 bits
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
GROUP = 64                  # values that share a scale and a min in the cache
EPS = 1e-6                  # of the RMSNorm
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
# query heads, KV heads, head_dim: the two Qwen3 layouts of the benchmark, and those of the trunk's tests
# (no grouping; wide heads; a group that is no power of two)
HEADS = {"30b": (32, 4, 128), "235b": (64, 4, 128), "mha": (8, 8, 64), "wide": (8, 2, 256), "five": (10, 2, 128)}
MOST_PAIRS = 64 * 8192 * 8192          # query heads x padded queries x padded keys of the largest prompt
MOST_CACHED = 16 * 4 * 32768 * 128     # sequences x KV heads x padded positions x head_dim of the largest cache


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def _case(kind, layout, **more):
    h, kv, d = HEADS[layout]
    return dict(kind=kind, heads=h, kv_heads=kv, head_dim=d, **more)


def listed():
    return [
        # a decode step of 17 conversations: the smallest call
        dict(_case("rows", "30b", type="f32", rows=17, fused=False), name="rows_17_30b_f32"),
        # a long prompt, its projections one matrix
        dict(_case("rows", "30b", type="bf16", rows=4096, fused=True), name="rows_4096_30b_bf16"),
        # a batch of short questions of 0 to some hundred tokens, packed
        dict(_case("prompt", "30b", type="bf16", seqs=24, tokens=1400, prefix=0, lay=3, fused=True),
             name="prompt_packed24_30b_bf16"),
        # the benchmark's prompt in the trunk's own type
        dict(_case("prompt", "30b", type="f32", seqs=1, tokens=512, prefix=0, lay=0, fused=False),
             name="prompt_512_30b_f32"),
        # a document
        dict(_case("prompt", "30b", type="bf16", seqs=1, tokens=4096, prefix=0, lay=0, fused=True),
             name="prompt_4096_30b_bf16"),
        # a long document and the large model: the largest call
        dict(_case("prompt", "235b", type="bf16", seqs=1, tokens=8192, prefix=0, lay=0, fused=False),
             name="prompt_8192_235b_bf16"),
        # one chunk of 64 tokens of a prompt that is taken in chunks, 8000 positions in
        dict(_case("prompt", "30b", type="f16", seqs=1, tokens=64, prefix=8000, lay=0, fused=False),
             name="prompt_chunk64_8000_30b_f16"),
        # a decode step's new rows of 48 conversations into the cache, and read back
        dict(_case("store", "30b", type="f32", seqs=48, rows=48, past=1500, lay=5), name="store_48_30b_f32"),
        # a batch of prompts of different lengths into the cache, and read back in the type of the prompt attention
        dict(_case("store", "235b", type="bf16", seqs=6, rows=6000, past=0, lay=7), name="store_6000_235b_bf16"),
        # one conversation some turns in
        dict(_case("kv4", "30b", type="f32", seqs=1, most=777, lay=0), name="kv4_777_30b_f32"),
        # a decode step of 32 conversations of different lengths
        dict(_case("kv4", "30b", type="bf16", seqs=32, most=8192, lay=9), name="kv4_32x8192_30b_bf16"),
        # a decode step over 16 long documents of the large model
        dict(_case("kv4", "235b", type="f32", seqs=16, most=32768, lay=0), name="kv4_16x32k_235b_f32"),
    ]


def _logint(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)) - 1e-9)))))


def draw(rng):
    kind = rng.choice(["rows", "prompt", "prompt", "prompt", "store", "kv4", "kv4"])
    layout = rng.choice(["30b", "30b", "235b", "mha", "wide", "five"])
    kind_of = rng.choice(["bf16", "bf16", "f16", "f32"])
    lay = rng.randrange(1, 1 << 20)
    if kind == "rows":
        return _case(kind, layout, type=kind_of, rows=_logint(rng, 1, 4096), fused=rng.random() < 0.5)
    if kind == "store":
        seqs = _logint(rng, 1, 64)
        return _case(kind, layout, type=kind_of, seqs=seqs, rows=max(seqs, _logint(rng, 1, 6000)),
                     past=rng.choice([0, _logint(rng, 1, 4000)]), lay=lay)
    if kind == "kv4":
        while True:
            c = _case(kind, layout, type=kind_of, seqs=_logint(rng, 1, 64), most=_logint(rng, 1, 32768),
                      lay=rng.choice([0, lay]))
            if c["seqs"] * c["kv_heads"] * c["most"] * c["head_dim"] <= MOST_CACHED:
                return c
    while True:
        c = _case(kind, layout, type=kind_of, seqs=rng.choice([1, _logint(rng, 1, 48)]), tokens=_logint(rng, 1, 8192),
                  prefix=rng.choice([0, 0, _logint(rng, 1, 16384)]), lay=lay, fused=rng.random() < 0.5)
        q, k = _lengths(c)
        if c["heads"] * len(q) * max(q) * max(k) <= MOST_PAIRS and sum(k) * c["kv_heads"] * c["head_dim"] <= 1 << 26:
            return c


def _parts(total, n, lay):
    """`total` as n lengths, some of them 0 or 1 (lay 0: as even as can be)."""
    if n == 1:
        return [total]
    if lay == 0:
        return [total // n + (i < total % n) for i in range(n)]
    r = random.Random(lay)
    w = [0.0 if r.random() < 0.06 else r.expovariate(1.0) ** 1.5 for _ in range(n)]
    w[0] += 0.01
    part = [int(total * x / sum(w)) for x in w]
    part[part.index(max(part))] += total - sum(part)
    return part


def _lengths(case):
    """Query and key lengths of a prompt's sequences: each sequence's last keys are its queries' own."""
    q = _parts(case["tokens"], case["seqs"], case["lay"])
    r = random.Random(case["lay"] + 1)
    some = case["seqs"] > 1
    k = [n + (int(case["prefix"] * r.random()) if some else case["prefix"]) for n in q]
    return q, k


def _lens(case):
    """Positions of each sequence in a cache: up to `most`, the first one all of them."""
    r = random.Random(case["lay"])
    return [case["most"] if i == 0 or case["lay"] == 0 else int(case["most"] * r.random()) for i in range(case["seqs"])]


def _past(case):
    r = random.Random(case["lay"] + 1)
    return [int(case["past"] * r.random()) for _ in range(case["seqs"])]


def _slots(case):
    """Sequence b's place in a cache of two places more than sequences: any order."""
    s = list(range(case["seqs"] + 2))
    random.Random(case["lay"] + 2).shuffle(s)
    return s[:case["seqs"]]


def _offsets(n):
    o = [0]
    for x in n:
        o.append(o[-1] + x)
    return o


def work(case):
    h, kv, d, z = case["heads"], case["kv_heads"], case["head_dim"], SIZE.get(case["type"])
    if case["kind"] == "rows":
        n = case["rows"]
        return {"bytes": 2.0 * n * (h + kv) * d * z + 4.0 * n * d, "flops": 8.0 * n * (h + kv) * d}
    if case["kind"] == "prompt":
        q, k = _lengths(case)
        pairs = sum(a * (b - a) + a * (a + 1) // 2 for a, b in zip(q, k))
        return {"bytes": float(2 * sum(q) * h * d * z + 2 * sum(k) * kv * d * z), "flops": 4.0 * pairs * h * d}
    held = d // 2 + d // GROUP * 4          # bytes of a position of one KV head, K or V
    if case["kind"] == "store":
        n = case["rows"] * kv
        return {"bytes": 2.0 * n * (2 * d * z + held), "flops": 8.0 * n * d}
    n = sum(_lens(case))
    return {"bytes": 2.0 * n * kv * held + 2.0 * case["seqs"] * h * d * z, "flops": 4.0 * n * h * d}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) & 0x7FFFFFFF)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _matrices(parts, fused):
    """The rows of q, k (and v): matrices of their own, or column ranges of one (as one projection leaves them)."""
    if not fused:
        return parts
    one, at, got = torch.cat(parts, 1), 0, []
    for p in parts:
        got.append(one[:, at:at + p.shape[1]])
        at += p.shape[1]
    return got


def _keys(g, rows, kv, d):
    """Key rows: some channels far from 0 in every position, as trained models have them."""
    away = torch.where(torch.rand(kv, d, generator=g, device=DEV) < 0.04, 3.0, 0.0) * _randn(g, kv, d)
    return (_randn(g, rows, kv, d) + away).reshape(rows, kv * d)


def _cache(case, g, capacity):
    """A cache: codes [slots, KV heads, capacity, head_dim / 2], scales and mins [.., head_dim / 64, 2], of K and V."""
    n, kv, d = case["seqs"] + 2, case["kv_heads"], case["head_dim"]
    held = {}
    for x in "kv":
        held[x + "_codes"] = torch.randint(0, 256, (n, kv, capacity, d // 2), dtype=torch.uint8, generator=g, device=DEV)
        s = 0.15 * torch.exp(0.4 * _randn(g, n, kv, capacity, d // GROUP))
        m = -s * (7.5 + 1.5 * _randn(g, n, kv, capacity, d // GROUP))
        held[x + "_params"] = torch.stack([s, m], -1).to(torch.bfloat16)
    return held


def prepare(case, seed):
    g, t = _gen(seed), TYPES[case["type"]]
    h, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
    s = {"case": case}
    if case["kind"] == "rows":
        n = case["rows"]
        q, k, v = (2.0 * _randn(g, n, x * d) for x in (h, kv, kv))
        s["q"], s["k"], _ = _matrices([x.to(t) for x in (q, k, v)], case["fused"])
        s["q_norm"], s["k_norm"] = ((1.0 + 0.3 * _randn(g, d)).to(torch.bfloat16) for _ in range(2))
        far = 8192
        turn = torch.arange(far, device=DEV, dtype=torch.float64)[:, None] / 1e6 ** (
            torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d)
        s["cos"], s["sin"] = turn.cos().float(), turn.sin().float()
        s["positions"] = torch.randint(0, far, (n,), generator=g, device=DEV).to(torch.int32)
        s["q_out"], s["k_out"] = torch.empty(n, h * d, dtype=t, device=DEV), torch.empty(n, kv * d, dtype=t, device=DEV)
    elif case["kind"] == "prompt":
        nq, nk = _lengths(case)
        oq, ok = _offsets(nq), _offsets(nk)
        q = (1.5 * _randn(g, oq[-1], h * d)).to(t)
        k, v = _keys(g, ok[-1], kv, d).to(t), _randn(g, ok[-1], kv * d).to(t)
        fused = case["fused"]
        if fused and oq == ok:
            s["q"], s["k"], s["v"] = _matrices([q, k, v], True)
        else:
            s["q"], (s["k"], s["v"]) = q, _matrices([k, v], fused)
        s["q_offsets"], s["k_offsets"] = _ints(oq), _ints(ok)
        s["nq"], s["nk"], s["max_q"], s["max_k"] = _ints(nq), _ints(nk), max(nq), max(nk)
        s["out"] = torch.empty(oq[-1], h * d, dtype=t, device=DEV)
    elif case["kind"] == "store":
        n, past, parts = case["rows"], _past(case), _parts(case["rows"], case["seqs"], case["lay"])
        if case["rows"] == case["seqs"]:
            parts = [1] * case["seqs"]
        s["k"], s["v"] = _keys(g, n, kv, d).to(t), _randn(g, n, kv * d).to(t)
        s["start"], s["offsets"], s["slots"] = _ints(past), _ints(_offsets(parts)), _ints(_slots(case))
        s["rows_of"] = _ints([b for b, p in enumerate(parts) for _ in range(p)]).long()
        s.update(_cache(case, g, max(a + b for a, b in zip(past, parts)) + 64))
        s["k_out"], s["v_out"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
        s["lens_out"] = torch.empty(case["seqs"], dtype=torch.int32, device=DEV)
    else:
        lens = _lens(case)
        s["q"] = (1.5 * _randn(g, case["seqs"], h * d)).to(t)
        s["lens"], s["slots"], s["most"] = _ints(lens), _ints(_slots(case)), max(lens)
        s.update(_cache(case, g, max(lens) + 32))
        s["out"] = torch.empty_like(s["q"])
    if own:
        s["call"] = _handle(s)
    return s


# ---------------------------------------------------------------------------
# one pass by the library's entry points
# ---------------------------------------------------------------------------
_context = None


def _handle(s):
    """The library's argument structures over the state's buffers, and the process's one context."""
    global _context
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "s-moe_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import smoe_amd
    if _context is None:
        _context = smoe_amd.Context()
        _context.set_stream(torch.cuda.current_stream().cuda_stream)
    c = s["case"]
    h, kv, d, t = c["heads"], c["kv_heads"], c["head_dim"], smoe_amd.TYPES[c["type"]]
    p = {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor)}
    st = {k: v.stride(0) for k, v in s.items() if isinstance(v, torch.Tensor) and v.dim() == 2}
    if c["kind"] == "rows":
        return smoe_amd.SmoeQkRowsArgs(
            q=p["q"], q_out=p["q_out"], k=p["k"], k_out=p["k_out"], q_norm_w=p["q_norm"], k_norm_w=p["k_norm"],
            rope_cos=p["cos"], rope_sin=p["sin"], positions=p["positions"], q_stride=st["q"],
            q_out_stride=st["q_out"], k_stride=st["k"], k_out_stride=st["k_out"], n_rows=c["rows"],
            n_positions=s["cos"].shape[0], num_heads=h, num_kv_heads=kv, head_dim=d, type=t)
    if c["kind"] == "prompt":
        return smoe_amd.SmoePromptAttnArgs(
            q=p["q"], k=p["k"], v=p["v"], out=p["out"], q_offsets=p["q_offsets"], k_offsets=p["k_offsets"],
            q_stride=st["q"], k_stride=st["k"], v_stride=st["v"], out_stride=st["out"], n_seqs=c["seqs"],
            q_rows=s["q"].shape[0], k_rows=s["k"].shape[0], max_k=s["max_k"], num_heads=h, num_kv_heads=kv,
            head_dim=d, type=t, scale=1.0 / math.sqrt(d))
    cache = smoe_amd.SmoeKv4Cache(
        k_codes=p["k_codes"], v_codes=p["v_codes"], k_params=p["k_params"], v_params=p["v_params"],
        n_slots=s["k_codes"].shape[0], capacity=s["k_codes"].shape[2], num_kv_heads=kv, head_dim=d)
    if c["kind"] == "store":
        both = dict(offsets=p["offsets"], slots=p["slots"], start=p["start"], n_seqs=c["seqs"], n_rows=c["rows"], type=t)
        return (cache, smoe_amd.SmoeKv4RowsArgs(k=p["k"], v=p["v"], k_stride=st["k"], v_stride=st["v"],
                                                lens_out=p["lens_out"], **both),
                smoe_amd.SmoeKv4RowsArgs(k=p["k_out"], v=p["v_out"], k_stride=st["k_out"], v_stride=st["v_out"], **both))
    return (cache, smoe_amd.SmoeKv4AttnArgs(
        q=p["q"], out=p["out"], slots=p["slots"], lens=p["lens"], q_stride=st["q"], out_stride=st["out"],
        n_seqs=c["seqs"], max_len=s["most"], num_heads=h, type=t, scale=1.0 / math.sqrt(d)))


def _run_own(s):
    kind, call = s["case"]["kind"], s["call"]
    if kind == "rows":
        _context.qk_norm_rope(call)
        return {"q": s["q_out"], "k": s["k_out"]}
    if kind == "prompt":
        _context.attention_prompt(call)
        return {"out": s["out"]}
    if kind == "store":
        _context.kv4_append(call[0], call[1])
        _context.kv4_read(call[0], call[2])
        return {"k": s["k_out"], "v": s["v_out"], "lens": s["lens_out"]}
    _context.attention_kv4(call[0], call[1])
    return {"out": s["out"]}


# ---------------------------------------------------------------------------
# one pass in plain torch
# ---------------------------------------------------------------------------
def _norm_rope(x, heads, d, w, cos, sin):
    x = x.float().reshape(x.shape[0], heads, d)
    x = x * (1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)) * w.float()
    a, b = x[..., :d // 2], x[..., d // 2:]
    c, n = cos[:, None], sin[:, None]
    return torch.cat([a * c - b * n, a * n + b * c], -1).reshape(x.shape[0], heads * d)


def _padded(x, offsets, n, most):
    """Packed rows [rows, cols] as [sequences, most, cols] (past a sequence's end: some row, masked later)."""
    at = offsets[:-1, None].long() + torch.arange(most, device=DEV)
    return x[at.clamp(max=x.shape[0] - 1)]


def _attend(q, k, v, may, scale):
    """q [B, KV, G, M, d], k and v [B, KV, N, d], may [B, 1, 1, M, N] -> [B, KV, G, M, d]; rows that may see nothing: 0."""
    b, kv, g, m, d = q.shape
    s = torch.matmul((q * scale).reshape(b, kv, g * m, d), k.transpose(2, 3).contiguous()).reshape(b, kv, g, m, -1)
    s = s.masked_fill_(~may, -math.inf)
    top = s.amax(-1, keepdim=True)
    e = s.sub_(torch.where(top > -math.inf, top, 0.0)).exp_()
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e.reshape(b, kv, g * m, -1), v).reshape(b, kv, g, m, d)
    return o / torch.where(total > 0, total, 1.0)


def _prompt(s):
    c = s["case"]
    h, kv, d, b = c["heads"], c["kv_heads"], c["head_dim"], c["seqs"]
    mq, mk, nq, nk = s["max_q"], s["max_k"], s["nq"], s["nk"]
    q = _padded(s["q"], s["q_offsets"], nq, mq).float().reshape(b, mq, kv, h // kv, d).permute(0, 2, 3, 1, 4)
    k, v = (_padded(s[x], s["k_offsets"], nk, mk).float().reshape(b, mk, kv, d).transpose(1, 2).contiguous()
            for x in "kv")
    i, j = torch.arange(mq, device=DEV)[:, None], torch.arange(mk, device=DEV)
    may = (j < nk[:, None, None]) & (j <= i + (nk - nq)[:, None, None])
    o = _attend(q, k, v, may[:, None, None], 1.0 / math.sqrt(d))
    o = o.permute(0, 3, 1, 2, 4).reshape(b, mq, h * d)
    live = torch.arange(mq, device=DEV) < nq[:, None]
    s["out"].copy_(o[live])
    return {"out": s["out"]}


def _quantized(x):
    """Rows [.., d] as codes of 0 to 15, scales and mins of their groups: every step rounded to 32 bits."""
    w = x.float().reshape(*x.shape[:-1], -1, GROUP)
    lo, hi = w.amin(-1), w.amax(-1)
    m = lo.to(torch.bfloat16)
    r = ((hi - lo) / torch.full_like(lo, 15.0)).to(torch.bfloat16)
    r = torch.where(r == 0, torch.ones_like(r), r)
    c = torch.round((w - m.float()[..., None]) / r.float()[..., None]).clamp(0, 15).to(torch.uint8)
    return c.reshape(x.shape), torch.stack([r, m], -1)


def _values(codes, params):
    """Codes, two a byte with the even value low, and their groups' scales and mins -> values."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    p = params.float().repeat_interleave(GROUP, -2)
    return c * p[..., 0] + p[..., 1]


def _store(s):
    c = s["case"]
    n, kv, d, b = c["rows"], c["kv_heads"], c["head_dim"], s["rows_of"]
    at = torch.arange(n, device=DEV) - s["offsets"][b] + s["start"][b]
    slot = s["slots"][b].long()
    got = {}
    for x in "kv":
        codes, params = _quantized(s[x].reshape(n, kv, d))
        s[x + "_codes"][slot, :, at] = codes[..., 0::2] | (codes[..., 1::2] << 4)
        s[x + "_params"][slot, :, at] = params
        got[x] = _values(s[x + "_codes"][slot, :, at], s[x + "_params"][slot, :, at]).reshape(n, kv * d).to(s[x].dtype)
    return {**got, "lens": s["start"] + s["offsets"][1:] - s["offsets"][:-1]}


def _kv4(s):
    c = s["case"]
    h, kv, d, b, m = c["heads"], c["kv_heads"], c["head_dim"], c["seqs"], s["most"]
    k, v = (_values(s[x + "_codes"][s["slots"].long(), :, :m], s[x + "_params"][s["slots"].long(), :, :m]) for x in "kv")
    q = s["q"].float().reshape(b, kv, h // kv, 1, d)
    may = torch.arange(m, device=DEV) < s["lens"][:, None]
    return {"out": _attend(q, k, v, may[:, None, None, None], 1.0 / math.sqrt(d)).reshape(b, h * d).to(s["q"].dtype)}


def run(state):
    if own:
        return _run_own(state)
    c = state["case"]
    if c["kind"] == "rows":
        at = state["positions"].long()
        cos, sin, t = state["cos"][at], state["sin"][at], TYPES[c["type"]]
        return {x: _norm_rope(state[x], c[n], c["head_dim"], state[x + "_norm"], cos, sin).to(t)
                for x, n in (("q", "heads"), ("k", "kv_heads"))}
    if c["kind"] == "prompt":
        return _prompt(state)
    return _store(state) if c["kind"] == "store" else _kv4(state)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _softmax64(score):
    top = score.max(-1, keepdim=True).values
    e = (score - top).exp()
    return e / e.sum(-1, keepdim=True)


def _exact_attend(q, k, v, before):
    """Causal attention of one sequence and KV head: q [n, G, d], k and v [N, d]; query i sees keys 0 .. before + i."""
    n, g, d = q.shape
    out = torch.zeros(n, g, d, dtype=torch.float64, device=DEV)
    for a in range(0, n, 1024):
        z = min(n, a + 1024)
        seen = before + z
        s = (q[a:z].reshape(-1, d) @ k[:seen].T.contiguous() / math.sqrt(d)).reshape(z - a, g, seen)
        late = torch.arange(seen, device=DEV) > before + torch.arange(a, z, device=DEV)[:, None]
        out[a:z] = (_softmax64(s.masked_fill(late[:, None], -math.inf)).reshape(-1, seen) @ v[:seen]).reshape(z - a, g, d)
    return out


def _exact_values(codes, params):
    d = 2 * codes.shape[-1]
    c = torch.zeros(*codes.shape[:-1], d, dtype=torch.float64, device=DEV)
    c[..., 0::2], c[..., 1::2] = (codes % 16).double(), (codes // 16).double()
    w = c.reshape(*codes.shape[:-1], d // GROUP, GROUP)
    return (w * params[..., 0, None].double() + params[..., 1, None].double()).reshape(c.shape)


def exact(case, seed):
    s = prepare(case, seed)
    h, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
    if case["kind"] == "rows":
        got = {}
        for x, n in (("q", h), ("k", kv)):
            r = s[x].double().reshape(-1, n, d)
            r = r / torch.sqrt(r.pow(2).sum(-1, keepdim=True) / d + EPS) * s[x + "_norm"].double()
            z = torch.complex(r[..., :d // 2], r[..., d // 2:])
            at = s["positions"].long()
            z = z * torch.complex(s["cos"][at].double(), s["sin"][at].double())[:, None]
            got[x] = torch.cat([z.real, z.imag], -1).reshape(-1, n * d)
        return got
    if case["kind"] == "prompt":
        nq, nk = _lengths(case)
        oq, ok = _offsets(nq), _offsets(nk)
        out = torch.zeros(oq[-1], kv, h // kv, d, dtype=torch.float64, device=DEV)
        for b, n in enumerate(nq):
            for j in range(kv if n else 0):
                q = s["q"][oq[b]:oq[b + 1]].double().reshape(n, kv, h // kv, d)[:, j]
                k, v = (s[x][ok[b]:ok[b + 1]].double().reshape(-1, kv, d)[:, j].contiguous() for x in "kv")
                out[oq[b]:oq[b + 1], j] = _exact_attend(q, k, v, nk[b] - n)
        return {"out": out.reshape(oq[-1], h * d)}
    if case["kind"] == "store":
        got = {"lens": None}
        for x in "kv":
            # the cache's roundings are part of its definition: scale and min have 8 bits, after one step in 32
            w = s[x].double().reshape(case["rows"], kv, d // GROUP, GROUP)
            lo, hi = w.min(-1).values, w.max(-1).values
            m = lo.float().to(torch.bfloat16).double()
            r = ((hi - lo).float().double() / 15.0).float().to(torch.bfloat16).double()
            r[r == 0] = 1.0
            c = ((w - m[..., None]).float().double() / r[..., None]).float().double().round().clamp(0, 15)
            got[x] = (c * r[..., None] + m[..., None]).reshape(case["rows"], kv * d)
        return got
    out = torch.zeros(case["seqs"], kv, h // kv, d, dtype=torch.float64, device=DEV)
    for b, n in enumerate(_lens(case)):
        slot = _slots(case)[b]
        for j in range(kv if n else 0):
            k, v = (_exact_values(s[x + "_codes"][slot, j, :n], s[x + "_params"][slot, j, :n]) for x in "kv")
            q = s["q"][b].double().reshape(kv, h // kv, d)[j]
            out[b, j] = _softmax64(q @ k.T.contiguous() / math.sqrt(d)) @ v
    return {"out": out.reshape(case["seqs"], h * d)}
