"""The row, prompt and 4-bit-cache calls as a program makes them: a prompt at once
against the single-token layer; prompts taken in chunks into a 4-bit cache and decode
steps after them, eager and as one captured step; contexts at once on streams of their
own; graphs that share a context's scratch.

Bound of the 4-bit steps against attention over the rows themselves: with dk, dv the
rows' errors in the cache (read back exactly), a score moves by at most
ds = scale max_j sum |q dk_j|, so the result by (e^(2 ds) - 1) A + sum w |dv| at most,
A = sum w |v| over the cache's values."""
import numpy as np
import pytest
import torch

import smoe_amd
from attention_ref import (DT, Cache, fused, gen, half_step, i32, kv4_64, kv4_args, offsets, prompt64, prompt_args, randn,
                           worst)
from gpu_helpers import rel_err
from test_gpu_kv4 import rows_args
from test_gpu_qk_rows import args as qk_args, exact, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv,hd,n", [(8, 2, 128, 40), (4, 4, 64, 33), (4, 1, 256, 17)])
def test_a_prompt_at_once_is_its_tokens_one_by_one(ctx, heads, kv, hd, n):
    d, qd, kd = 256, heads * hd, kv * hd
    g = gen(heads + hd)
    w = {x: (0.06 * randn(g, *s)).to(torch.bfloat16) for x, s in
         dict(q=(qd, d), k=(kd, d), v=(kd, d), o=(d, qd)).items()}
    qw, kw = ((1 + 0.3 * randn(g, hd)).to(torch.bfloat16) for _ in range(2))
    cos, sin = tables(hd, 64)
    x = randn(g, n, d)
    buf = [torch.zeros(m, device="cuda") for m in (qd, kd, kd, qd, d)]
    kc, vc = torch.zeros(64, kd, device="cuda"), torch.zeros(64, kd, device="cuda")
    one = torch.empty(n, d, device="cuda")
    a = smoe_amd.SmoeAttnLayerArgs(
        w_q=w["q"].data_ptr(), w_k=w["k"].data_ptr(), w_v=w["v"].data_ptr(), w_o=w["o"].data_ptr(),
        q_norm_w=qw.data_ptr(), k_norm_w=kw.data_ptr(), qbuf=buf[0].data_ptr(), kbuf=buf[1].data_ptr(),
        vbuf=buf[2].data_ptr(), attn_out=buf[3].data_ptr(), o_out=buf[4].data_ptr(), k_cache=kc.data_ptr(),
        v_cache=vc.data_ptr(), d_model=d, q_dim=qd, kv_dim=kd, head_dim=hd, num_heads=heads, num_kv_heads=kv,
        attn_ctx=64, attn_scale=hd ** -0.5)
    for i in range(n):
        a.normed_in, a.rope_cos, a.rope_sin = x[i].data_ptr(), cos[i].data_ptr(), sin[i].data_ptr()
        a.slot, a.valid = i, i + 1
        ctx.attention_layer(a)
        one[i] = buf[4]
    q, k, v = ((x.double() @ w[m].double().T.contiguous()).float() for m in "qkv")
    q, k, v = fused([q, k, v])
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    ctx.qk_norm_rope(qk_args(q, k, q, k, qw, kw, cos, sin, pos, heads, kv, hd, "f32"))
    out = torch.empty(n, qd, device="cuda")
    ctx.attention_prompt(prompt_args(q, k, v, out, i32([0, n]), None, heads, kv, hd, "f32", hd ** -0.5, n))
    ctx.synchronize()
    assert rel_err(k.cpu().numpy(), kc[:n].cpu().numpy())[0] <= 1e-4
    got = (out.double() @ w["o"].double().T.contiguous()).float()
    e = rel_err(got.cpu().numpy(), one.cpu().numpy())[0]
    print(f"prompt of {n} against {n} tokens, {heads}/{kv} x {hd}: {e:.2e}")
    assert e <= 1e-3


class Conversations:
    """Packed rows of sequences, their cache and what is needed to attend to them."""

    def __init__(self, ctx, t, heads=8, kv=2, hd=128, slots=(2, 0, 3), capacity=400, seed=1):
        self.ctx, self.t, self.heads, self.kv, self.hd, self.slots = ctx, t, heads, kv, hd, slots
        g = self.g = gen(seed)
        self.cache = Cache(g, max(slots) + 1, kv, capacity, hd)
        self.qw, self.kw = ((1 + 0.3 * randn(g, hd)).to(torch.bfloat16) for _ in range(2))
        self.cos, self.sin = tables(hd, capacity)
        self.scale = hd ** -0.5
        self.at = i32(slots)
        self.lens = i32([0] * len(slots))
        self.next = torch.zeros_like(self.lens)
        self.k = [torch.zeros(0, kv * hd, device="cuda", dtype=DT[t]) for _ in slots]
        self.v = [x.clone() for x in self.k]

    def rows(self, n):
        """n rows of q, k, v as a fused projection leaves them."""
        return fused([randn(self.g, n, m * self.hd).to(DT[self.t]) for m in (self.heads, self.kv, self.kv)])

    def rotate(self, q, k, pos):
        self.ctx.qk_norm_rope(qk_args(q, k, q, k, self.qw, self.kw, self.cos, self.sin, pos, self.heads, self.kv, self.hd,
                                      self.t))

    def chunk(self, n):
        """The next n[b] tokens of every sequence."""
        past = self.lens.tolist()
        q, k, v = self.rows(sum(n))
        pos = i32([p + i for p, m in zip(past, n) for i in range(m)])
        self.rotate(q, k, pos)
        offs = i32(offsets(n))
        self.ctx.kv4_append(self.cache.struct(), rows_args(k, v, self.lens, self.t, offs, self.at, self.next))
        nk = [p + m for p, m in zip(past, n)]
        ko, vo = (torch.empty(sum(nk), self.kv * self.hd, dtype=DT[self.t], device="cuda") for _ in range(2))
        koffs, zero = i32(offsets(nk)), i32([0] * len(n))
        self.ctx.kv4_read(self.cache.struct(), rows_args(ko, vo, zero, self.t, koffs, self.at))
        out = torch.empty(sum(n), self.heads * self.hd, dtype=DT[self.t], device="cuda")
        self.ctx.attention_prompt(prompt_args(q, ko, vo, out, offs, koffs, self.heads, self.kv, self.hd, self.t, self.scale,
                                              max(nk)))
        self.lens.copy_(self.next)
        self.ctx.synchronize()
        ref, tol = prompt64(q, ko, vo, n, nk, 0, 0, self.heads, self.kv, self.hd, self.scale, self.t)
        assert worst(out, ref, tol) <= 1.0
        o = offsets(n)
        for b in range(len(n)):
            self.k[b] = torch.cat([self.k[b], k[o[b]:o[b + 1]]])
            self.v[b] = torch.cat([self.v[b], v[o[b]:o[b + 1]]])

    def step(self, q, k, v, out):
        """One token a sequence: everything a graph can hold."""
        self.rotate(q, k, self.lens)
        c = self.cache.struct()
        self.ctx.kv4_append(c, rows_args(k, v, self.lens, self.t, None, self.at, self.next))
        self.ctx.attention_kv4(c, kv4_args(q, out, self.next, self.heads, self.t, self.scale, self.at, self.cache.capacity))
        self.lens.copy_(self.next)

    def check_step(self, q, k, v, out):
        lens = self.lens.tolist()
        ref, tol = kv4_64(self.cache, q, lens, self.slots, self.heads, self.scale, self.t)
        assert worst(out, ref, tol) <= 1.0
        G, hd = self.heads // self.kv, self.hd
        for b, n in enumerate(lens):
            self.k[b] = torch.cat([self.k[b], k[b:b + 1]])
            self.v[b] = torch.cat([self.v[b], v[b:b + 1]])
            for h in range(self.heads):
                j = h // G
                x, y = (z[b][:, j * hd:(j + 1) * hd].double() for z in (self.k, self.v))
                kc, vc = (lambda c, s, m: c * s + m)(*self.cache.parts(0, self.slots[b], j, n)), \
                    (lambda c, s, m: c * s + m)(*self.cache.parts(1, self.slots[b], j, n))
                qq = q[b, h * hd:(h + 1) * hd].double()
                w = torch.softmax(self.scale * (x @ qq), 0)
                ds = float(self.scale * ((x - kc).abs() @ qq.abs()).max())
                bound = (np.exp(2 * ds) - 1) * (w @ vc.abs()) + w @ (y - vc).abs()
                o = slice(h * hd, (h + 1) * hd)
                assert ((out[b, o].double() - w @ y).abs() <= bound + tol[b, o] + 1e-12).all()


@pytest.mark.parametrize("t,hd", [("f32", 128), ("bf16", 128), ("f16", 64), ("bf16", 256)])
def test_prompts_in_chunks_then_decode(ctx, t, hd):
    c = Conversations(ctx, t, hd=hd)
    c.chunk([70, 1, 129])
    c.chunk([0, 64, 33])
    for _ in range(3):
        q, k, v = c.rows(3)
        out = torch.empty(3, c.heads * hd, dtype=DT[t], device="cuda")
        c.step(q, k, v, out)
        ctx.synchronize()
        c.check_step(q, k, v, out)


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_one_captured_step_decodes(ctx, t):
    """One graph for every step (lengths and positions live on the device), checked against eager steps."""
    own = smoe_amd.Context()
    stream = torch.cuda.Stream()
    own.set_stream(stream.cuda_stream)
    with torch.cuda.stream(stream):
        pair = [Conversations(own, t, seed=5) for _ in range(2)]
        for c in pair:
            c.chunk([40, 7, 100])
            q, k, v = c.rows(3)
            out = torch.empty(3, c.heads * c.hd, dtype=DT[t], device="cuda")
            c.bufs = (q, k, v, out)
            c.step(*c.bufs)                      # (the first step, and the scratch)
        own.synchronize()
        stream.synchronize()
        a, b = pair
        assert torch.equal(a.bufs[3], b.bufs[3])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            a.step(*a.bufs)
        for i in range(4):
            for x, y in zip(a.bufs[:3], b.bufs[:3]):
                r = randn(gen(100 + i), *x.shape).to(x.dtype)
                x.copy_(r)
                y.copy_(r)
            graph.replay()
            b.step(*b.bufs)
            own.synchronize()
            stream.synchronize()
            assert torch.equal(a.bufs[3], b.bufs[3]) and a.lens.tolist() == b.lens.tolist()
            assert all(torch.equal(x, y) for x, y in zip(a.cache.codes + a.cache.params, b.cache.codes + b.cache.params))
    stream.synchronize()
    del graph
    own.close()


def test_contexts_at_once_on_streams_of_their_own(ctx):
    """Calls with scratch (parts, f16 halves), two contexts, nothing but the streams' own order."""
    jobs = []
    for i, (t, nq, nk, lens) in enumerate((("f32", [300], [300], [5000, 3, 700]), ("bf16", [20], [3000], [4, 4000, 900]))):
        own, stream = smoe_amd.Context(), torch.cuda.Stream()
        own.set_stream(stream.cuda_stream)
        g = gen(20 + i)
        q, k, v = (randn(g, n, m * 128).to(DT[t]) for n, m in ((nq[0], 8), (nk[0], 2), (nk[0], 2)))
        cache = Cache(g, 3, 2, 5000, 128)
        q1 = randn(g, 3, 8 * 128).to(DT[t])
        o, o1 = torch.empty(nq[0], 8 * 128, dtype=DT[t], device="cuda"), torch.empty_like(q1)
        keep = (i32([0, nq[0]]), i32([0, nk[0]]), i32(lens))
        call = (prompt_args(q, k, v, o, keep[0], keep[1], 8, 2, 128, t, 0.09, nk[0]),
                cache.struct(), kv4_args(q1, o1, keep[2], 8, t, 0.09, None, 5000))
        jobs.append((own, call, o, o1, (q, k, v, cache, q1, keep, stream), (t, nq, nk, lens)))
    torch.cuda.synchronize()
    for own, call, *_ in jobs:
        own.attention_prompt(call[0])
        own.attention_kv4(call[1], call[2])
        own.synchronize()
    want = [(j[2].clone(), j[3].clone()) for j in jobs]
    for j in jobs:
        j[2].fill_(3)
        j[3].fill_(3)
    torch.cuda.synchronize()
    for _ in range(20):
        for own, call, *_ in jobs:
            own.attention_prompt(call[0])
            own.attention_kv4(call[1], call[2])
    for j, (o, o1) in zip(jobs, want):
        j[0].synchronize()
        assert torch.equal(j[2], o) and torch.equal(j[3], o1)
        q, k, v, cache, q1 = j[4][:5]
        t, nq, nk, lens = j[5]
        ref, tol = prompt64(q, k, v, nq, nk, 0, 0, 8, 2, 128, 0.09, t)
        assert worst(o, ref, tol) <= 1.0
        ref, tol = kv4_64(cache, q1, lens, range(3), 8, 0.09, t)
        assert worst(o1, ref, tol) <= 1.0
        j[0].close()


def test_graphs_of_one_context_and_scratch_that_grows_after_capture(ctx):
    own, stream = smoe_amd.Context(), torch.cuda.Stream()
    own.set_stream(stream.cuda_stream)
    g = gen(30)

    def call(t, nq, nk):
        q, k, v = (randn(g, n, m * 128).to(DT[t]) for n, m in ((nq, 8), (nk, 2), (nk, 2)))
        out = torch.empty(nq, 8 * 128, dtype=DT[t], device="cuda")
        keep = q, k, v, i32([0, nq]), i32([0, nk])
        return prompt_args(q, k, v, out, keep[3], keep[4], 8, 2, 128, t, 0.09, nk), out, keep

    calls = [call("bf16", 20, 3000), call("f32", 90, 500)]
    torch.cuda.synchronize()
    graphs, want = [], []
    for a, out, _ in calls:
        own.attention_prompt(a)
        own.synchronize()
        want.append(out.clone())
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            own.attention_prompt(a)
    torch.cuda.synchronize()
    big = call("f32", 700, 9000)
    torch.cuda.synchronize()
    for i in range(3):
        for _, out, _ in calls:
            out.fill_(4)
        torch.cuda.synchronize()
        if i:
            own.attention_prompt(big[0])         # its scratch is larger than what the graphs hold
        with torch.cuda.stream(stream):
            for x in graphs:
                x.replay()
        own.synchronize()
        for (_, out, _), w in zip(calls, want):
            assert torch.equal(out, w)
    ref, tol = prompt64(*big[2][:3], [700], [9000], 0, 0, 8, 2, 128, 0.09, "f32")
    assert worst(big[1], ref, tol) <= 1.0
    del graphs
    own.close()
