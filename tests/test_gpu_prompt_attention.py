"""smoe_hip_attention_prompt against its definition in 64 bits (attention_ref.py has
the bounds): packed sequences, lengths from 0 on, chunks behind a prefix, queries
that see nothing, every head layout and type, strided rows, split keys, graphs."""
import pytest
import torch

import smoe_amd
from attention_ref import DT, fused, gen, i32, offsets, prompt64, prompt_args, randn, worst

pytestmark = pytest.mark.gpu


def make(nq, nk, heads, kv, hd, t, seed, strided=False, q0=0, k0=0, behind=3):
    """Rows of the sequences with some before and behind them."""
    g = gen(seed)
    q = randn(g, q0 + sum(nq) + behind, heads * hd, std=1.5).to(DT[t])
    k = randn(g, k0 + sum(nk) + behind, kv * hd).to(DT[t])
    v = randn(g, k0 + sum(nk) + behind, kv * hd).to(DT[t])
    if strided:
        k, v = fused([k, v])
        q = fused([q, torch.zeros(q.shape[0], 64, dtype=q.dtype, device="cuda")])[0]
    out = torch.full((q.shape[0], heads * hd), 9.0, dtype=DT[t], device="cuda")
    return q, k, v, out, i32(offsets(nq, q0)), i32(offsets(nk, k0))


def check(ctx, nq, nk, heads, kv, hd, t, strided=False, q0=0, k0=0, max_k=0, seed=1):
    q, k, v, out, qo, ko = make(nq, nk, heads, kv, hd, t, seed, strided, q0, k0)
    scale = hd ** -0.5
    ctx.attention_prompt(prompt_args(q, k, v, out, qo, ko, heads, kv, hd, t, scale, max_k or max(nk)))
    ctx.synchronize()
    ref, tol = prompt64(q, k, v, nq, nk, q0, k0, heads, kv, hd, scale, t)
    n = q0 + sum(nq)
    assert (out[:q0] == 9).all() and (out[n:] == 9).all()      # rows outside the sequences
    e = worst(out[q0:n], ref[q0:n], tol[q0:n])
    print(f"prompt {nq} x {nk}, {heads}/{kv} x {hd} {t}: error / bound {e:.3f}")
    assert e <= 1.0
    return out


LAYOUTS = [(32, 4, 128), (64, 4, 128), (8, 8, 64), (8, 2, 256), (10, 2, 128), (1, 1, 64), (6, 3, 128), (16, 16, 64),
           (48, 1, 128), (5, 5, 256)]


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,kv,hd", LAYOUTS)
def test_layouts(ctx, heads, kv, hd, t):
    n = [1, 65, 0, 200, 31]
    check(ctx, n, n, heads, kv, hd, t, strided=heads % 2 == 0)


@pytest.mark.parametrize("t", ["bf16", "f32"])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 511, 1000])
def test_lengths(ctx, n, t):
    check(ctx, [n], [n], 8, 1, 128, t, seed=n)


@pytest.mark.parametrize("nq,nk,q0,k0", [
    ([5], [70], 0, 0), ([64], [1064], 0, 0), ([1], [777], 2, 5), ([3, 1, 0, 40], [300, 1, 90, 41], 1, 7),
    ([0, 0], [0, 0], 2, 2), ([1, 1, 1, 1], [1, 64, 65, 2], 0, 0),
])
@pytest.mark.parametrize("t,hd", [("bf16", 128), ("f16", 64), ("f32", 128), ("bf16", 256), ("f32", 256)])
def test_chunks_behind_a_prefix(ctx, nq, nk, q0, k0, t, hd):
    check(ctx, nq, nk, 16, 2, hd, t, q0=q0, k0=k0, strided=True)


@pytest.mark.parametrize("t", ["bf16", "f32"])
def test_queries_that_see_nothing(ctx, t):
    nq, nk = [70, 3, 9], [6, 0, 9]
    out = check(ctx, nq, nk, 8, 2, 128, t)
    assert (out[:64] == 0).all() and (out[70:73] == 0).all()


@pytest.mark.parametrize("t,hd", [("bf16", 128), ("f16", 128), ("f32", 64), ("bf16", 64), ("bf16", 256)])
def test_long_keys_split(ctx, t, hd):
    """Few rows over many keys: parts of the keys, joined; the same rows whatever the hint."""
    a = check(ctx, [33], [5000], 8, 2, hd, t, seed=3)
    b = check(ctx, [33], [5000], 8, 2, hd, t, seed=3, max_k=64)          # one part
    tol = 2 ** -6 if t == "bf16" else 2 ** -9
    assert (a.double() - b.double()).abs().max() <= tol
    check(ctx, [3, 30, 1, 0], [4000, 30, 2900, 700], 8, 2, hd, t, seed=4)


def test_long_prompt(ctx):
    check(ctx, [2300], [2300], 8, 2, 128, "bf16", seed=8)
    check(ctx, [1500], [1500], 16, 2, 128, "f32", seed=9)


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
def test_large_scores(ctx, t):
    """One key takes all the weight, late in the row, and the first ones take it from nothing."""
    g = gen(11)
    q = randn(g, 300, 256).to(DT[t])
    k = randn(g, 300, 128).to(DT[t])
    k[200] *= 40
    v = randn(g, 300, 128).to(DT[t])
    out = torch.empty_like(q)
    qo = i32([0, 300])
    ctx.attention_prompt(prompt_args(q, k, v, out, qo, None, 2, 1, 128, t, 0.5))
    ctx.synchronize()
    ref, tol = prompt64(q, k, v, [300], [300], 0, 0, 2, 1, 128, 0.5, t)
    assert worst(out, ref, tol) <= 1.0


@pytest.mark.parametrize("t", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("n,over", [(8000, 10.4), (8000, 14.0), (300, 12.0)])
def test_many_small_weights_beside_a_large_one(ctx, t, n, over):
    """Weights e^-over each beside one of 1: in f16 far below its normal numbers, together a good part of the sum."""
    g = gen(n)
    q, k, v = (torch.zeros(m, 128, device="cuda") for m in (40, n, n))
    q[:, 0], k[5, 0] = 4.0, over / 4.0
    q[:, 1:], k[:, 1:] = randn(g, 40, 127, std=0.3), randn(g, n, 127, std=0.02)
    v.copy_(1.0 + randn(g, n, 128, std=0.2))
    v[5] = -1.0
    q, k, v = (x.to(DT[t]) for x in (q, k, v))
    out = torch.empty_like(q)
    ctx.attention_prompt(prompt_args(q, k, v, out, i32([0, 40]), i32([0, n]), 1, 1, 128, t, 1.0, n))
    ctx.synchronize()
    ref, tol = prompt64(q, k, v, [40], [n], 0, 0, 1, 1, 128, 1.0, t)
    e = worst(out, ref, tol)
    print(f"prompt {n} keys, one {over} above, {t}: error / bound {e:.3f}")
    assert e <= 1.0


def test_not_a_number_stays_in_its_sequence(ctx):
    nq = [70, 40, 30]
    q, k, v, out, qo, ko = make(nq, nq, 4, 2, 128, "bf16", 2)
    k[70:110] = float("nan")
    v[75] = float("inf")
    k[140:] = float("nan")      # rows behind the last sequence
    v[140:] = float("nan")
    ctx.attention_prompt(prompt_args(q, k, v, out, qo, ko, 4, 2, 128, "bf16", 0.1))
    ctx.synchronize()
    assert torch.isfinite(out[:70].float()).all() and torch.isfinite(out[110:140].float()).all()
    assert torch.isnan(out[70:110].float()).all()


def test_infinite_keys_that_are_hidden(ctx):
    """A key that a query does not see does not reach it, whatever it holds."""
    q, k, v, out, qo, ko = make([50], [50], 2, 1, 64, "f16", 3)
    ctx.attention_prompt(prompt_args(q, k, v, out, qo, ko, 2, 1, 64, "f16", 0.1))
    ctx.synchronize()
    want = out.clone()
    k[30] = float("inf")
    k[31] = float("nan")
    ctx.attention_prompt(prompt_args(q, k, v, out, qo, ko, 2, 1, 64, "f16", 0.1))
    ctx.synchronize()
    assert torch.equal(out[:30], want[:30])


@pytest.mark.parametrize("bad_q", [True, False])
def test_bad_offsets_are_reported(ctx, bad_q):
    q, k, v, out, qo, ko = make([20, 20], [20, 20], 2, 1, 64, "bf16", 4, behind=0)
    o = qo if bad_q else ko
    o[2] = 41
    ctx.attention_prompt(prompt_args(q, k, v, out, qo, ko, 2, 1, 64, "bf16", 0.1))
    with pytest.raises(smoe_amd.SmoeError) as e:
        ctx.synchronize()
    assert e.value.code == smoe_amd.SMOE_ERR_ARG
    ctx.synchronize()
    ref, tol = prompt64(q, k, v, [20], [20], 0, 0, 2, 1, 64, 0.1, "bf16")
    assert worst(out[:20], ref[:20], tol[:20]) <= 1.0           # the sequence that is right
    assert (out[20:] == 9).all()


def test_many_sequences(ctx):
    """More sequences than one wave's lanes, empty ones among them."""
    n = [(7 * i) % 13 for i in range(200)]
    check(ctx, n, [x + (i % 3) for i, x in enumerate(n)], 8, 4, 64, "bf16")


@pytest.mark.parametrize("nq,nk", [([130], [130]), ([20], [3000])])
def test_graph_replays(ctx, nq, nk):
    q, k, v, out, qo, ko = make(nq, nk, 8, 2, 128, "bf16", 5)
    a = prompt_args(q, k, v, out, qo, ko, 8, 2, 128, "bf16", 0.1, max(nk))
    ctx.attention_prompt(a)
    ctx.synchronize()
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph, stream=stream):
            ctx.set_stream(torch.cuda.current_stream().cuda_stream)
            ctx.attention_prompt(a)
    finally:
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    for i in range(4):
        q.copy_(randn(gen(50 + i), *q.shape).to(q.dtype))
        ctx.attention_prompt(a)
        torch.cuda.synchronize()
        want = out.clone()
        out.fill_(1.0)
        graph.replay()
        torch.cuda.synchronize()
        n = sum(nq)
        assert torch.equal(out[:n], want[:n])


def test_same_bits_again(ctx):
    for nq, nk in (([200, 31], [200, 31]), ([9], [4000])):
        q, k, v, out, qo, ko = make(nq, nk, 8, 2, 128, "bf16", 6)
        a = prompt_args(q, k, v, out, qo, ko, 8, 2, 128, "bf16", 0.1, max(nk))
        got = []
        for _ in range(3):
            ctx.attention_prompt(a)
            torch.cuda.synchronize()
            got.append(out.clone())
        assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
