"""smoe_hip_attention_prompt of f32 rows: its products take every value as two f16 at a
power of two, for a query row and for 32 keys of a KV head, so values far from 1, tiles
of very different size, zeros and values that are not finite.

Bounds, on top of attention_ref.py's: a value x is taken to 2^-22 |x| + 2^-38 M, M the
largest of its row (q) or of its tile (k, v); a weight w <= 1 to 2^-22 w plus at most
2^-39 V / |v| of it, V the largest value of the sequence (the powers differ by V's
magnitude over the tile's), so 2^-39 V a key."""
import pytest
import torch

import smoe_amd
from attention_ref import U, gen, i32, offsets, prompt_args, randn

pytestmark = pytest.mark.gpu


def tile_max(x):
    """Of each row the largest magnitude of the 32 rows it shares a tile with."""
    n = x.shape[0]
    pad = torch.zeros((n + 31) // 32 * 32, x.shape[1], dtype=torch.float64, device="cuda")
    pad[:n] = x.double().abs()
    return pad.reshape(-1, 32 * x.shape[1]).amax(1).repeat_interleave(32)[:n, None]


def check(ctx, q, k, v, heads, kv, scale, rows=None):
    """One sequence: every row of q (or `rows` of them) against the definition."""
    n, N = q.shape[0], k.shape[0]
    hd, G = q.shape[1] // heads, heads // kv
    out = torch.full_like(q, 9.0)
    ctx.attention_prompt(prompt_args(q, k, v, out, i32([0, n]), i32([0, N]), heads, kv, hd, "f32", scale, N))
    ctx.synchronize()
    hidden = torch.arange(N, device="cuda") > torch.arange(n, device="cuda")[:, None] + N - n
    worst = 0.0
    for h in range(heads):
        j = h // G
        qq, kk, vv = q[:, h * hd:(h + 1) * hd].double(), k[:, j * hd:(j + 1) * hd], v[:, j * hd:(j + 1) * hd]
        km, vm = tile_max(kk), tile_max(vv)
        kk, vv = kk.double(), vv.double()
        s = scale * (qq @ kk.T.contiguous())
        ek = 2.0 ** -22 * kk.abs() + 2.0 ** -38 * km
        eq = 2.0 ** -22 * qq.abs() + 2.0 ** -38 * qq.abs().amax(1, keepdim=True)
        mag = scale * (qq.abs() @ kk.abs().T.contiguous())
        ds = mag * (4 * hd ** 0.5 * U + 4 * U) + scale * (qq.abs() @ ek.T.contiguous() + eq @ (kk.abs() + ek).T.contiguous())
        s, ds = s.masked_fill(hidden, -float("inf")), ds.masked_fill(hidden, 0.0)
        w = torch.softmax(s, -1)
        ref = w @ vv
        tol = (w @ vv.abs()) * (2 * ds.amax(-1, keepdim=True) + 2.0 ** -21 + 4 * (N + 64) ** 0.5 * U + 2.0 ** -20)
        tol = tol + w @ (2.0 ** -38 * vm).expand_as(vv) + N * 2.0 ** -39 * vv.abs().max() + U * ref.abs()
        got = out[:, h * hd:(h + 1) * hd].double()
        pick = slice(None) if rows is None else rows
        r = (got[pick] - ref[pick]).abs() / (tol[pick] + 1e-300)
        assert not torch.isnan(r).any()
        worst = max(worst, float(r.max()))
    print(f"f32 prompt {n} x {N}, {heads}/{kv} x {hd}: error / bound {worst:.3f}")
    assert worst <= 1.0
    return out


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("a,b", [(0, 0), (40, 60), (-40, -60), (90, 100), (-90, -90)])
def test_magnitudes(ctx, hd, a, b):
    g = gen(3)
    q, k, v = randn(g, 70, 4 * hd) * 2.0 ** a, randn(g, 200, 2 * hd) * 2.0 ** -a, randn(g, 200, 2 * hd) * 2.0 ** b
    check(ctx, q, k, v, 4, 2, hd ** -0.5)


@pytest.mark.parametrize("step", [24, -24, 7])
@pytest.mark.parametrize("n", [40, 300])
def test_tiles_of_different_size(ctx, step, n):
    """V grows or shrinks from tile to tile, so what was added is rescaled; a KV head of zeros beside it."""
    g = gen(4)
    q, k, v = randn(g, n, 4 * 128), randn(g, 300, 2 * 128), randn(g, 300, 2 * 128)
    tile = torch.arange(300, device="cuda") // 32
    v = v * torch.exp2(((tile * step + 17) % 97 - 48).float())[:, None]
    v[:, :128] = 0
    out = check(ctx, q, k, v, 4, 2, 128 ** -0.5)
    assert (out[:, :256] == 0).all()


def test_keys_of_different_size(ctx):
    g = gen(5)
    q, k, v = randn(g, 200, 4 * 128), randn(g, 200, 2 * 128), randn(g, 200, 2 * 128)
    k = k * torch.exp2(torch.randint(-30, 5, (200, 1), generator=g, device="cuda").float())
    k[64:96] = 0
    q[::3] *= 2.0 ** -80
    q[5] = 0
    check(ctx, q, k, v, 4, 2, 128 ** -0.5)


def test_first_tiles_of_zeros(ctx):
    g = gen(6)
    q, k, v = randn(g, 180, 4 * 64), randn(g, 180, 2 * 64), randn(g, 180, 2 * 64)
    v[:70] = 0
    v[100:140] = 0
    out = check(ctx, q, k, v, 4, 2, 0.125)
    assert (out[:70] == 0).all()


def test_not_a_number_stays_in_its_row_and_its_queries(ctx):
    g = gen(7)
    q, k, v = randn(g, 160, 4 * 128), randn(g, 160, 2 * 128), randn(g, 160, 2 * 128)
    q[33, 5] = float("nan")
    q[40, 130] = float("inf")
    keep = torch.tensor([i for i in range(160) if i not in (33, 40)], device="cuda")
    out = check(ctx, torch.where(torch.isfinite(q), q, 0.0), k, v, 4, 2, 0.09, keep)
    bad = torch.full_like(q, 9.0)
    ctx.attention_prompt(prompt_args(q, k, v, bad, i32([0, 160]), i32([0, 160]), 4, 2, 128, "f32", 0.09, 160))
    ctx.synchronize()
    assert torch.equal(bad[keep], out[keep])
    assert torch.isnan(bad[33, :128]).all() and torch.isfinite(bad[33, 128:]).all()


def test_sequences_that_share_rows_around_a_bad_one(ctx):
    """The bad sequence makes its neighbours overlap: more key tiles than rows allow, never written or followed."""
    g = gen(8)
    q, k, v = randn(g, 96, 4 * 128), randn(g, 96, 2 * 128), randn(g, 96, 2 * 128)
    out = torch.full((96, 512), 9.0, device="cuda")
    off = i32([0, 96, 0, 96, 0, 96, 0, 96])
    ctx.attention_prompt(prompt_args(q, k, v, out, off, off, 4, 2, 128, "f32", 0.09, 96))
    with pytest.raises(smoe_amd.SmoeError):
        ctx.synchronize()
    check(ctx, q, k, v, 4, 2, 0.09)


def test_same_bits_again_and_whatever_ran_between(ctx):
    """The f16 halves lie in scratch that calls of other sizes use too."""
    g = gen(9)
    q, k, v = randn(g, 500, 8 * 128), randn(g, 500, 128), randn(g, 500, 128)
    one = check(ctx, q, k, v, 8, 1, 0.09, slice(0, 4))
    check(ctx, q[:3].contiguous(), k, v, 8, 1, 0.09)
    two = check(ctx, q, k, v, 8, 1, 0.09, slice(0, 4))
    assert torch.equal(one, two)


def test_capture_needs_scratch_of_an_earlier_call(ctx):
    own = smoe_amd.Context()
    stream = torch.cuda.Stream()
    own.set_stream(stream.cuda_stream)
    g = gen(10)
    n = 300
    q, k, v = randn(g, n, 4 * 128), randn(g, n, 2 * 128), randn(g, n, 2 * 128)
    out, off = torch.zeros(n, 512, device="cuda"), i32(offsets([n]))
    args = prompt_args(q, k, v, out, off, None, 4, 2, 128, "f32", 0.09, n)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        with pytest.raises(smoe_amd.SmoeError):
            own.attention_prompt(args)
        torch.zeros(1, device="cuda")
    own.attention_prompt(args)
    own.synchronize()
    eager = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        own.attention_prompt(args)
    for _ in range(3):
        out.fill_(9)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        out.fill_(7)
        torch.cuda.synchronize()
        own.attention_prompt(args)
        own.synchronize()
        assert torch.equal(out, eager)
    del graph
    own.close()
