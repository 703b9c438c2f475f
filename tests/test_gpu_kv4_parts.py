"""smoe_hip_attention_kv4 over sequences of very different lengths, whose positions are
shared out over the blocks by length: batches of one and of several passes of 64
sequences, empty and single positions, indexes out of range anywhere in the batch, the
most parts of a sequence, and hints that are wrong."""
import pytest
import torch

import smoe_amd
from attention_ref import DT, Cache, gen, i32, kv4_64, kv4_args, randn, worst

pytestmark = pytest.mark.gpu


def run(ctx, cache, q, lens, slots, heads, t, max_len):
    out = torch.full_like(q, 9.0)
    ctx.attention_kv4(cache.struct(), kv4_args(q, out, i32(lens), heads, t, 0.09, i32(slots), max_len))
    return out


def lengths(n, most, seed):
    g = torch.Generator().manual_seed(seed)
    lens = [int(most * float(x) ** 3) for x in torch.rand(n, generator=g)]
    lens[n // 2], lens[n // 3], lens[-1] = 0, 1, most
    return lens


@pytest.mark.parametrize("n,most,heads,kv,hd,t", [
    (3, 4000, 8, 1, 128, "bf16"), (33, 2000, 8, 1, 128, "f32"), (64, 1500, 4, 2, 64, "f16"), (65, 1500, 4, 1, 64, "bf16"),
    (130, 900, 2, 1, 128, "f32"), (300, 700, 1, 1, 64, "bf16"), (20, 3000, 20, 1, 128, "bf16"), (12, 2500, 4, 2, 256, "f32"),
])
@pytest.mark.parametrize("hint", [0, 1])
def test_ragged(ctx, n, most, heads, kv, hd, t, hint):
    """hint 0: the longest length, 1: the capacity."""
    g = gen(n)
    slots = [(7 * i) % n for i in range(n)] if n % 7 else list(range(n))
    cache = Cache(g, n, kv, most + 40, hd)
    lens = lengths(n, most, n)
    q = randn(g, n, heads * hd).to(DT[t])
    out = run(ctx, cache, q, lens, slots, heads, t, 0 if hint else most)
    ctx.synchronize()
    ref, tol = kv4_64(cache, q, lens, slots, heads, 0.09, t)
    e = worst(out, ref, tol)
    print(f"kv4 {n} of up to {most}, {heads}/{kv} x {hd} {t}: error / bound {e:.3f}")
    assert e <= 1.0
    assert all((out[i] == 0).all() for i in range(n) if lens[i] == 0)


@pytest.mark.parametrize("n,most,heads,kv,hd,t", [
    (8, 4200, 8, 4, 128, "bf16"), (4, 9000, 64, 4, 128, "f32"), (4, 4200, 4, 4, 256, "bf16"), (16, 4100, 2, 2, 128, "f16"),
    (8, 8300, 8, 2, 64, "f32"), (2, 9000, 34, 2, 256, "f32"),
])
def test_blocks_of_eight_waves(ctx, n, most, heads, kv, hd, t):
    """Enough positions for every resident block to take eight tiles and more."""
    g = gen(n + hd)
    cache = Cache(g, n, kv, most, hd)
    for lens in (lengths(n, most, 1), [most] * n, [most] + [3] * (n - 1)):
        q = randn(g, n, heads * hd).to(DT[t])
        out = run(ctx, cache, q, lens, range(n), heads, t, most)
        ctx.synchronize()
        ref, tol = kv4_64(cache, q, lens, range(n), heads, 0.09, t)
        e = worst(out, ref, tol)
        print(f"kv4 {n} of up to {most}, {heads}/{kv} x {hd} {t}: error / bound {e:.3f}")
        assert e <= 1.0


@pytest.mark.parametrize("bad", [0, 40, 63, 64, 99])
@pytest.mark.parametrize("what", ["long", "negative", "slot", "negative slot"])
def test_out_of_range_anywhere(ctx, bad, what):
    n, most = 100, 1200
    g = gen(5)
    cache = Cache(g, n, 1, most, 64)
    lens, slots = lengths(n, most, 3), list(range(n))
    good = [i for i in range(n) if i != bad]
    q = randn(g, n, 64)
    fair = list(lens)
    fair[bad] = 0
    ref, tol = kv4_64(cache, q, fair, slots, 1, 0.09, "f32")
    if what == "long":
        lens[bad] = most + 1
    elif what == "negative":
        lens[bad] = -3
    else:
        slots[bad] = n if what == "slot" else -1
        lens[bad] = 70
    out = run(ctx, cache, q, lens, slots, 1, "f32", most)
    with pytest.raises(smoe_amd.SmoeError):
        ctx.synchronize()
    assert worst(out[good], ref[good], tol[good]) <= 1.0
    assert (out[bad] == 0).all()


@pytest.mark.parametrize("lens", [[150000], [150000, 3], [0, 90000, 0, 17, 130000], [40000] * 3])
def test_most_parts_of_a_sequence(ctx, lens):
    g = gen(6)
    cache = Cache(g, len(lens), 1, 150016, 64)
    q = randn(g, len(lens), 8 * 64)
    slots = list(range(len(lens)))
    for max_len in (max(lens), 0):
        out = run(ctx, cache, q, lens, slots, 8, "f32", max_len)
        ctx.synchronize()
        ref, tol = kv4_64(cache, q, lens, slots, 8, 0.09, "f32")
        assert worst(out, ref, tol) <= 1.0


@pytest.mark.parametrize("max_len", [1, 200, 700, 5000])
def test_the_hint_may_be_wrong(ctx, max_len):
    g = gen(7)
    lens = [900, 0, 4000, 64, 333]
    cache = Cache(g, 5, 2, 4000, 128)
    q = randn(g, 5, 8 * 128).to(torch.bfloat16)
    out = run(ctx, cache, q, lens, [4, 2, 0, 1, 3], 8, "bf16", max_len)
    ctx.synchronize()
    ref, tol = kv4_64(cache, q, lens, [4, 2, 0, 1, 3], 8, 0.09, "bf16")
    assert worst(out, ref, tol) <= 1.0


def test_in_place(ctx):
    """out may be q: a row's blocks have read it before anyone writes it."""
    g = gen(10)
    lens = [2500, 1, 40, 0, 900]
    cache = Cache(g, 5, 2, 2500, 128)
    q = randn(g, 5, 40 * 128)
    want = run(ctx, cache, q, lens, range(5), 40, "f32", 2500)
    for max_len in (2500, 100):                  # in parts, and each sequence whole
        x = q.clone()
        ctx.attention_kv4(cache.struct(), kv4_args(x, x, i32(lens), 40, "f32", 0.09, None, max_len))
        ctx.synchronize()
        if max_len == 2500:
            assert torch.equal(x, want)
        else:
            ref, tol = kv4_64(cache, q, lens, range(5), 40, 0.09, "f32")
            assert worst(x, ref, tol) <= 1.0


def test_all_empty(ctx):
    g = gen(8)
    cache = Cache(g, 4, 2, 3000, 128)
    q = randn(g, 4, 8 * 128)
    out = run(ctx, cache, q, [0] * 4, range(4), 8, "f32", 3000)
    ctx.synchronize()
    assert (out == 0).all()


def test_same_bits_alone_and_again(ctx):
    """The same call twice, with other lengths in the same scratch between them."""
    g = gen(9)
    cache = Cache(g, 6, 2, 6000, 128)
    q = randn(g, 6, 8 * 128)
    lens = [6000, 17, 0, 2500, 1, 5999]
    one = run(ctx, cache, q, lens, range(6), 8, "f32", 6000)
    run(ctx, cache, q, lens[::-1], range(6), 8, "f32", 6000)
    two = run(ctx, cache, q, lens, range(6), 8, "f32", 6000)
    ctx.synchronize()
    assert torch.equal(one, two)
