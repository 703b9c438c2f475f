"""The 4-bit KV cache on the GPU: rows into it bit for bit as the CPU oracle's scale+min
quantizer, rows out of it exactly, and attention over it against 64 bits."""
import numpy as np
import pytest
import torch

import smoe_amd
from attention_ref import DT, Cache, fused, gen, i32, kv4_64, kv4_args, np_u16, offsets, randn, worst

pytestmark = pytest.mark.gpu


def rows_args(k, v, start, t, offs=None, slots=None, lens_out=None):
    p = lambda x: x.data_ptr() if x is not None else None
    return smoe_amd.SmoeKv4RowsArgs(
        k=k.data_ptr(), v=v.data_ptr(), offsets=p(offs), slots=p(slots), start=start.data_ptr(),
        lens_out=p(lens_out), k_stride=k.stride(0), v_stride=v.stride(0), n_seqs=start.numel(),
        n_rows=k.shape[0], type=smoe_amd.TYPES[t])


def quantized(oracle, x):
    """x [.., hd] on the CPU as (packed codes [.., hd / 2], scale and min bits [.., hd / 64, 2])."""
    w = x.float().cpu().numpy().reshape(-1)
    packed, s, m = oracle.quantize_q4_min(w)
    shape = tuple(x.shape[:-1])
    return (np.asarray(packed).reshape(*shape, x.shape[-1] // 2),
            np.stack([np.asarray(s).reshape(*shape, -1), np.asarray(m).reshape(*shape, -1)], -1))


def from_cache(c, side, slot, pos):
    return c.codes[side][slot, :, pos].cpu().numpy(), np_u16(c.params[side][slot, :, pos].contiguous())


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kv,hd", [(4, 128), (8, 64), (2, 256), (1, 64), (3, 128)])
def test_append_and_read(ctx, oracle, kv, hd, t):
    g = gen(kv * hd)
    n, slots, start = [3, 0, 17, 1, 40], [4, 0, 2, 6, 1], [0, 5, 100, 127, 7]
    rows = sum(n) + 2                                              # two behind the last sequence
    k, v = fused([randn(g, rows, kv * hd, std=2.0).to(DT[t]) for _ in range(2)])
    k[2, :64] = 0.75                                               # a constant group
    v[5] = 0
    c = Cache(g, 7, kv, 128, hd)
    before = [x.clone() for x in c.codes + c.params]
    lens = torch.zeros(5, dtype=torch.int32, device="cuda")
    ctx.kv4_append(c.struct(), rows_args(k, v, i32(start), t, i32(offsets(n)), i32(slots), lens))
    ko, vo = torch.full_like(k, 5.0), torch.full_like(v, 5.0)
    ctx.kv4_read(c.struct(), rows_args(ko, vo, i32(start), t, i32(offsets(n)), i32(slots)))
    ctx.synchronize()
    assert lens.tolist() == [a + b for a, b in zip(start, n)]
    touched = torch.zeros(7, 128, dtype=torch.bool, device="cuda")
    r = 0
    for b, m in enumerate(n):
        for i in range(m):
            for side, (x, o) in enumerate(((k, ko), (v, vo))):
                want = quantized(oracle, x[r].reshape(kv, hd))
                got = from_cache(c, side, slots[b], start[b] + i)
                assert np.array_equal(want[0], got[0]) and np.array_equal(want[1], got[1].reshape(want[1].shape))
                for head in range(kv):
                    codes, s, z = c.parts(side, slots[b], head, 128)
                    val = codes[start[b] + i] * s[start[b] + i] + z[start[b] + i]
                    assert torch.equal(o[r, head * hd:(head + 1) * hd], val.float().to(DT[t]))
            touched[slots[b], start[b] + i] = True
            r += 1
    assert (ko[r:] == 5).all() and (vo[r:] == 5).all()
    for x, y in zip(before, c.codes + c.params):
        keep = ~touched[:, None, :].expand(7, kv, 128)
        assert torch.equal(x[keep], y[keep])


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_one_row_a_sequence(ctx, oracle, t):
    """offsets and slots NULL."""
    g = gen(3)
    k, v = (randn(g, 70, 2 * 128).to(DT[t]) for _ in range(2))
    c = Cache(g, 70, 2, 33, 128)
    start = i32([i % 33 for i in range(70)])
    lens = torch.zeros(70, dtype=torch.int32, device="cuda")
    ctx.kv4_append(c.struct(), rows_args(k, v, start, t, lens_out=lens))
    ctx.synchronize()
    assert torch.equal(lens, start + 1)
    for b in (0, 1, 32, 33, 69):
        want = quantized(oracle, v[b].reshape(2, 128))
        got = from_cache(c, 1, b, b % 33)
        assert np.array_equal(want[0], got[0]) and np.array_equal(want[1], got[1].reshape(want[1].shape))


def test_many_sequences_and_large_batches(ctx):
    g = gen(4)
    n = [(5 * i) % 11 for i in range(300)]
    k, v = (randn(g, sum(n), 4 * 128).to(torch.bfloat16) for _ in range(2))
    c = Cache(g, 300, 4, 40, 128)
    a = rows_args(k, v, i32([i % 20 for i in range(300)]), "bf16", i32(offsets(n)))
    ctx.kv4_append(c.struct(), a)
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    ctx.kv4_read(c.struct(), rows_args(ko, vo, i32([i % 20 for i in range(300)]), "bf16", i32(offsets(n))))
    ctx.synchronize()
    # half a step of the group's scale (range / 15, rounded to 8 bits), the min's and the type's rounding
    for x, o in ((k, ko), (v, vo)):
        w = x.double().reshape(-1, 64)
        step = (w.amax(1) - w.amin(1)) / 15
        tol = step * (0.5 + 16 * 2.0 ** -9) + 2.0 ** -8 * w.abs().amax(1)
        assert ((o.double().reshape(-1, 64) - w).abs() <= tol[:, None] * (1 + 2.0 ** -7)).all()


def test_the_last_of_two_rows_is_kept(ctx, oracle):
    g = gen(6)
    n, slots, start = [4, 3, 5, 2], [1, 0, 1, 1], [2, 0, 4, 5]
    k, v = (randn(g, sum(n), 64) for _ in range(2))
    c = Cache(g, 2, 1, 16, 64)
    ctx.kv4_append(c.struct(), rows_args(k, v, i32(start), "f32", i32(offsets(n)), i32(slots)))
    ctx.synchronize()
    owner = {2: 0, 3: 1, 4: 7, 5: 12, 6: 13, 7: 10, 8: 11}      # position of slot 1 -> row
    for pos, r in owner.items():
        want = quantized(oracle, k[r].reshape(1, 64))
        assert np.array_equal(want[0], from_cache(c, 0, 1, pos)[0])


def test_places_outside_the_cache(ctx):
    g = gen(7)
    k, v = (randn(g, 6, 64) for _ in range(2))
    c = Cache(g, 3, 1, 8, 64)
    before = [x.clone() for x in c.codes + c.params]
    a = rows_args(k, v, i32([8, -1, 0, 2 ** 31 - 1, 0, 0]), "f32", slots=i32([0, 0, 3, 0, -1, -(2 ** 31)]))
    ctx.kv4_append(c.struct(), a)
    with pytest.raises(smoe_amd.SmoeError) as e:
        ctx.synchronize()
    assert e.value.code == smoe_amd.SMOE_ERR_ARG
    assert all(torch.equal(x, y) for x, y in zip(before, c.codes + c.params))
    ctx.kv4_read(c.struct(), a)
    with pytest.raises(smoe_amd.SmoeError):
        ctx.synchronize()
    assert (k == 0).all() and (v == 0).all()
    ctx.synchronize()


def attend(ctx, lens, heads, kv, hd, t, capacity, seed=1, max_len=0, slots=None, strided=False, scale=None):
    g = gen(seed)
    n = len(lens)
    c = Cache(g, n + 2, kv, capacity, hd)
    slots = slots if slots is not None else list(range(n))
    q = randn(g, n, heads * hd, std=1.5).to(DT[t])
    if strided:
        q = fused([q, torch.zeros(n, 64, dtype=q.dtype, device="cuda")])[0]
    out = torch.full((n + 1, heads * hd), 9.0, dtype=DT[t], device="cuda")
    scale = scale or hd ** -0.5
    ctx.attention_kv4(c.struct(), kv4_args(q, out[:n], i32(lens), heads, t, scale, i32(slots), max_len or max(lens)))
    ctx.synchronize()
    ref, tol = kv4_64(c, q, lens, slots, heads, scale, t)
    e = worst(out[:n], ref, tol)
    print(f"kv4 {lens}, {heads}/{kv} x {hd} {t}: error / bound {e:.3f}")
    assert e <= 1.0 and (out[n:] == 9).all()
    return out[:n]


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,kv,hd", [(32, 4, 128), (64, 4, 128), (8, 8, 64), (8, 2, 256), (10, 2, 128), (1, 1, 64),
                                         (34, 2, 64), (20, 1, 256), (17, 1, 128)])
def test_attention_layouts(ctx, heads, kv, hd, t):
    attend(ctx, [1, 70, 0, 300, 31], heads, kv, hd, t, 301, slots=[4, 0, 6, 1, 3], strided=heads % 2 == 0)


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 64, 127, 128, 129, 1000, 4097])
def test_attention_lengths(ctx, n):
    attend(ctx, [n], 8, 1, 128, "f32", n, seed=n)           # the last position is the buffer's


@pytest.mark.parametrize("hint", [1, 64, 9000, 2 ** 31])
def test_attention_any_split(ctx, hint):
    attend(ctx, [9000, 3, 777], 16, 2, 128, "f32", 9001, max_len=hint)


def test_attention_long(ctx):
    attend(ctx, [60000], 16, 1, 128, "f32", 60010)
    attend(ctx, [40000, 5], 8, 2, 256, "bf16", 40000)


def test_attention_over_offsets_past_32_bits(ctx):
    """Cache buffers of more than 2^32 bytes: the last slot's rows."""
    hd, kv, cap = 256, 8, 1 << 20
    c = Cache.__new__(Cache)
    c.kv, c.hd, c.capacity, c.slots = kv, hd, cap, 5
    c.codes = [torch.zeros(5, kv, cap, hd // 2, dtype=torch.uint8, device="cuda") for _ in range(2)]
    c.params = [torch.zeros(5, kv, cap, hd // 64, 2, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    g = gen(12)
    small = Cache(g, 1, kv, 200, hd)
    for x, y in zip(c.codes + c.params, small.codes + small.params):
        x[4, :, :200] = y[0]
    q = randn(g, 1, 16 * hd)
    out = torch.empty_like(q)
    ctx.attention_kv4(c.struct(), kv4_args(q, out, i32([200]), 16, "f32", 0.1, i32([4]), 200))
    k, v = (randn(g, 1, kv * hd) for _ in range(2))
    ctx.kv4_append(c.struct(), rows_args(k, v, i32([cap - 1]), "f32", slots=i32([4])))
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    ctx.kv4_read(c.struct(), rows_args(ko, vo, i32([cap - 1]), "f32", slots=i32([4])))
    ctx.synchronize()
    ref, tol = kv4_64(small, q, [200], [0], 16, 0.1, "f32")
    assert worst(out, ref, tol) <= 1.0
    assert (ko - k).abs().max() < 0.5 and (vo - v).abs().max() < 0.5
    assert int((c.codes[1][:4] != 0).sum()) == 0 and int((c.codes[1][4, :, 200:cap - 1] != 0).sum()) == 0


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_attention_extreme_scales(ctx, t):
    """A first position that takes nearly all the weight and holds small values, groups whose scales differ by
    2^60, and large scores: the weighted scales keep their bits."""
    g = gen(13)
    c = Cache(g, 1, 1, 500, 128)
    c.params[1][0, 0, :, 0] *= 2.0 ** 40
    c.params[1][0, 0, :, 1] *= 2.0 ** -20
    c.params[1][0, 0, 0] *= 2.0 ** -30
    c.params[1][0, 0, 250:] *= 64
    c.params[0][0, 0, 0] *= 6
    q = randn(g, 1, 4 * 128, std=3.0).to(DT[t])
    out = torch.empty_like(q)
    for scale in (0.05, 1.0):
        ctx.attention_kv4(c.struct(), kv4_args(q, out, i32([500]), 4, t, scale))
        ctx.synchronize()
        ref, tol = kv4_64(c, q, [500], [0], 4, scale, t)
        assert worst(out, ref, tol) <= 1.0


def test_attention_query_sizes(ctx):
    """Queries of any size, zeros among them."""
    g = gen(14)
    c = Cache(g, 3, 2, 100, 64)
    q = randn(g, 3, 4 * 64)
    q[0] *= 1e-30
    q[1, :128] = 0
    q[2] *= 1e4
    out = torch.empty_like(q)
    ctx.attention_kv4(c.struct(), kv4_args(q, out, i32([100, 64, 33]), 4, "f32", 0.125))
    ctx.synchronize()
    ref, tol = kv4_64(c, q, [100, 64, 33], [0, 1, 2], 4, 0.125, "f32")
    assert worst(out, ref, tol) <= 1.0


def test_attention_what_lies_behind_does_not_matter(ctx):
    g = gen(15)
    c = Cache(g, 1, 2, 90, 128)
    q = randn(g, 1, 8 * 128)
    out, again = torch.empty_like(q), torch.empty_like(q)
    ctx.attention_kv4(c.struct(), kv4_args(q, out, i32([41]), 8, "f32", 0.1))
    for x in c.params:
        x[:, :, 41:] = float("nan")
    ctx.attention_kv4(c.struct(), kv4_args(q, again, i32([41]), 8, "f32", 0.1))
    ctx.synchronize()
    assert torch.equal(out, again)


def test_attention_bad_slots_and_lengths(ctx):
    g = gen(16)
    c = Cache(g, 3, 1, 50, 64)
    q = randn(g, 5, 64)
    out = torch.full_like(q, 9.0)
    ctx.attention_kv4(c.struct(), kv4_args(q, out, i32([50, 51, -1, 5, 5]), 1, "f32", 0.1, i32([0, 1, 2, 3, -1])))
    with pytest.raises(smoe_amd.SmoeError) as e:
        ctx.synchronize()
    assert e.value.code == smoe_amd.SMOE_ERR_ARG
    ctx.synchronize()
    ref, tol = kv4_64(c, q, [50], [0], 1, 0.1, "f32")
    assert worst(out[:1], ref[:1], tol[:1]) <= 1.0 and (out[1:] == 0).all()


def test_attention_graph_follows_lens(ctx):
    g = gen(17)
    c = Cache(g, 3, 2, 2000, 128)
    q = randn(g, 3, 16 * 128).to(torch.bfloat16)
    out = torch.empty_like(q)
    lens = i32([1, 1, 1])
    a = kv4_args(q, out, lens, 16, "bf16", 0.1, max_len=2000)
    ctx.attention_kv4(c.struct(), a)
    ctx.synchronize()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph, stream=stream):
            ctx.set_stream(torch.cuda.current_stream().cuda_stream)
            ctx.attention_kv4(c.struct(), a)
    finally:
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    for n in ([3, 0, 2000], [1999, 64, 33], [700, 701, 702], [0, 0, 1]):
        lens.copy_(i32(n))
        ctx.attention_kv4(c.struct(), a)
        torch.cuda.synchronize()
        want = out.clone()
        out.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        ref, tol = kv4_64(c, q, n, [0, 1, 2], 16, 0.1, "bf16")
        assert worst(out, ref, tol) <= 1.0
