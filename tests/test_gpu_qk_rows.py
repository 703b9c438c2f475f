"""smoe_hip_qk_norm_rope against its definition in 64 bits.

Bound of an element, before the type's own rounding: the mean square is a sum of
16 products a lane and at most 4 lane steps, 20 u; square root halves it (10), then
division by head_dim, + eps, sqrt, reciprocal, two products (6) and the rotation's
two products and sum (3): 20 u times |x cos| + |y sin| covers them."""
import pytest
import torch

import smoe_amd
from attention_ref import DT, U, fused, gen, half_step, i32, randn

pytestmark = pytest.mark.gpu


def args(q, k, qo, ko, qw, kw, cos, sin, pos, heads, kv, hd, t):
    p = lambda x: x.data_ptr() if x is not None else None
    st = lambda x: x.stride(0) if x is not None else 0
    return smoe_amd.SmoeQkRowsArgs(
        q=p(q), q_out=p(qo), k=p(k), k_out=p(ko), q_norm_w=p(qw), k_norm_w=p(kw), rope_cos=p(cos), rope_sin=p(sin),
        positions=p(pos), q_stride=st(q), q_out_stride=st(qo), k_stride=st(k), k_out_stride=st(ko),
        n_rows=(q if q is not None else k).shape[0], n_positions=cos.shape[0] if cos is not None else 0,
        num_heads=heads, num_kv_heads=kv, head_dim=hd, type=smoe_amd.TYPES[t])


def exact(x, heads, hd, w, cos, sin, pos):
    x = x.double().reshape(x.shape[0], heads, hd)
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.double()
    if cos is None:
        return x.flatten(1), x.abs().flatten(1)
    a, b = x[..., :hd // 2], x[..., hd // 2:]
    c, s = cos[pos.long()].double()[:, None], sin[pos.long()].double()[:, None]
    mag = (a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()
    return torch.cat([a * c - b * s, a * s + b * c], -1).flatten(1), torch.cat(mag, -1).flatten(1)


def tables(hd, n=500):
    inv = 1e6 ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
    a = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * inv
    return a.cos().float(), a.sin().float()


@pytest.mark.parametrize("rows,heads,kv,hd,t,strided", [
    (1, 32, 4, 128, "f32", False), (17, 32, 4, 128, "bf16", True), (300, 64, 4, 128, "f16", False),
    (5, 8, 8, 64, "bf16", False), (77, 8, 2, 256, "f32", True), (33, 10, 2, 128, "f16", True),
    (2000, 7, 1, 64, "bf16", False), (1200, 40, 8, 256, "bf16", True), (3, 1, 1, 64, "f32", False),
])
@pytest.mark.parametrize("norm,rope", [(True, True), (True, False), (False, True)])
def test_rows(ctx, rows, heads, kv, hd, t, strided, norm, rope):
    g = gen(rows * 131 + heads)
    q, k, v = (randn(g, rows, n * hd, std=3.0).to(DT[t]) for n in (heads, kv, kv))
    if strided:
        q, k, v = fused([q, k, v])
    qw, kw = ((1 + 0.3 * randn(g, hd)).to(torch.bfloat16) for _ in range(2)) if norm else (None, None)
    cos, sin = tables(hd) if rope else (None, None)
    pos = torch.randint(0, 500, (rows,), generator=g, device="cuda").to(torch.int32)
    qo = torch.full((rows + 1, heads * hd), 7.0, dtype=DT[t], device="cuda")
    ko = torch.full((rows + 1, kv * hd), 7.0, dtype=DT[t], device="cuda")
    before = [x.clone() for x in (q, k, v)]
    ctx.qk_norm_rope(args(q, k, qo[:rows], ko[:rows], qw, kw, cos, sin, pos, heads, kv, hd, t))
    ctx.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, (q, k, v)))
    assert (qo[rows] == 7).all() and (ko[rows] == 7).all()
    for x, o, w, n in ((q, qo, qw, heads), (k, ko, kw, kv)):
        ref, mag = exact(x, n, hd, w, cos, sin, pos)
        tol = 20 * U * mag + half_step(t) * (ref.abs() + 20 * U * mag) + 1e-30
        if t == "f16":
            tol = tol + 2.0 ** -25          # f16 steps end at 2^-24
        e = float(((o[:rows].double() - ref).abs() / tol).max())
        print(f"rows {rows} x {n} x {hd} {t}: error / bound {e:.2f}")
        assert e <= 1.0


def test_in_place_and_one_side(ctx):
    g = gen(5)
    q, k = (randn(g, 40, n * 128).to(torch.bfloat16) for n in (16, 2))
    w = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    cos, sin = tables(128)
    pos = i32(list(range(40)))
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    ctx.qk_norm_rope(args(q, k, qo, ko, w, w, cos, sin, pos, 16, 2, 128, "bf16"))
    q1, k1 = q.clone(), k.clone()
    ctx.qk_norm_rope(args(q1, None, q1, None, w, w, cos, sin, pos, 16, 0, 128, "bf16"))
    ctx.qk_norm_rope(args(None, k1, None, k1, w, w, cos, sin, pos, 0, 2, 128, "bf16"))
    ctx.synchronize()
    assert torch.equal(q1, qo) and torch.equal(k1, ko)


def test_zero_rows_and_zero_heads_values(ctx):
    """A row of zeros stays one (eps keeps the norm finite)."""
    q = torch.zeros(2, 128, device="cuda")
    k = torch.zeros(2, 128, device="cuda")
    w = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    o = torch.full_like(q, 3.0)
    ctx.qk_norm_rope(args(q, k, o, k, w, w, None, None, None, 1, 1, 128, "f32"))
    ctx.synchronize()
    assert (o == 0).all() and (k == 0).all()


def test_bad_position_is_reported(ctx):
    q = torch.ones(3, 64, device="cuda")
    o = torch.empty_like(q)
    cos, sin = tables(64, 10)
    a = args(q, None, o, None, None, None, cos, sin, i32([0, 10, -1]), 1, 0, 64, "f32")
    ctx.qk_norm_rope(a)
    with pytest.raises(smoe_amd.SmoeError) as e:
        ctx.synchronize()
    assert e.value.code == smoe_amd.SMOE_ERR_ARG
    ctx.synchronize()           # reported once
