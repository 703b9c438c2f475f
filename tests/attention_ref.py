"""Shared pieces of the prompt and 4-bit-cache attention tests: packed buffers,
the operators' definitions in 64 bits, and the error bounds of their arithmetic.

Bounds.  u = 2^-24 is half a step of fp32, h(T) = finfo(T).eps / 2 that of the row
type.  A sum of n fp32 terms in any order is taken to be off by at most
4 sqrt(n) u times the sum of their magnitudes.  A score error d (natural units)
moves a weight by a factor within e^d, so an output by at most 2 d times
A = sum_j w_j |v_j| (numerator and denominator)."""
import numpy as np
import torch

import smoe_amd

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24


def half_step(t):
    return torch.finfo(DT[t]).eps / 2


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, std=1.0):
    return std * torch.randn(*shape, generator=g, device="cuda")


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def offsets(lens, first=0):
    o = [first]
    for n in lens:
        o.append(o[-1] + n)
    return o


def fused(parts):
    """The rows of `parts` as column ranges of one matrix."""
    one, at, out = torch.cat(parts, 1), 0, []
    for p in parts:
        out.append(one[:, at:at + p.shape[1]])
        at += p.shape[1]
    return out


def prompt_args(q, k, v, out, qo, ko, heads, kv, hd, t, scale, max_k=0):
    return smoe_amd.SmoePromptAttnArgs(
        q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), out=out.data_ptr(), q_offsets=qo.data_ptr(),
        k_offsets=ko.data_ptr() if ko is not None else None, q_stride=q.stride(0), k_stride=k.stride(0),
        v_stride=v.stride(0), out_stride=out.stride(0), n_seqs=qo.numel() - 1, q_rows=q.shape[0], k_rows=k.shape[0],
        max_k=max_k, num_heads=heads, num_kv_heads=kv, head_dim=hd, type=smoe_amd.TYPES[t], scale=scale)


def attend64(q, k, v, limit, scale, rel_p, rel_s=0.0):
    """q [n, G, d], k and v [N, d] (any type), query i sees keys 0 .. limit[i]: (output, bound) in 64 bits.
    rel_p: the weights' own relative rounding; rel_s: the scores' relative to sum |q k|, beyond fp32 sums."""
    q, k, v = q.double(), k.double(), v.double()
    n, g, d = q.shape
    N = k.shape[0]
    if N == 0:
        z = torch.zeros_like(q)
        return z, z
    kt = k.T.contiguous()
    s = scale * (q.reshape(-1, d) @ kt).reshape(n, g, N)
    mag = scale * (q.abs().reshape(-1, d) @ kt.abs()).reshape(n, g, N)
    hidden = torch.arange(N, device=q.device) > limit[:, None]
    s = s.masked_fill(hidden[:, None], -float("inf"))
    mag = mag.masked_fill(hidden[:, None], 0.0)
    top = s.amax(-1, keepdim=True)
    e = (s - torch.where(top > -float("inf"), top, 0.0)).exp()
    tot = e.sum(-1, keepdim=True)
    w = e / torch.where(tot > 0, tot, 1.0)
    out = (w.reshape(-1, N) @ v).reshape(n, g, d)
    a = (w.reshape(-1, N) @ v.abs()).reshape(n, g, d)
    # scores: fp32 sums of d products, the scaled score and maximum (3 roundings of values up to mag)
    ds = mag.amax(-1, keepdim=True) * (4 * d ** 0.5 * U + 4 * U + rel_s)
    return out, a * (rel_p + 2 * ds + 4 * (N + 64) ** 0.5 * U + 2.0 ** -20)


def prompt64(q, k, v, nq, nk, q0, k0, heads, kv, hd, scale, t):
    """Outputs and bounds of all rows of the sequences; rows outside them: NaN bounds."""
    G = heads // kv
    out = torch.zeros(q.shape[0], heads, hd, dtype=torch.float64, device="cuda")
    tol = torch.full_like(out, float("nan"))
    rel_p = 0.0 if t == "f32" else half_step(t)
    qo, ko = offsets(nq, q0), offsets(nk, k0)
    for b in range(len(nq)):
        a, z = qo[b], qo[b + 1]
        if a == z:
            continue
        limit = torch.arange(nq[b], device="cuda") + nk[b] - nq[b]
        for j in range(kv):
            ks, vs = (x[ko[b]:ko[b + 1], j * hd:(j + 1) * hd].contiguous() for x in (k, v))
            o, e = attend64(q[a:z].reshape(-1, heads, hd)[:, j * G:(j + 1) * G], ks, vs, limit, scale, rel_p)
            out[a:z, j * G:(j + 1) * G], tol[a:z, j * G:(j + 1) * G] = o, e
    return out.reshape(q.shape[0], -1), (tol + half_step(t) * out.abs()).reshape(q.shape[0], -1)


def worst(got, ref, tol):
    """max |got - ref| / tol over the rows that have a bound (<= 1 passes)."""
    r = (got.double() - ref).abs() / (tol + 1e-300)
    r = r[~torch.isnan(tol)]
    assert not torch.isnan(r).any()
    return float(r.max()) if r.numel() else 0.0


class Cache:
    """A 4-bit cache of random codes, scales and mins."""

    def __init__(self, g, slots, kv, capacity, hd, std=0.15):
        self.kv, self.hd, self.capacity, self.slots = kv, hd, capacity, slots
        self.codes = [torch.randint(0, 256, (slots, kv, capacity, hd // 2), dtype=torch.uint8, generator=g,
                                    device="cuda") for _ in range(2)]
        self.params = []
        for _ in range(2):
            s = std * torch.exp(0.5 * randn(g, slots, kv, capacity, hd // 64))
            m = -s * (7.5 + 2 * randn(g, slots, kv, capacity, hd // 64))
            self.params.append(torch.stack([s, m], -1).to(torch.bfloat16))

    def struct(self):
        return smoe_amd.SmoeKv4Cache(
            k_codes=self.codes[0].data_ptr(), v_codes=self.codes[1].data_ptr(), k_params=self.params[0].data_ptr(),
            v_params=self.params[1].data_ptr(), n_slots=self.slots, capacity=self.capacity, num_kv_heads=self.kv,
            head_dim=self.hd)

    def parts(self, side, slot, head, n):
        """codes [n, hd] and their scales and mins [n, hd] in 64 bits."""
        c = self.codes[side][slot, head, :n]
        codes = torch.stack([c & 15, c >> 4], -1).reshape(n, self.hd).double()
        p = self.params[side][slot, head, :n].double().repeat_interleave(64, 1)
        return codes, p[..., 0], p[..., 1]


def kv4_args(q, out, lens, heads, t, scale, slots=None, max_len=0):
    return smoe_amd.SmoeKv4AttnArgs(
        q=q.data_ptr(), out=out.data_ptr(), slots=slots.data_ptr() if slots is not None else None,
        lens=lens.data_ptr(), q_stride=q.stride(0), out_stride=out.stride(0), n_seqs=q.shape[0], max_len=max_len,
        num_heads=heads, type=smoe_amd.TYPES[t], scale=scale)


def kv4_64(cache, q, lens, slots, heads, scale, t):
    """Outputs and bounds.  Codes and their scale and min enter apart, so the magnitudes of a sum are those of
    15 s + |m| (value times 2 at most); q and the weighted V scales carry 21 bits."""
    G, hd = heads // cache.kv, cache.hd
    out = torch.zeros(q.shape[0], heads, hd, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    for b, n in enumerate(lens):
        for j in range(cache.kv if n else 0):
            (kc, ks, km), (vc, vs, vm) = (cache.parts(x, slots[b], j, n) for x in range(2))
            qq = q[b].double().reshape(heads, hd)[j * G:(j + 1) * G]
            s = scale * (qq @ (kc * ks + km).T.contiguous())
            mag = scale * (qq.abs() @ (kc * ks.abs() + km.abs()).T.contiguous())
            # (q in f16 halves: 2^-21 of the head's largest value)
            mag += scale * qq.abs().amax(-1, keepdim=True) * (kc * ks.abs()).sum(-1)
            w = torch.softmax(s, -1)
            a = w @ (vc * vs.abs() + vm.abs())
            ds = mag.amax(-1, keepdim=True) * (4 * hd ** 0.5 * U + 4 * U + 2.0 ** -21)
            out[b, j * G:(j + 1) * G] = w @ (vc * vs + vm)
            tol[b, j * G:(j + 1) * G] = a * (2 * ds + 4 * (n + 64) ** 0.5 * U + 2.0 ** -19)
    out = out.reshape(q.shape[0], -1)
    return out, tol.reshape(q.shape[0], -1) + half_step(t) * out.abs()


def np_u16(x):
    return x.cpu().view(torch.int16).numpy().view(np.uint16)
