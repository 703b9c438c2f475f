// attn_rows.hip -- row kernels on either side of the attention kernels (gfx950):
//
//   k_qk_rows     RMSNorm of every query and key head (x / sqrt(mean(x^2) + 1e-6) * w)
//                 and RoPE on its pairs (d, d + head_dim / 2) by the tables' row
//                 positions[row]: what k_attn_decode does for one token, for many
//                 (decode.cpp:155-186).  A lane holds eight dims of both halves of
//                 a head, so a pair never leaves its lane; the eight cosines and
//                 sines of a lane serve all heads of its wave.
//   k_kv4_append  K and V rows to the 4-bit cache: groups of 64 values quantized as
//                 k_quantize_q4_min does (bf16 min and scale, the same operations in
//                 the same order, so the same bits).
//   k_kv4_read    the inverse, code * scale + min (exact products, one rounding).
//
// All three move each value once and are bound by that (or, for few rows, by their
// latency).  A lane's piece is eight consecutive values: 16 bytes of a 16-bit type.
// Measured (heads of 128; a large copy reaches 5.1 TB/s): 4096 rows of 32 + 4 heads, bf16,
// 75 MB in 13.5 us; 17 rows, f32, 2.9 us.  6000 rows of 4 + 4 heads, bf16, appended in 8.2
// us (16 MB: a look-up of the row's place, one dependent load, then the quantizer's
// arithmetic), read in 5.5; 48 rows, f32, 3.3 and 3.0.
// Floating-point contraction is off: the quantizer's steps round one by one.
#include <algorithm>

#include "attn_common.hpp"
#include "kernels.hpp"

#pragma clang fp contract(off)

namespace smoe {

constexpr int RW_WAVES = 4;
constexpr int RW_THREADS = RW_WAVES * WAVE;

// (the entry points keep rows times heads under 2^31)
static dim3 row_grid(uint32_t n_rows, uint32_t per_row) { return dim3((n_rows * per_row + RW_WAVES - 1) / RW_WAVES); }

// sum over segments of N = 2, 4, 8 or 16 lanes, left in every lane
template <int N>
__device__ __forceinline__ float seg_sum(float v)
{
    if constexpr (N >= 2) v += dpp_f32<DPP_QUAD_XOR1>(0.f, v);
    if constexpr (N >= 4) v += dpp_f32<DPP_QUAD_XOR2>(0.f, v);
    if constexpr (N >= 8) v += dpp_f32<DPP_ROW_HALF_MIRROR>(0.f, v);
    if constexpr (N >= 16) v += dpp_f32<DPP_ROW_ROR8>(0.f, v);
    return v;
}
__device__ __forceinline__ float seg8_min(float v)
{
    v = fminf(v, dpp_f32<DPP_QUAD_XOR1>(v, v));
    v = fminf(v, dpp_f32<DPP_QUAD_XOR2>(v, v));
    return fminf(v, dpp_f32<DPP_ROW_HALF_MIRROR>(v, v));
}

// ---------------------------------------------------------------------------
// RMSNorm + RoPE: a wave takes hpw heads of one row
// ---------------------------------------------------------------------------
template <int HD, typename T>
__global__ __launch_bounds__(RW_THREADS)
void k_qk_rows(QkRows p, uint32_t hpw, uint32_t waves_per_row)
{
    constexpr int HALF = HD / 2, LPH = HALF / 8, HPS = WAVE / LPH;   // lanes a head, heads a step
    const int lane = threadIdx.x & 63;
    const uint32_t w = blockIdx.x * RW_WAVES + (threadIdx.x >> 6), row = w / waves_per_row;
    if (row >= p.n_rows) return;
    const uint32_t heads = p.num_heads + p.num_kv_heads;
    const uint32_t h0 = w % waves_per_row * hpw, h1 = min(h0 + hpw, heads);
    const int li = lane % LPH, d = li * 8;
    float cs[8], sn[8];
    const bool turn = p.rope_cos != nullptr;
    if (turn) {
        int32_t pos = p.positions[row];
        if (static_cast<uint32_t>(pos) >= p.n_positions) {
            if (lane == 0) flag_range(p.err);
            pos = 0;
        }
        load8(p.rope_cos + static_cast<size_t>(pos) * HALF + d, cs);
        load8(p.rope_sin + static_cast<size_t>(pos) * HALF + d, sn);
    }
    for (uint32_t h = h0 + lane / LPH; h < h1; h += HPS) {
        const bool is_q = h < p.num_heads;
        const uint32_t hh = is_q ? h : h - p.num_heads;
        const T* src = static_cast<const T*>(is_q ? p.q : p.k) + row * (is_q ? p.q_stride : p.k_stride) + hh * HD;
        T* dst = static_cast<T*>(is_q ? p.q_out : p.k_out) + row * (is_q ? p.q_out_stride : p.k_out_stride) + hh * HD;
        const uint16_t* nw = is_q ? p.q_norm_w : p.k_norm_w;
        float a[8], b[8];
        load8(src + d, a);
        load8(src + HALF + d, b);
        if (nw) {
            float ss = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) ss = fmaf(a[j], a[j], fmaf(b[j], b[j], ss));
            ss = seg_sum<LPH>(ss);
            const float inv = 1.0f / sqrtf(ss / static_cast<float>(HD) + 1e-6f);
            float wa[8], wb[8];
            load8(reinterpret_cast<const __bf16*>(nw) + d, wa);
            load8(reinterpret_cast<const __bf16*>(nw) + HALF + d, wb);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                a[j] = (a[j] * inv) * wa[j];
                b[j] = (b[j] * inv) * wb[j];
            }
        }
        if (turn) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float x = a[j], y = b[j];
                a[j] = x * cs[j] - y * sn[j];
                b[j] = x * sn[j] + y * cs[j];
            }
        }
        store8(dst + d, a);
        store8(dst + HALF + d, b);
    }
}

hipError_t launch_qk_rows(const QkRows& a, uint32_t head_dim, uint32_t type, hipStream_t s)
{
    return with_type_and_head(type, head_dim, [&](auto t, auto hd) {
        constexpr int HD = decltype(hd)::value;
        constexpr uint32_t step = WAVE / (HD / 16);            // heads of one step
        const uint32_t heads = a.num_heads + a.num_kv_heads;
        // one step a wave until there are some 8 waves a SIMD; then all heads of a
        // row in one, whose tables are read once
        uint32_t hpw = step;
        while (hpw < heads && static_cast<uint64_t>(a.n_rows) * ((heads + hpw - 1) / hpw) > 8192) hpw += step;
        const uint32_t per_row = (heads + hpw - 1) / hpw;
        launch_kernel(k_qk_rows<HD, decltype(t)>, row_grid(a.n_rows, per_row), dim3(RW_THREADS), s, a, hpw, per_row);
        return hipGetLastError();
    });
}

// ---------------------------------------------------------------------------
// the 4-bit cache: a wave takes some groups of one row
// ---------------------------------------------------------------------------
// what the call says of 64 sequences, one a lane
struct CallSeqs {
    int32_t first, end, start, slot;                       // rows first .. end - 1, position of the first, slot
};
__device__ __forceinline__ CallSeqs load_seqs(const Kv4Rows& p, uint32_t i, int lane)
{
    const uint32_t b = min(i + lane, p.n_seqs - 1);
    CallSeqs s;
    s.first = p.offsets ? p.offsets[b] : static_cast<int32_t>(b);
    s.end = p.offsets ? p.offsets[b + 1] : static_cast<int32_t>(b) + 1;
    s.start = p.start[b];
    s.slot = p.slots ? p.slots[b] : static_cast<int32_t>(b);
    if (i + lane >= p.n_seqs) s.end = s.first;
    return s;
}

struct CachePlace {
    uint32_t slot, pos;
    bool in_seq, ok;       // the row is of a sequence; its place is in the cache
    bool later;            // a later sequence of the call names the same place
};
// Sequence, slot and position of a row, by the whole wave; U passes of 64 sequences have their loads in flight at once
// (4000 appended rows of 4000 sequences: 24 us against 26 with one)
template <int U>
__device__ __forceinline__ CachePlace place_by(const Kv4Rows& p, uint32_t row, int lane)
{
    CachePlace c{};
    uint32_t seq = 0;
    // (without offsets row r is sequence r's)
    for (uint32_t i0 = p.offsets ? 0u : row / WAVE * WAVE; i0 < p.n_seqs; i0 += U * WAVE) {
        CallSeqs ss[U];
#pragma unroll
        for (int u = 0; u < U; ++u) ss[u] = load_seqs(p, i0 + u * WAVE, lane);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const CallSeqs& s = ss[u];
            const uint32_t i = i0 + u * WAVE;
            if (!c.in_seq) {
                // the first sequence that ends behind the row
                const uint64_t after = __ballot(s.end > static_cast<int32_t>(row) && i + lane < p.n_seqs);
                if (!after) continue;
                const int f = __ffsll(static_cast<unsigned long long>(after)) - 1;
                seq = i + f;
                const int32_t at = static_cast<int32_t>(row) - __builtin_amdgcn_readlane(s.first, f);
                if (at < 0) return c;
                c.in_seq = true;
                c.slot = __builtin_amdgcn_readlane(s.slot, f);
                c.pos = static_cast<uint32_t>(__builtin_amdgcn_readlane(s.start, f)) + static_cast<uint32_t>(at);
                c.ok = c.slot < p.c.n_slots && c.pos < p.c.capacity;
                if (!c.ok) {
                    if (lane == 0) flag_range(p.err);
                    return c;
                }
                if (!p.slots) return c;
            }
            // (a lane without a sequence of its own has first = end)
            c.later = __ballot(i + lane > seq && static_cast<uint32_t>(s.slot) == c.slot &&
                               c.pos - static_cast<uint32_t>(s.start) < static_cast<uint32_t>(s.end - s.first)) != 0;
            if (c.later) return c;
        }
    }
    return c;
}
__device__ __forceinline__ CachePlace place_of_row(const Kv4Rows& p, uint32_t row, int lane)
{
    return p.n_seqs <= WAVE ? place_by<1>(p, row, lane) : place_by<4>(p, row, lane);
}

// eight lanes' group of 64 values to its place
template <int HD>
__device__ __forceinline__ void store_group(const Kv4Rows& p, const CachePlace& c, uint32_t side, uint32_t hg, int lane,
                                            const float (&x)[8])
{
    constexpr uint32_t NG = HD / 64;
    const uint32_t head = hg / NG, part = hg % NG;
    float lo = x[0], hi = x[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) {
        lo = fminf(lo, x[j]);
        hi = fmaxf(hi, x[j]);
    }
    lo = seg8_min(lo);
    hi = -seg8_min(-hi);
    const float span = (hi - lo) / 15.0f;
    uint32_t sb = __builtin_bit_cast(uint16_t, static_cast<__bf16>(span));
    if ((sb & 0x7FFFu) == 0) sb = 0x3F80u;                     // a constant group: scale 1
    const uint32_t mb = __builtin_bit_cast(uint16_t, static_cast<__bf16>(lo));
    const float s = bf16_to_f32(sb), m = bf16_to_f32(mb);
    // code = rint((x - m) / s), the difference and the quotient each rounded.  The quotient by s's reciprocal r:
    // one step makes r the rounded 1 / s (checked for all 128 mantissas that a bf16 scale has, from any first r
    // within two steps), and with that q + (d - q s) r is the rounded d / s (Markstein), in three operations
    // instead of a division's two dozen.  Scales near the ends of the range divide.
    uint32_t word = 0;
    if (s > 0x1p-100f && s < 0x1p100f) {
        float r = __builtin_amdgcn_rcpf(s);
        r = __builtin_fmaf(__builtin_fmaf(-s, r, 1.f), r, r);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float d = x[j] - m, q = d * r;
            const float c0 = rintf(__builtin_fmaf(__builtin_fmaf(-q, s, d), r, q));
            word |= static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(c0, 0.f), 15.f))) << (4 * j);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float q = x[j] - m;
            q = q / s;
            word |= static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(rintf(q), 0.f), 15.f))) << (4 * j);
        }
    }
    const size_t line = (static_cast<size_t>(c.slot) * p.c.num_kv_heads + head) * p.c.capacity + c.pos;
    reinterpret_cast<uint32_t*>(p.c.codes[side] + line * (HD / 2) + part * 32)[lane & 7] = word;
    if ((lane & 7) == 0) reinterpret_cast<uint32_t*>(p.c.params[side])[line * NG + part] = sb | (mb << 16);
}

template <int HD, typename T>
__global__ __launch_bounds__(RW_THREADS)
void k_kv4_append(Kv4Rows p, uint32_t gpw, uint32_t waves_per_row)
{
    constexpr uint32_t NG = HD / 64, STEP = WAVE / 8;          // eight lanes a group, eight groups a step
    const int lane = threadIdx.x & 63;
    const uint32_t w = blockIdx.x * RW_WAVES + (threadIdx.x >> 6), row = w / waves_per_row;
    if (p.lens_out && blockIdx.x == 0) {
        for (uint32_t b = threadIdx.x; b < p.n_seqs; b += RW_THREADS)
            p.lens_out[b] = p.start[b] + (p.offsets ? p.offsets[b + 1] - p.offsets[b] : 1);
    }
    if (row >= p.n_rows) return;
    const uint32_t per_side = p.c.num_kv_heads * NG, groups = 2 * per_side;
    const uint32_t g0 = w % waves_per_row * gpw, g1 = min(g0 + gpw, groups);
    auto load = [&](uint32_t g, float (&x)[8]) {
        const uint32_t side = g >= per_side, hg = g - side * per_side;
        load8(static_cast<const T*>(p.rows[side]) + row * p.stride[side] + hg * 64 + (lane & 7) * 8, x);
    };
    uint32_t g = g0 + (lane >> 3);
    float x[8];
    if (g < g1) load(g, x);                                    // (requested before its place is known)
    const CachePlace c = place_of_row(p, row, lane);
    if (!c.ok || c.later) return;
    while (g < g1) {
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = x[j];
        if (g + STEP < g1) load(g + STEP, x);
        const uint32_t side = g >= per_side;
        store_group<HD>(p, c, side, g - side * per_side, lane, y);
        g += STEP;
    }
}

template <int HD, typename T>
__global__ __launch_bounds__(RW_THREADS)
void k_kv4_read(Kv4Rows p, uint32_t gpw, uint32_t waves_per_row)
{
    constexpr uint32_t NG = HD / 64, STEP = WAVE / 8;
    const int lane = threadIdx.x & 63;
    const uint32_t w = blockIdx.x * RW_WAVES + (threadIdx.x >> 6), row = w / waves_per_row;
    if (row >= p.n_rows) return;
    const uint32_t per_side = p.c.num_kv_heads * NG, groups = 2 * per_side;
    const uint32_t g0 = w % waves_per_row * gpw, g1 = min(g0 + gpw, groups);
    const CachePlace c = place_of_row(p, row, lane);
    if (!c.in_seq) return;                                     // rows behind the last sequence stay
    for (uint32_t g = g0 + (lane >> 3); g < g1; g += STEP) {
        const uint32_t side = g >= per_side, hg = g - side * per_side, head = hg / NG, part = hg % NG;
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = 0.f;                // a place outside the cache reads as zeros
        if (c.ok) {
            const size_t line = (static_cast<size_t>(c.slot) * p.c.num_kv_heads + head) * p.c.capacity + c.pos;
            const uint32_t word = reinterpret_cast<const uint32_t*>(p.c.codes[side] + line * (HD / 2) + part * 32)[lane & 7];
            const uint32_t sm = reinterpret_cast<const uint32_t*>(p.c.params[side])[line * NG + part];
            const float s = __uint_as_float(sm << 16), m = __uint_as_float(sm & 0xFFFF0000u);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = static_cast<float>((word >> (4 * j)) & 15u) * s + m;
        }
        store8(static_cast<T*>(p.rows[side]) + row * p.stride[side] + hg * 64 + (lane & 7) * 8, x);
    }
}

// waves of a row: one step (eight groups) each until there are some 8 waves a SIMD
static uint32_t row_waves(uint32_t n_rows, uint32_t groups, uint32_t& gpw)
{
    gpw = WAVE / 8;
    while (gpw < groups && static_cast<uint64_t>(n_rows) * ((groups + gpw - 1) / gpw) > 8192) gpw += WAVE / 8;
    return (groups + gpw - 1) / gpw;
}

hipError_t launch_kv4_append(const Kv4Rows& a, uint32_t head_dim, uint32_t type, hipStream_t s)
{
    return with_type_and_head(type, head_dim, [&](auto t, auto hd) {
        constexpr int HD = decltype(hd)::value;
        uint32_t gpw;
        const uint32_t per_row = row_waves(a.n_rows, 2 * a.c.num_kv_heads * (HD / 64), gpw);
        const dim3 grid = a.n_rows ? row_grid(a.n_rows, per_row) : dim3(1);   // (no rows: the lengths alone)
        launch_kernel(k_kv4_append<HD, decltype(t)>, grid, dim3(RW_THREADS), s, a, gpw, per_row);
        return hipGetLastError();
    });
}
hipError_t launch_kv4_read(const Kv4Rows& a, uint32_t head_dim, uint32_t type, hipStream_t s)
{
    return with_type_and_head(type, head_dim, [&](auto t, auto hd) {
        constexpr int HD = decltype(hd)::value;
        uint32_t gpw;
        const uint32_t per_row = row_waves(a.n_rows, 2 * a.c.num_kv_heads * (HD / 64), gpw);
        launch_kernel(k_kv4_read<HD, decltype(t)>, row_grid(a.n_rows, per_row), dim3(RW_THREADS), s, a, gpw, per_row);
        return hipGetLastError();
    });
}

}  // namespace smoe
