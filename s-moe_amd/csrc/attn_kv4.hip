// attn_kv4.hip -- attention of one token a sequence over the 4-bit cache (gfx950):
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(s_j - max s),  s_j = scale log2(e) q . k_j,
//   k_j = c s_g + m_g in groups of 64 dims, codes c of 0 .. 15
//
//   k_attn_kv4   one block per (sequence, KV head, up to 16 of its query heads, part of
//                the positions), four waves that take tiles of 32 positions in turn and
//                are merged in LDS.
//     Codes go through v_mfma_f32_16x16x32_f16 as they are: 0 .. 15 are exact in f16
//     (two codes a word by one and-or with the bits of 1024 or 64 and one packed
//     subtraction), the scales and mins are applied to the fp32 sums of a group:
//       q . k_j = sum_g s_g (sum c q) + m_g (sum_g q)
//     The query is put in f16 twice, the value and what its rounding left (22 bits;
//     a power of two a head keeps it in range), so a score is as exact as an fp32 sum.
//     Scores come out transposed, S^T = K Q^T: lane (m = l & 15, q = l >> 4) has the
//     scores of head m at positions 4 q + i (+ 16), which are the B operand of the
//     weighted sum O^T = V^T P^T as they stand.  P is multiplied by the V scale of its
//     position and group first and put in f16 twice like q, at a power of two that the
//     largest scale of the group so far sets: the mins' part, sum p m_g, is one fp32 sum a group.
//     K rows are read 8 bytes a lane and group (16 dims), V rows 2 bytes (4 dims of
//     group g: 64 g + 4 m), the next tile's while this one is computed.
//   k_kv4_join   the parts of each (sequence, head) joined.
#include <algorithm>

#include "attn_common.hpp"
#include "kernels.hpp"

namespace smoe {

constexpr int KA_WAVES = 4;
constexpr int KA_THREADS = KA_WAVES * WAVE;
constexpr int KA_TILE = 32;             // positions of a wave step
constexpr int KA_HEADS = 16;            // query heads of a block (MFMA columns)

// 8 codes of a word as f16: codes 0 4 | 1 5 | 2 6 | 3 7
__device__ __forceinline__ f16x8_t codes8(uint32_t w)
{
    const uint32_t v = w >> 8;
    const uint4 b = make_uint4((w & 0x000F000Fu) | 0x64006400u, (w & 0x00F000F0u) | 0x54005400u,
                               (v & 0x000F000Fu) | 0x64006400u, (v & 0x00F000F0u) | 0x54005400u);
    const _Float16 lo = static_cast<_Float16>(-1024.f), hi = static_cast<_Float16>(-64.f);
    const f16x8_t bias = {lo, lo, hi, hi, lo, lo, hi, hi};
    return __builtin_bit_cast(f16x8_t, b) + bias;
}
// place j of codes8 holds code code_at(j)
__device__ constexpr int code_at(int j) { return (j >> 1) + 4 * (j & 1); }

// x = hi + lo in f16
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo)
{
    const auto h = __builtin_amdgcn_cvt_pkrtz(a, b);
    hi = __builtin_bit_cast(uint32_t, h);
    const f16x2_t hv = __builtin_bit_cast(f16x2_t, hi);
    const auto l = __builtin_amdgcn_cvt_pkrtz(a - static_cast<float>(hv.x), b - static_cast<float>(hv.y));
    lo = __builtin_bit_cast(uint32_t, l);
}

// maximum / sum over the lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float quads_max(float v)
{
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return half_max(fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1])));
}
__device__ __forceinline__ float quads_sum(float v)
{
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return half_sum(__uint_as_float(a[0]) + __uint_as_float(a[1]));
}
__device__ __forceinline__ uint32_t quads_max_u32(uint32_t v)
{
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return max(b[0], b[1]);
}

// the raw bytes of 32 positions that a lane needs
template <int NG>
struct Kv4Tile {
    uint2 k[2][NG];          // codes of position 16 u + m, dims 64 g + 16 q ..
    uint32_t v[8][NG];       // codes of position 16 (j / 4) + 4 q + j % 4, dims 64 g + 4 m ..
    uint32_t kp[8][NG];      // scale | min << 16 of the same positions
    uint32_t vp[8][NG];
};

template <int HD, typename T>
__global__ __launch_bounds__(KA_THREADS, (HD == 256 ? 1 : 2))
void k_attn_kv4(Kv4Attn p, uint32_t n_sub)
{
    constexpr int NG = HD / 64;
    constexpr int RS = HD + 4;                  // padded row of a head in LDS
    extern __shared__ __align__(16) float buf[];    // [KA_WAVES][KA_HEADS][RS]
    __shared__ float qsum[KA_HEADS * NG], mw[KA_WAVES * KA_HEADS], lw[KA_WAVES * KA_HEADS];

    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m16 = lane & 15, q = lane >> 4;
    const uint32_t G = p.group, nkv = p.c.num_kv_heads;
    const uint32_t sub = blockIdx.x % n_sub, kvh = blockIdx.x / n_sub % nkv, seq = blockIdx.x / n_sub / nkv;
    const uint32_t hbase = kvh * G + sub * KA_HEADS;            // first query head of the block
    const uint32_t ng = min(static_cast<uint32_t>(KA_HEADS), G - sub * KA_HEADS);

    // ---- the block's positions ------------------------------------------------
    const int32_t slot = p.slots ? p.slots[seq] : static_cast<int32_t>(seq), len = p.lens[seq];
    uint32_t n = static_cast<uint32_t>(len);
    if (static_cast<uint32_t>(slot) >= p.c.n_slots || len < 0 || n > p.c.capacity) {
        if (threadIdx.x == 0) flag_range(p.err);
        n = 0;                                                  // (a row of zeros)
    }
    const uint32_t tiles = (n + KA_TILE - 1) / KA_TILE, part = (tiles + p.splits - 1) / p.splits;
    const uint32_t t0 = min(tiles, blockIdx.y * part), t1 = min(tiles, t0 + part);
    const size_t line0 = (static_cast<size_t>(n ? slot : 0) * nkv + kvh) * p.c.capacity;
    const uint8_t* kc = p.c.codes[0] + line0 * (HD / 2);
    const uint8_t* vc = p.c.codes[1] + line0 * (HD / 2);
    const uint32_t* kpar = reinterpret_cast<const uint32_t*>(p.c.params[0]) + line0 * NG;
    const uint32_t* vpar = reinterpret_cast<const uint32_t*>(p.c.params[1]) + line0 * NG;

    // positions past the end: the last one again (masked, and its V weights 0)
    auto load_tile = [&](uint32_t t, Kv4Tile<NG>& x) {
        const uint32_t b = t * KA_TILE, last = n - 1;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const size_t at = min(b + 16 * u + m16, last);
#pragma unroll
            for (int g = 0; g < NG; ++g)
                x.k[u][g] = *reinterpret_cast<const uint2*>(kc + at * (HD / 2) + 32 * g + 8 * q);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const size_t at = min(b + 16 * (j / 4) + 4 * q + j % 4, last);
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                x.v[j][g] = *reinterpret_cast<const uint16_t*>(vc + at * (HD / 2) + 32 * g + 2 * m16);
                x.kp[j][g] = kpar[at * NG + g];
                x.vp[j][g] = vpar[at * NG + g];
            }
        }
    };
    Kv4Tile<NG> ta;
    if (t0 + wv < t1) load_tile(t0 + wv, ta);

    // ---- the query heads: scaled, then f16 halves ---------------------------------
    for (uint32_t g = wv; g < KA_HEADS; g += KA_WAVES) {
        const T* src = static_cast<const T*>(p.q) + seq * p.q_stride + (hbase + min(g, ng - 1)) * HD;
        float x[HD / WAVE], top = 0.f;
#pragma unroll
        for (int j = 0; j < HD / WAVE; ++j) {
            x[j] = g < ng ? static_cast<float>(src[j * WAVE + lane]) * p.scale_log2 : 0.f;
            top = fmaxf(top, fabsf(x[j]));
        }
        // a power of two that brings the largest value to 8 .. 16 (none for 0 or an infinity)
        const uint32_t e = (__float_as_uint(wave_max(top)) >> 23) & 0xFFu;
        const uint32_t es = e == 0 || e == 255 ? 127u : min(max(e, 4u), 250u);
        const float down = __uint_as_float((257u - es) << 23);       // 2^(130 - es)
#pragma unroll
        for (int j = 0; j < HD / WAVE; ++j) {
            x[j] *= down;
            buf[g * RS + j * WAVE + lane] = x[j];
            const float gs = wave_sum(x[j]);                      // group j
            if (lane == 0) qsum[g * NG + j] = gs;
        }
        if (lane == 0) mw[g] = __uint_as_float((es - 3u) << 23);   // 2^(es - 130), 1 / down
    }
    __syncthreads();
    f16x8_t qh[NG][2], ql[NG][2];
    float qs[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        qs[g] = qsum[m16 * NG + g];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float* r = buf + m16 * RS + 64 * g + 16 * q + 8 * i;
            uint4 hi, lo;
            split2(r[code_at(0)], r[code_at(1)], hi.x, lo.x);
            split2(r[code_at(2)], r[code_at(3)], hi.y, lo.y);
            split2(r[code_at(4)], r[code_at(5)], hi.z, lo.z);
            split2(r[code_at(6)], r[code_at(7)], hi.w, lo.w);
            qh[g][i] = __builtin_bit_cast(f16x8_t, hi);
            ql[g][i] = __builtin_bit_cast(f16x8_t, lo);
        }
    }
    const float up = mw[m16];
    __syncthreads();

    // ---- the positions --------------------------------------------------------------
    float mx = -INFINITY, sum = 0.f, vmin[NG];  // of head m16 (sums: this lane's positions)
    f32x4v_t acc[NG][4];                        // dim 64 g + 4 (4 q + i) + d of head m16 at [g][d][i]
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        vmin[g] = 0.f;
#pragma unroll
        for (int d = 0; d < 4; ++d) acc[g][d] = f32x4v_t{0.f, 0.f, 0.f, 0.f};
    }
    int ebits[NG];                              // exponent field of the group's largest V scale so far
    float vup[NG];                              // 2^(14 - (ebits - 127)): brings P times a V scale under 2^15
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        ebits[g] = 27;
        vup[g] = __builtin_amdgcn_ldexpf(1.f, 127 + 14 - 27);
    }

    auto step = [&](uint32_t t, const Kv4Tile<NG>& x) {
        const uint32_t b = t * KA_TILE;
        f32x4v_t sc[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            sc[u] = f32x4v_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                f32x4v_t d = {0.f, 0.f, 0.f, 0.f};
                const f16x8_t c0 = codes8(x.k[u][g].x), c1 = codes8(x.k[u][g].y);
                d = __builtin_amdgcn_mfma_f32_16x16x32_f16(c0, ql[g][0], d, 0, 0, 0);
                d = __builtin_amdgcn_mfma_f32_16x16x32_f16(c1, ql[g][1], d, 0, 0, 0);
                d = __builtin_amdgcn_mfma_f32_16x16x32_f16(c0, qh[g][0], d, 0, 0, 0);
                d = __builtin_amdgcn_mfma_f32_16x16x32_f16(c1, qh[g][1], d, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t w = x.kp[4 * u + i][g];
                    sc[u][i] = fmaf(__uint_as_float(w << 16), d[i], fmaf(__uint_as_float(w & 0xFFFF0000u), qs[g], sc[u][i]));
                }
            }
        }
        float s[8], mt = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const bool in = b + 16 * (j / 4) + 4 * q + j % 4 < n;
            s[j] = in ? sc[j / 4][j % 4] * up : -INFINITY;
            mt = fmaxf(mt, s[j]);
        }
        // V scales: the largest exponent of a group sets the power of two of its P
        bool grown = false;
        int eb[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            uint32_t vs = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) vs = max(vs, x.vp[j][g] & 0x7FFFu);
            eb[g] = static_cast<int>(__builtin_amdgcn_readfirstlane(quads_max_u32(vs)) >> 7);
            grown |= eb[g] > ebits[g];
        }
        mt = quads_max(mt);
        if (__ballot(mt > mx) || grown) {
            const float mn = fmaxf(mx, mt);
            const float f = mx > -INFINITY ? __builtin_amdgcn_exp2f(mx - mn) : 0.f;
            sum *= f;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                vmin[g] *= f;
                const int e = max(eb[g], ebits[g]);
                const float fg = __builtin_amdgcn_ldexpf(f, ebits[g] - e);
                ebits[g] = e;
                vup[g] = __builtin_amdgcn_ldexpf(1.f, 127 + 14 - e);
#pragma unroll
                for (int d = 0; d < 4; ++d) acc[g][d] *= fg;
            }
            mx = mn;
        }
        const float m0 = mx > -INFINITY ? mx : 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            s[j] = __builtin_amdgcn_exp2f(s[j] - m0);
            sum += s[j];
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            uint4 hi, lo;
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t w = x.vp[j][g];
                y[j] = s[j] * vup[g] * __uint_as_float(w << 16);
                vmin[g] = fmaf(s[j], __uint_as_float(w & 0xFFFF0000u), vmin[g]);
            }
            split2(y[0], y[1], hi.x, lo.x);
            split2(y[2], y[3], hi.y, lo.y);
            split2(y[4], y[5], hi.z, lo.z);
            split2(y[6], y[7], hi.w, lo.w);
            const f16x8_t ph = __builtin_bit_cast(f16x8_t, hi), pl = __builtin_bit_cast(f16x8_t, lo);
            // positions j, j + 1 of a dim side by side
            uint32_t w2[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w2[j] = x.v[2 * j][g] | (x.v[2 * j + 1][g] << 16);
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const uint32_t mask = d & 1 ? 0x00F000F0u : 0x000F000Fu, one = d & 1 ? 0x54005400u : 0x64006400u;
                const _Float16 neg = static_cast<_Float16>(d & 1 ? -64.f : -1024.f);
                const f16x8_t bias = {neg, neg, neg, neg, neg, neg, neg, neg};
                const int sh = d & 2 ? 8 : 0;
                const uint4 cb = make_uint4(((w2[0] >> sh) & mask) | one, ((w2[1] >> sh) & mask) | one,
                                            ((w2[2] >> sh) & mask) | one, ((w2[3] >> sh) & mask) | one);
                const f16x8_t cv = __builtin_bit_cast(f16x8_t, cb) + bias;
                acc[g][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(cv, pl, acc[g][d], 0, 0, 0);
                acc[g][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(cv, ph, acc[g][d], 0, 0, 0);
            }
        }
    };
    if constexpr (HD <= 128) {
        Kv4Tile<NG> tb;
        for (uint32_t t = t0 + wv; t < t1; t += 2 * KA_WAVES) {
            if (t + KA_WAVES < t1) load_tile(t + KA_WAVES, tb);
            step(t, ta);
            if (t + KA_WAVES >= t1) break;
            if (t + 2 * KA_WAVES < t1) load_tile(t + 2 * KA_WAVES, ta);
            step(t + KA_WAVES, tb);
        }
    } else {
        // (no registers for a second tile)
        for (uint32_t t = t0 + wv; t < t1; t += KA_WAVES) {
            step(t, ta);
            if (t + KA_WAVES < t1) load_tile(t + KA_WAVES, ta);
        }
    }

    // ---- merge: the four lanes of a head, then the waves, then parts ------------------
    sum = quads_sum(sum);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        vmin[g] = quads_sum(vmin[g]);
        const float down = __builtin_amdgcn_ldexpf(1.f, ebits[g] - 127 - 14);
#pragma unroll
        for (int i = 0; i < 4; ++i)             // dims 64 g + 4 (4 q + i) + 0 .. 3
            *reinterpret_cast<float4*>(buf + (wv * KA_HEADS + m16) * RS + 64 * g + 16 * q + 4 * i) =
                make_float4(fmaf(acc[g][0][i], down, vmin[g]), fmaf(acc[g][1][i], down, vmin[g]),
                            fmaf(acc[g][2][i], down, vmin[g]), fmaf(acc[g][3][i], down, vmin[g]));
    }
    if (q == 0) {
        mw[wv * KA_HEADS + m16] = mx;
        lw[wv * KA_HEADS + m16] = sum;
    }
    __syncthreads();
    const uint32_t heads = nkv * G;
    const size_t nrow = static_cast<size_t>(p.n_seqs) * heads;
    for (uint32_t o = threadIdx.x; o < ng * HD; o += KA_THREADS) {
        const uint32_t g = o / HD, d = o % HD, head = hbase + g;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < KA_WAVES; ++w) M = fmaxf(M, mw[w * KA_HEADS + g]);
        const float m0 = M > -INFINITY ? M : 0.f;
        float L = 0.f, A = 0.f;
#pragma unroll
        for (int w = 0; w < KA_WAVES; ++w) {
            const float f = __builtin_amdgcn_exp2f(mw[w * KA_HEADS + g] - m0);
            L = fmaf(f, lw[w * KA_HEADS + g], L);
            A = fmaf(f, buf[(w * KA_HEADS + g) * RS + d], A);
        }
        if (p.splits == 1) {
            static_cast<T*>(p.out)[seq * p.out_stride + head * HD + d] = static_cast<T>(L == 0.f ? 0.f : A * (1.0f / L));
        } else {
            const size_t at = (static_cast<size_t>(seq) * heads + head) * p.splits + blockIdx.y;
            p.part[part_acc_at(nrow, p.splits) + at * HD + d] = A;
            if (d == 0) {
                p.part[2 * at] = M;
                p.part[2 * at + 1] = L;
            }
        }
    }
}

// one wave per (sequence, head)
template <int HD, typename T>
__global__ __launch_bounds__(KA_THREADS)
void k_kv4_join(Kv4Attn p)
{
    const int lane = threadIdx.x & 63;
    const uint32_t heads = p.c.num_kv_heads * p.group;
    const uint32_t w = blockIdx.x * KA_WAVES + (threadIdx.x >> 6), seq = w / heads;
    if (seq >= p.n_seqs) return;
    const size_t nrow = static_cast<size_t>(p.n_seqs) * heads, at = static_cast<size_t>(w) * p.splits;
    float o[HD / WAVE];
    join_parts<HD>(p.part + 2 * at, p.part + part_acc_at(nrow, p.splits) + at * HD, p.splits, lane, o);
    store_row<HD>(static_cast<T*>(p.out) + seq * p.out_stride + (w % heads) * HD, o, lane);
}

void kv4_plan(Kv4Attn& a, uint32_t head_dim, uint32_t max_len)
{
    const uint32_t n_sub = (a.group + KA_HEADS - 1) / KA_HEADS;
    const uint64_t blocks = static_cast<uint64_t>(a.n_seqs) * a.c.num_kv_heads * n_sub;
    const uint32_t tiles = max_len / KA_TILE + (max_len % KA_TILE != 0);
    // some four blocks a CU, a tile a wave or more
    const uint64_t want = std::min<uint64_t>(JOIN_MAX, std::max<uint64_t>(1, 1024 / std::max<uint64_t>(1, blocks)));
    a.splits = std::max<uint32_t>(1, std::min<uint32_t>(static_cast<uint32_t>(want), tiles / KA_WAVES));
}

size_t kv4_scratch_bytes(const Kv4Attn& a, uint32_t head_dim)
{
    if (a.splits == 1) return 0;
    return part_floats(static_cast<size_t>(a.n_seqs) * a.c.num_kv_heads * a.group, a.splits, head_dim) * sizeof(float);
}

hipError_t launch_attention_kv4(const Kv4Attn& a, uint32_t head_dim, uint32_t type, hipStream_t s)
{
    return with_type_and_head(type, head_dim, [&](auto t, auto hd) {
        constexpr int HD = decltype(hd)::value;
        using T = decltype(t);
        const uint32_t n_sub = (a.group + KA_HEADS - 1) / KA_HEADS, heads = a.c.num_kv_heads * a.group;
        constexpr uint32_t lds = KA_WAVES * KA_HEADS * (HD + 4) * sizeof(float);
        if constexpr (lds > 64 * 1024) {
            const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(k_attn_kv4<HD, T>),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, lds);
            if (e != hipSuccess) return e;
        }
        launch_kernel_lds(k_attn_kv4<HD, T>, dim3(a.n_seqs * a.c.num_kv_heads * n_sub, a.splits), dim3(KA_THREADS),
                          lds, s, a, n_sub);
        if (a.splits > 1)
            launch_kernel(k_kv4_join<HD, T>, dim3((a.n_seqs * heads + KA_WAVES - 1) / KA_WAVES), dim3(KA_THREADS), s, a);
        return hipGetLastError();
    });
}

}  // namespace smoe
