// attn_kv4.hip -- attention of one token a sequence over the 4-bit cache (gfx950):
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(s_j - max s),  s_j = scale log2(e) q . k_j,
//   k_j = c s_g + m_g in groups of 64 dims, codes c of 0 .. 15
//
//   k_attn_kv4   one block per (sequence, KV head, up to 16 of its query heads, part of
//                the positions), four or eight waves that take tiles of 32 positions in turn and
//                are merged in LDS.
//     Codes go through v_mfma_f32_16x16x32_f16 as they are: 0 .. 15 are exact in f16
//     (two codes a word by one and-or with the bits of 1024 or 64 and one packed
//     subtraction), the scales and mins are applied to the fp32 sums of a group:
//       q . k_j = sum_g s_g (sum c q) + m_g (sum_g q)
//     The query goes in as f16, at a power of two that brings the head's largest value to
//     8 .. 16: 16-bit types once (exact, but for values under 2^-17 of that one, which keep
//     2^-28 of it), f32 twice, the value and what its rounding left (22 bits).
//     Scores come out transposed, S^T = K Q^T: lane (m = l & 15, q = l >> 4) has the
//     scores of head m at positions 4 q + i (+ 16), which are the B operand of the
//     weighted sum O^T = V^T P^T as they stand.  P is multiplied by the V scale of its
//     position and group first and put in f16 twice like q, at a power of two that the
//     largest scale of the group so far sets (once would save 5 % of a bf16 call, but code
//     times scale and min may cancel, and then its 11 bits are not enough for a bf16 result):
//     the mins' part, sum p m_g, is one fp32 sum a group.
//     A tile's bytes come by direct loads into the wave's own two LDS buffers, one tile
//     ahead, with no register held meanwhile: 128 registers leave four waves a SIMD, whose
//     loads in flight and whose arithmetic cover each other.  K operands are 8-byte reads
//     (16 dims of a position), V operands 4-bit transposing reads (a lane gets 8 positions
//     of two dims); 16-byte pieces of a row are exchanged so that neither meets a bank
//     twice.  The 16 lanes that share a position would unpack the same scales and mins, so
//     each pair is put into floats by one lane and passed on through LDS.
//     Bound: the cache's bytes where there are many (head_dim 128, 4 KV heads: 48 sequences of
//     8192, bf16, 226 MB in 51 us, 4.4 TB/s; 16 of 32768, 64 query heads, f32, 302 MB in
//     66 us, 4.6 TB/s, of which the loads alone take 58; a large copy reaches 5.1 TB/s), else
//     the launch and one chain of length, tile and query loads: one sequence of 777, 7.5 us.
//   k_kv4_join   the parts of each (sequence, head) joined (4 us, 5 with 64 parts a row).
#include <algorithm>

#include "attn_common.hpp"
#include "kernels.hpp"

namespace smoe {

constexpr int KA_JOIN_WAVES = 4;
constexpr int KA_TILE = 32;             // positions of a wave step
constexpr int KA_HEADS = 16;            // query heads of a block (MFMA columns)

// A constant that the compiler holds in a vector register: (w & mask) | bits is then one
// v_and_or_b32, which takes no literals.
__device__ __forceinline__ uint32_t in_vgpr(uint32_t c)
{
    uint32_t r;
    asm("v_mov_b32 %0, %1" : "=v"(r) : "s"(c));
    return r;
}
// 8 codes of a word as f16: codes 0 4 | 1 5 | 2 6 | 3 7
__device__ __forceinline__ f16x8_t codes8(uint32_t w, uint32_t even, uint32_t odd)
{
    const uint32_t v = w >> 8;
    const uint4 b = make_uint4((w & even) | 0x64006400u, (w & odd) | 0x54005400u, (v & even) | 0x64006400u,
                               (v & odd) | 0x54005400u);
    const _Float16 lo = static_cast<_Float16>(-1024.f), hi = static_cast<_Float16>(-64.f);
    const f16x8_t bias = {lo, lo, hi, hi, lo, lo, hi, hi};
    return __builtin_bit_cast(f16x8_t, b) + bias;
}
// place j of codes8 holds code code_at(j)
__device__ constexpr int code_at(int j) { return (j >> 1) + 4 * (j & 1); }

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
// maximum over the lanes that agree in l % N (N = 1, 2, 4), left in every lane
template <int N>
__device__ __forceinline__ uint32_t residue_max(uint32_t v)
{
    if constexpr (N < 2) v = max(v, dpp_u32<DPP_QUAD_XOR1>(0u, v));
    if constexpr (N < 4) v = max(v, dpp_u32<DPP_QUAD_XOR2>(0u, v));
    v = max(v, dpp_u32<DPP_ROW_ROR4>(0u, v));
    v = max(v, dpp_u32<DPP_ROW_ROR8>(0u, v));
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return max(b[0], b[1]);
}
// orders this wave's LDS writes before its later reads of other lanes' values, and reads before writes
__device__ __forceinline__ void wave_lds_order()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
// lane l's 16 (4) bytes at base + off (off per lane) land at LDS byte address lds + 16 l (4 l)
__device__ __forceinline__ void lds_load16(const void* base, uint32_t off, uint32_t lds)
{
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds)
                 : "memory", "m0");
}
__device__ __forceinline__ void lds_load4(const void* base, uint32_t off, uint32_t lds)
{
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(off), "s"(base), "s"(lds)
                 : "memory", "m0");
}

// a wave's buffer of one tile: K codes, V codes (rows of RB bytes), then the scale and min
// words of K and of V as they are, later the floats of one of them
template <int HD, int KW>
struct Kv4Shape {
    static constexpr int NG = HD / 64;
    static constexpr int RB = HD / 2, PIECES = RB / 16;
    static constexpr int CODES = KA_TILE * RB;
    static constexpr int NC = CODES / 1024;                    // direct loads of a tile's codes
    static constexpr int PAIRS = KA_TILE * NG;
    static constexpr int NP = (PAIRS + 63) / 64;               // direct loads of a tile's pairs
    static constexpr int BUF = 2 * CODES + 2 * NP * 256;
    static constexpr int RS = HD + 4;                          // padded row of a head in the merge
    static constexpr int LDS = KW * (2 * BUF > KA_HEADS * RS * 4 ? 2 * BUF : KA_HEADS * RS * 4);
    static constexpr int WAVES_PER_SIMD = HD == 256 ? 2 : 4;
    static_assert(2 * PAIRS * 4 <= 2 * NP * 256, "the floats of K or V fit the words' place");
    // piece c of row r stands at piece c ^ swz(r)
    __host__ __device__ static constexpr int swz(int r) { return r / (256 / RB) & (PIECES - 1); }
};

// ---------------------------------------------------------------------------
// Which positions a block takes.  The sequences' tiles are cut into p.units parts or fewer
// of the same length, as near as may be, so that sequences of different lengths give every
// block the same work (32 sequences of up to 8192, as it was then: 24 us against 26 with the longest one's
// parts for all): the shortest length at which the parts of all sequences are few enough.
// Every wave works it out from the lengths, 64 sequences a pass; for more than 64 it takes
// the length that is enough at any rate.
// ---------------------------------------------------------------------------
struct Kv4Seq {                                 // a lane's sequence
    int32_t slot;
    uint32_t n, tiles;                          // positions (0: none, or an index out of range)
};
__device__ __forceinline__ Kv4Seq kv4_seq(const Kv4Attn& p, uint32_t b, bool flag)
{
    const uint32_t at = min(b, p.n_seqs - 1);
    Kv4Seq s{p.slots ? p.slots[at] : static_cast<int32_t>(at), static_cast<uint32_t>(p.lens[at]), 0};
    if (static_cast<uint32_t>(s.slot) >= p.c.n_slots || s.n > p.c.capacity) {   // (or below zero)
        if (flag && b < p.n_seqs) flag_range(p.err);
        s.slot = 0;
        s.n = 0;
    }
    if (b >= p.n_seqs) s.n = 0;
    s.tiles = (s.n + KA_TILE - 1) / KA_TILE;
    return s;
}
// ceil(tiles / part), for tiles below 2^20: the product may fall short of a whole quotient by
// its rounding, never reach past the next
__device__ __forceinline__ uint32_t kv4_parts(uint32_t tiles, uint32_t part)
{
    const uint32_t c = static_cast<uint32_t>(static_cast<float>(tiles) * __builtin_amdgcn_rcpf(static_cast<float>(part)));
    return c * part < tiles ? c + 1 : c;
}
// a / b, off by less than 2 or 2^-18 of itself (three roundings, each under 2^-22)
__device__ __forceinline__ uint32_t quotient(uint32_t a, uint32_t b)
{
    return static_cast<uint32_t>(static_cast<float>(a) * __builtin_amdgcn_rcpf(static_cast<float>(b)));
}
__device__ __forceinline__ uint32_t wave_total(uint32_t v) { return readlane_u32(wave_scan(v), WAVE - 1); }
// tiles of a part; s: the lane's sequence of the first 64; flag: says so if one of the others is out of range
__device__ __forceinline__ uint32_t kv4_part_tiles(const Kv4Attn& p, int lane, const Kv4Seq& s, bool flag)
{
    uint32_t total = wave_total(s.tiles), top = wave_max_u32(s.tiles);
    for (uint32_t i = WAVE; i < p.n_seqs; i += WAVE) {
        const uint32_t t = kv4_seq(p, i + lane, flag).tiles;
        total += wave_total(t);
        top = max(top, wave_max_u32(t));
    }
    // (a tile a wave, and no more parts than the join takes; lo may be one less than total / units)
    uint32_t lo = max(max(p.waves, (top + JOIN_MAX - 1) / JOIN_MAX), quotient(total, p.units));
    // enough at any rate: total / part + one a sequence
    const uint32_t q = quotient(total, p.units - p.n_seqs);
    uint32_t hi = max(lo, min(q + (q >> 18) + 2, top));
    if (p.n_seqs > WAVE) return hi;
    while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2;
        if (wave_total(kv4_parts(s.tiles, mid)) <= p.units) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

// behind the parts in the scratch: first part and number of parts of every sequence
template <int HD>
__device__ __forceinline__ uint2* kv4_info(const Kv4Attn& p)
{
    return reinterpret_cast<uint2*>(p.part + part_floats(static_cast<size_t>(p.units) * p.c.num_kv_heads * p.group, 1, HD));
}

template <int HD, typename T, int KW>
__global__ __launch_bounds__(KW * WAVE, (Kv4Shape<HD, KW>::WAVES_PER_SIMD))
void k_attn_kv4(Kv4Attn p, uint32_t n_sub)
{
    using S = Kv4Shape<HD, KW>;
    constexpr int NG = S::NG, RB = S::RB, RS = S::RS;
    constexpr bool Q2 = sizeof(T) == 4;         // q as two f16
    extern __shared__ __align__(16) float buf[];    // the waves' tiles; before and after, rows of heads
    __shared__ float qsum[KA_HEADS * NG], mw[KW * KA_HEADS], lw[KW * KA_HEADS];

    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m16 = lane & 15, q = lane >> 4;
    const uint32_t G = p.group, nkv = p.c.num_kv_heads;
    const uint32_t sub = blockIdx.x % n_sub, kvh = blockIdx.x / n_sub % nkv;
    const uint32_t unit = blockIdx.x / n_sub / nkv;
    const uint32_t hbase = kvh * G + sub * KA_HEADS;            // first query head of the block
    const uint32_t ng = min(static_cast<uint32_t>(KA_HEADS), G - sub * KA_HEADS);
    const uint32_t heads = nkv * G;

    // ---- the block's positions ------------------------------------------------
    uint32_t seq = unit, n, t0 = 0, t1, parts = 1;
    int32_t slot;
    if (p.units) {
        Kv4Seq s = kv4_seq(p, lane, blockIdx.x == 0);
        const uint32_t part = kv4_part_tiles(p, lane, s, blockIdx.x == 0);
        if (blockIdx.x == 0 && wv == 0) {                       // for the join: each sequence's first part and parts
            Kv4Seq z = s;
            for (uint32_t i = 0, base = 0; i < p.n_seqs; i += WAVE) {
                if (i) z = kv4_seq(p, i + lane, false);
                const uint32_t c = kv4_parts(z.tiles, part), upto = base + wave_scan(c);
                if (i + lane < p.n_seqs) kv4_info<HD>(p)[i + lane] = make_uint2(upto - c, c);
                base = readlane_u32(upto, WAVE - 1);
            }
        }
        for (uint32_t i = 0, base = 0;;) {
            const uint32_t c = kv4_parts(s.tiles, part), upto = base + wave_scan(c);
            if (const uint64_t past = __ballot(upto > unit)) {
                const int f = __ffsll(static_cast<unsigned long long>(past)) - 1;
                seq = i + f;
                n = readlane_u32(s.n, f);
                slot = __builtin_amdgcn_readlane(s.slot, f);
                parts = readlane_u32(c, f);
                const uint32_t tiles = readlane_u32(s.tiles, f), len = kv4_parts(tiles, parts);
                t0 = (unit - (readlane_u32(upto, f) - parts)) * len;
                t1 = min(tiles, t0 + len);
                break;
            }
            base = readlane_u32(upto, WAVE - 1);
            i += WAVE;
            if (i >= p.n_seqs) return;                          // (fewer parts than units)
            s = kv4_seq(p, i + lane, false);
        }
    } else {
        const Kv4Seq s = kv4_seq(p, seq, threadIdx.x == 0);
        n = __builtin_amdgcn_readfirstlane(s.n);
        slot = __builtin_amdgcn_readfirstlane(s.slot);
        t1 = __builtin_amdgcn_readfirstlane(s.tiles);
    }
    const size_t line0 = (static_cast<size_t>(slot) * nkv + kvh) * p.c.capacity;
    const uint8_t* kc = p.c.codes[0] + line0 * RB;
    const uint8_t* vc = p.c.codes[1] + line0 * RB;
    const uint8_t* kpar = reinterpret_cast<const uint8_t*>(p.c.params[0]) + line0 * (4 * NG);
    const uint8_t* vpar = reinterpret_cast<const uint8_t*>(p.c.params[1]) + line0 * (4 * NG);

    // ---- direct loads of tile t into buffer b of this wave --------------------------
    uint8_t* mine = reinterpret_cast<uint8_t*>(buf) + wv * (2 * S::BUF);
    const uint32_t lds = static_cast<uint32_t>(
        reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)mine));
    auto issue = [&](uint32_t t, int b) {
        const uint64_t at = static_cast<uint64_t>(t) * KA_TILE;
        const uint32_t last = n - 1 - t * KA_TILE;              // past the end: the last position again
        const uint32_t to = lds + b * S::BUF;
#pragma unroll
        for (int i = 0; i < S::NC; ++i) {
            const int byte = i * 1024 + lane * 16, row = byte / RB, piece = (byte % RB / 16) ^ S::swz(row);
            const uint32_t off = min(static_cast<uint32_t>(row), last) * RB + piece * 16;
            lds_load16(kc + at * RB, off, to + i * 1024);
            lds_load16(vc + at * RB, off, to + S::CODES + i * 1024);
        }
#pragma unroll
        for (int i = 0; i < S::NP; ++i) {
            const uint32_t pr = (lane + 64 * i) % S::PAIRS;
            const uint32_t off = (min(pr / NG, last) * NG + pr % NG) * 4;
            lds_load4(kpar + at * (4 * NG), off, to + 2 * S::CODES + i * 256);
            lds_load4(vpar + at * (4 * NG), off, to + 2 * S::CODES + (S::NP + i) * 256);
        }
    };

    if (t0 + wv < t1) issue(t0 + wv, 0);

    // ---- the query heads: a power of two each, then f16 --------------------------
    // (through the waves' second buffers, which the first tile leaves alone)
    constexpr int HPW = KA_HEADS / KW;
    static_assert(HPW * RS * 4 <= S::BUF, "a wave's heads fit its second buffer");
    auto head_row = [&](uint32_t g) {
        return reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(buf) + g / HPW * (2 * S::BUF) + S::BUF) + g % HPW * RS;
    };
    float x[HPW][NG];
#pragma unroll
    for (int i = 0; i < HPW; ++i) {
        const uint32_t g = wv * HPW + i;
        const T* src = static_cast<const T*>(p.q) + seq * p.q_stride + (hbase + min(g, ng - 1)) * HD;
#pragma unroll
        for (int j = 0; j < NG; ++j) x[i][j] = static_cast<float>(src[j * WAVE + lane]);
    }
#pragma unroll
    for (int i = 0; i < HPW; ++i) {
        const uint32_t g = wv * HPW + i;
        float top = 0.f;
#pragma unroll
        for (int j = 0; j < NG; ++j) top = fmaxf(top, fabsf(x[i][j]));
        // brings the largest value to 8 .. 16 (nothing for 0 or an infinity)
        const uint32_t e = (__float_as_uint(wave_max(top)) >> 23) & 0xFFu;
        const uint32_t es = e == 0 || e == 255 ? 130u : min(max(e, 4u), 250u);
        const float down = __uint_as_float((257u - es) << 23);       // 2^(130 - es)
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            const float v = g < ng ? x[i][j] * down : 0.f;
            head_row(g)[j * WAVE + lane] = v;
            const float gs = wave_sum(v);                     // group j
            if (lane == 0) qsum[g * NG + j] = gs;
        }
        if (lane == 0) mw[g] = __uint_as_float((es - 3u) << 23);     // 2^(es - 130)
    }
    __syncthreads();
    f16x8_t qh[NG][2], ql[NG][2];
    float qs[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        qs[g] = qsum[m16 * NG + g];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float* r = head_row(m16) + 64 * g + 16 * q + 8 * i;
            uint4 hi, lo;
            split2(r[code_at(0)], r[code_at(1)], hi.x, lo.x);
            split2(r[code_at(2)], r[code_at(3)], hi.y, lo.y);
            split2(r[code_at(4)], r[code_at(5)], hi.z, lo.z);
            split2(r[code_at(6)], r[code_at(7)], hi.w, lo.w);
            qh[g][i] = __builtin_bit_cast(f16x8_t, hi);
            ql[g][i] = __builtin_bit_cast(f16x8_t, lo);
        }
    }
    const float up = mw[m16] * p.scale_log2;    // of the sums below: scores in powers of two
    __syncthreads();

    // ---- the positions --------------------------------------------------------------
    const uint32_t even = in_vgpr(0x000F000Fu), odd = in_vgpr(0x00F000F0u);
    float mx = -INFINITY, sum = 0.f, vmin[NG];  // of head m16 (sums: this lane's positions)
    f32x4v_t acc[NG][4];                        // dim 64 g + 16 d + 4 q + i of head m16 at [g][d][i]
    int ebits[NG];                              // exponent field of the group's largest V scale so far
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        vmin[g] = 0.f;
        ebits[g] = 27;
#pragma unroll
        for (int d = 0; d < 4; ++d) acc[g][d] = f32x4v_t{0.f, 0.f, 0.f, 0.f};
    }

    // this lane's operand places in a buffer: K row 16 u + m16, V rows of positions 16 (k / 4) + 4 q + k % 4
    // for k = m16 % 8 (dims 16 (2 e + m16 / 8) of a transposing read e)
    const uint32_t kat = m16 * RB + (((q >> 1) ^ S::swz(m16)) * 16) + (q & 1) * 8;
    const uint32_t vrow = 16 * ((m16 >> 2) & 1) + 4 * q + (m16 & 3);
    const uint32_t vat = vrow * RB + (S::swz(vrow) * 16) + (m16 >> 3) * 8;
    // the sums are rescaled when a head's maximum has grown by more than 2^SLACK: weights up to that
    constexpr float SLACK = 4.f;
    constexpr int VLIFT = 10;
    auto step = [&](uint32_t t, int b0) {
        const uint8_t* kl = mine + b0 * S::BUF;
        const uint8_t* vl = kl + S::CODES;
        uint32_t* words = reinterpret_cast<uint32_t*>(mine + b0 * S::BUF + 2 * S::CODES);
        float* par = reinterpret_cast<float*>(words);           // scale, min: [NG][KA_TILE] each
        uint32_t kp[S::NP], vp[S::NP];
#pragma unroll
        for (int i = 0; i < S::NP; ++i) {
            kp[i] = words[lane + 64 * i];
            vp[i] = words[(S::NP + i) * 64 + lane];
        }
        // scales and mins as floats, one pair a lane; read back as the lane's positions 16 u + 4 q + 0 .. 3
        auto put_pairs = [&](const uint32_t (&w)[S::NP], float f) {
            wave_lds_order();
#pragma unroll
            for (int i = 0; i < S::NP; ++i) {
                const uint32_t pr = (lane + 64 * i) % S::PAIRS, at = pr % NG * KA_TILE + pr / NG;
                par[at] = __uint_as_float(w[i] << 16) * f;
                par[NG * KA_TILE + at] = __uint_as_float(w[i] & 0xFFFF0000u);
            }
            wave_lds_order();
        };
        auto pairs = [&](int what, int g, int u) {
            return *reinterpret_cast<const f32x4v_t*>(par + (what * NG + g) * KA_TILE + 16 * u + 4 * q);
        };
        put_pairs(kp, 1.f);
        // ---- scores ----
        float s[8];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            f32x4v_t sc;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                f32x4v_t d = {0.f, 0.f, 0.f, 0.f};
                const uint2 w = *reinterpret_cast<const uint2*>(kl + u * (16 * RB) + (kat ^ (32 * g)));
                const f16x8_t c0 = codes8(w.x, even, odd), c1 = codes8(w.y, even, odd);
                if constexpr (Q2) {
                    d = __builtin_amdgcn_mfma_f32_16x16x32_f16(c0, ql[g][0], d, 0, 0, 0);
                    d = __builtin_amdgcn_mfma_f32_16x16x32_f16(c1, ql[g][1], d, 0, 0, 0);
                }
                d = __builtin_amdgcn_mfma_f32_16x16x32_f16(c0, qh[g][0], d, 0, 0, 0);
                d = __builtin_amdgcn_mfma_f32_16x16x32_f16(c1, qh[g][1], d, 0, 0, 0);
                const f32x4v_t ks = pairs(0, g, u), km = pairs(1, g, u);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    sc[i] = g ? fmaf(ks[i], d[i], fmaf(km[i], qs[g], sc[i])) : fmaf(ks[i], d[i], km[i] * qs[g]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) s[4 * u + i] = sc[i];
        }
        const uint32_t b = t * KA_TILE;
        if (b + KA_TILE > n) {
            asm volatile("" : "+v"(s[0]));      // (a branch, not selects in every tile)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (b + 16 * (j / 4) + 4 * q + j % 4 >= n) s[j] = -INFINITY;
        }
        float mt = fmaxf(s[0], s[1]);
#pragma unroll
        for (int j = 2; j < 8; ++j) mt = fmaxf(mt, s[j]);
        mt = quads_max(mt) * up;
        // V scales: the largest exponent of a group sets the power of two of its P
        int eb[NG], e = 0;
        bool grown = false;
        uint32_t vs = 0;
#pragma unroll
        for (int i = 0; i < S::NP; ++i) vs = max(vs, vp[i] & 0x7FFFu);
        vs = residue_max<NG>(vs);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            eb[g] = max(ebits[g], static_cast<int>(readlane_u32(vs, g) >> 7));
            grown |= eb[g] != ebits[g];
            e = lane % NG == g ? eb[g] : e;
        }
        if (__ballot(mt > mx + SLACK) || grown) {
            const float mn = fmaxf(mx, mt);
            const float f = mx > -INFINITY ? __builtin_amdgcn_exp2f(mx - mn) : 0.f;
            sum *= f;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                vmin[g] *= f;
                const float fg = __builtin_amdgcn_ldexpf(f, ebits[g] - eb[g]);
                ebits[g] = eb[g];
#pragma unroll
                for (int d = 0; d < 4; ++d) acc[g][d] *= fg;
            }
            mx = mn;
        }
        put_pairs(vp, __builtin_amdgcn_ldexpf(1.f, 127 + VLIFT - e));  // P times a scale stays under 2^15
        const float m0 = mx > -INFINITY ? mx : 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            s[j] = __builtin_amdgcn_exp2f(fmaf(s[j], up, -m0));
            sum += s[j];
        }
        // ---- weighted values ----
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            uint4 hi, lo;
            float y[8];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const f32x4v_t vs = pairs(0, g, u), vm = pairs(1, g, u);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    y[4 * u + i] = s[4 * u + i] * vs[i];
                    vmin[g] = fmaf(s[4 * u + i], vm[i], vmin[g]);
                }
            }
            // in the order of codes8's places
            split2(y[code_at(0)], y[code_at(1)], hi.x, lo.x);
            split2(y[code_at(2)], y[code_at(3)], hi.y, lo.y);
            split2(y[code_at(4)], y[code_at(5)], hi.z, lo.z);
            split2(y[code_at(6)], y[code_at(7)], hi.w, lo.w);
            const f16x8_t ph = __builtin_bit_cast(f16x8_t, hi), pl = __builtin_bit_cast(f16x8_t, lo);
#pragma unroll
            for (int e2 = 0; e2 < 2; ++e2) {
                typedef int i32x2_t __attribute__((ext_vector_type(2)));
                typedef __attribute__((address_space(3))) i32x2_t lds_i32x2;
                const i32x2_t w = __builtin_amdgcn_ds_read_tr4_b64_v2i32((lds_i32x2*)(vl + (vat ^ (32 * g + 16 * e2))));
#pragma unroll
                for (int d2 = 0; d2 < 2; ++d2) {
                    const f16x8_t cv = codes8(static_cast<uint32_t>(w[d2]), even, odd);
                    f32x4v_t& o = acc[g][2 * e2 + d2];
                    o = __builtin_amdgcn_mfma_f32_16x16x32_f16(cv, pl, o, 0, 0, 0);
                    o = __builtin_amdgcn_mfma_f32_16x16x32_f16(cv, ph, o, 0, 0, 0);
                }
            }
        }
    };
    int b = 0;
    for (uint32_t t = t0 + wv; t < t1; t += KW, b ^= 1) {
        // tile t has arrived, and nothing of the other buffer is still being read
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        if (t + KW < t1) issue(t + KW, b ^ 1);
        step(t, b);
    }

    // ---- merge: the four lanes of a head, then the waves, then parts ------------------
    __syncthreads();                            // (every wave's tiles are read)
    sum = quads_sum(sum);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        vmin[g] = quads_sum(vmin[g]);
        const float down = __builtin_amdgcn_ldexpf(1.f, ebits[g] - 127 - VLIFT);
#pragma unroll
        for (int d = 0; d < 4; ++d)
            *reinterpret_cast<float4*>(buf + (wv * KA_HEADS + m16) * RS + 64 * g + 16 * d + 4 * q) =
                make_float4(fmaf(acc[g][d][0], down, vmin[g]), fmaf(acc[g][d][1], down, vmin[g]),
                            fmaf(acc[g][d][2], down, vmin[g]), fmaf(acc[g][d][3], down, vmin[g]));
    }
    if (q == 0) {
        mw[wv * KA_HEADS + m16] = mx;
        lw[wv * KA_HEADS + m16] = sum;
    }
    __syncthreads();
    for (uint32_t o = threadIdx.x; o < ng * HD; o += KW * WAVE) {
        const uint32_t g = o / HD, d = o % HD, head = hbase + g;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < KW; ++w) M = fmaxf(M, mw[w * KA_HEADS + g]);
        const float m0 = M > -INFINITY ? M : 0.f;
        float L = 0.f, A = 0.f;
#pragma unroll
        for (int w = 0; w < KW; ++w) {
            const float f = __builtin_amdgcn_exp2f(mw[w * KA_HEADS + g] - m0);
            L = fmaf(f, lw[w * KA_HEADS + g], L);
            A = fmaf(f, buf[(w * KA_HEADS + g) * RS + d], A);
        }
        if (parts == 1) {
            static_cast<T*>(p.out)[seq * p.out_stride + head * HD + d] = static_cast<T>(L == 0.f ? 0.f : A * (1.0f / L));
        } else {
            const size_t at = static_cast<size_t>(unit) * heads + head;
            p.part[part_acc_at(static_cast<size_t>(p.units) * heads, 1) + at * HD + d] = A;
            if (d == 0) {
                p.part[2 * at] = M;
                p.part[2 * at + 1] = L;
            }
        }
    }
}

// one wave per (sequence, head)
template <int HD, typename T>
__global__ __launch_bounds__(KA_JOIN_WAVES * WAVE)
void k_kv4_join(Kv4Attn p)
{
    const int lane = threadIdx.x & 63;
    const uint32_t heads = p.c.num_kv_heads * p.group;
    const uint32_t w = blockIdx.x * KA_JOIN_WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), seq = w / heads;
    if (seq >= p.n_seqs) return;
    const uint2 info = kv4_info<HD>(p)[seq];
    const uint32_t first = info.x, parts = info.y;
    if (parts == 1) return;                                     // (its block wrote the row)
    const size_t at = static_cast<size_t>(first) * heads + w % heads;
    float o[HD / WAVE];
    join_parts<HD>(p.part + 2 * at, p.part + part_acc_at(static_cast<size_t>(p.units) * heads, 1) + at * HD, parts, heads,
                   lane, o);
    store_row<HD>(static_cast<T*>(p.out) + seq * p.out_stride + (w % heads) * HD, o, lane);
}

void kv4_plan(Kv4Attn& a, uint32_t head_dim, uint32_t max_len)
{
    const uint32_t n_sub = (a.group + KA_HEADS - 1) / KA_HEADS;
    const uint32_t tiles = max_len / KA_TILE + (max_len % KA_TILE != 0);
    // As many parts as blocks are resident at once (1024 of four waves, 512 of eight; half at head_dim 256), each with
    // a tile a wave or more: 16 sequences of 32768 over 4 KV heads 72.8 us in 16 parts (1024 blocks of four waves),
    // 78.0 in 8, 74.8 in 12, 76.2 in 24; one of 777 over 4 KV heads 6.9 us in 7 parts, 8.5 in 6, 15.5 in one.
    // Sequences whole where they fill half of that, or no sequence has a second part.
    auto most = [&](uint32_t waves) { return (head_dim == 256 ? 2048 : 4096) / waves / (a.c.num_kv_heads * n_sub); };
    auto units = [&](uint32_t waves) {
        return static_cast<uint32_t>(std::min<uint64_t>(most(waves), static_cast<uint64_t>(a.n_seqs) * ((tiles + waves - 1) / waves)));
    };
    // Eight waves a block (half the query set-ups, merges and parts: 16 of 32768 65.4 us against 68.4, 16 of 3000 14.0
    // against 17.5) where the sequences fill the resident blocks with them, four parts or more each and no more than a
    // tenth of the blocks left over (48 of 8192 58.8 against 51.2, 64 ragged ones 27.7 against 26.3, one of 777 7.8
    // against 7.6 and a longer join).
    const uint32_t m8 = most(8);
    const bool eight = units(8) == m8 && m8 >= 4 * static_cast<uint64_t>(a.n_seqs) && m8 % a.n_seqs * 10 <= m8;
    a.waves = eight ? 8 : 4;
    a.units = units(a.waves);
    if (a.units < 2 * static_cast<uint64_t>(a.n_seqs)) a.units = 0;
}

size_t kv4_scratch_bytes(const Kv4Attn& a, uint32_t head_dim)
{
    if (a.units == 0) return 0;
    return part_floats(static_cast<size_t>(a.units) * a.c.num_kv_heads * a.group, 1, head_dim) * sizeof(float) +
           a.n_seqs * sizeof(uint2);
}

template <int HD, typename T, int KW>
static hipError_t launch_kv4(const Kv4Attn& a, uint32_t n_sub, hipStream_t s)
{
    constexpr uint32_t lds = Kv4Shape<HD, KW>::LDS;
    static_assert(lds <= 155 * 1024, "LDS of a CU, beside the static arrays");
    if constexpr (lds > 60 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(k_attn_kv4<HD, T, KW>),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return e;
    }
    launch_kernel_lds(k_attn_kv4<HD, T, KW>, dim3((a.units ? a.units : a.n_seqs) * a.c.num_kv_heads * n_sub), dim3(KW * WAVE),
                      lds, s, a, n_sub);
    return hipGetLastError();
}

hipError_t launch_attention_kv4(const Kv4Attn& a, uint32_t head_dim, uint32_t type, hipStream_t s)
{
    return with_type_and_head(type, head_dim, [&](auto t, auto hd) {
        constexpr int HD = decltype(hd)::value;
        using T = decltype(t);
        const uint32_t n_sub = (a.group + KA_HEADS - 1) / KA_HEADS, heads = a.c.num_kv_heads * a.group;
        const hipError_t e = a.waves == 8 ? launch_kv4<HD, T, 8>(a, n_sub, s) : launch_kv4<HD, T, 4>(a, n_sub, s);
        if (e != hipSuccess || a.units == 0) return e;
        launch_kernel(k_kv4_join<HD, T>, dim3((a.n_seqs * heads + KA_JOIN_WAVES - 1) / KA_JOIN_WAVES),
                      dim3(KA_JOIN_WAVES * WAVE), s, a);
        return hipGetLastError();
    });
}

}  // namespace smoe
