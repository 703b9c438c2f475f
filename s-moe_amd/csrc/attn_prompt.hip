// attn_prompt.hip -- causal attention of whole prompts (gfx950):
//
//   o_i = sum_{j <= i + n_k - n_q} p_ij v_j / sum_j p_ij,  p_ij = 2^(s_ij - max_j s_ij),
//   s_ij = scale log2(e) q_i . k_j
//
// over packed sequences (n_q query rows, n_k >= n_q key rows or fewer) with `group`
// query heads on each KV head.
//
//   k_attn_prompt   one block per (row tile, KV head, part of the keys): RW waves of 32
//     rows, KG groups of them that take the key tiles in turn and merge in LDS at the end.
//     Rows.  A tile's rows are (query, head of the group) pairs, the head fastest: all
//     rows of a tile read the same K and V whatever the group, and with a group of 8
//     a tile of 128 rows (RW = 4) spans 16 queries, so little of the causal diagonal is wasted
//     and a call of few tokens still fills its tiles.
//     Products.  Both run transposed, S^T = K Q^T and O^T = V^T P^T, on 32x32 MFMA:
//     a lane then holds the scores of ONE row (column l & 31), so maximum, sum, mask
//     and rescaling are per-lane values, and the scores' registers are the next
//     product's B operand as they stand (lane half h has keys 8b + 4h + i; V^T is
//     read in that key order).  The rows' only exchange is between lanes l and l ^ 32.
//     Tiles.  K and V tiles go to LDS by direct loads, one tile ahead, in 16-byte
//     pieces whose place in a row is exchanged (kswz, vswz) so that the operand reads
//     meet no bank twice: K as 16-byte pieces of 32 rows, V by transposing reads of 8 rows.
//     Order.  LDS operands are requested a few products ahead, and the weights of 16 keys
//     are formed between the products of the 16 before (sched_group_barrier; left to the
//     compiler 1 to 5 % slower).
//     16-bit types: v_mfma_f32_32x32x16 with P rounded to their type (the weights' sum is
//     of the rounded ones, in fp32).  f32: every operand as two f16 (hi + lo, 22 bits) and
//     three products for one, 16 / 3 times the rate of the fp32 MFMA.  K and V are split
//     by k_prompt_planes, at a power of two for 32 keys, Q here (one for a row), P here at
//     2^14 and the V tile's power against the smallest so far.
//     One accumulator takes the three: no cancellation sets them apart.
//     Bound: large calls by matrix cores and VALU at the clock that the power limit leaves
//     (64 query heads of 128 on 4, 8192 tokens, bf16: 1.02 ms, 1.08 PF/s of causal products; a
//     large matrix product reaches 1.2), small ones by launch, tile search and first loads
//     (~6 us) and by one wave a SIMD.  f32, 32 heads on 4: 4096 tokens 400 us, 512 tokens 22 us
//     after 4 us of k_prompt_planes; on the fp32 MFMA 45 us at 512.
//   k_prompt_planes the f16 planes of f32 K and V: one read, one write (34 MB of 4096 tokens
//     in 10 us; 3 to 5 us for the few blocks of a short prompt).
//   k_prompt_join   where the keys were split: the parts of each row rescaled to
//     their common maximum and normalised.
#include <algorithm>
#include <type_traits>

#include "attn_common.hpp"
#include "kernels.hpp"

namespace smoe {

constexpr int JOIN_WAVES = 4;

template <int HD, typename T>
struct PromptShape {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int PLANES = F32 ? 2 : 1;                 // f16 matrices that K, and V, are read as
    static constexpr int KT = F32 || HD == 256 ? 32 : 64;      // keys of a tile
    static constexpr int RB = 2 * HD;                            // bytes of a row
    static constexpr int TILE = KT * RB;                         // bytes of a plane's tile
    static constexpr int BUF = 2 * PLANES * TILE;                // K planes, then V planes
    static constexpr int LDS = 2 * BUF;                          // of a key group
    static constexpr int WAVES_PER_SIMD = HD == 256 ? 1 : 2;
    // piece c of row r stands at piece c ^ kswz(r) (K), c ^ vswz(r) (V): the rows that one
    // pass of an operand read touches then lie in different banks of the 256-byte width
    __host__ __device__ static constexpr int kswz(int r) { return RB >= 256 ? (r & 15) : ((r >> 1) & 7); }
    __host__ __device__ static constexpr int vswz(int r) { return RB >= 256 ? (r & 3) << 2 : ((r >> 1) & 1) << 2; }
};

// lane l's 16 bytes at base + off (off per lane) land at LDS byte address lds + 16 l
__device__ __forceinline__ void load_to_lds(const void* base, uint32_t off, uint32_t lds)
{
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds)
                 : "memory", "m0");
}

template <typename T>
__device__ __forceinline__ f32x16_t mma16(uint4 a, uint4 b, f32x16_t c)
{
    if constexpr (__is_same(T, _Float16))
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c,
                                                      0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b),
                                                       c, 0, 0, 0);
}
// transposing reads at `at` and eight rows on: this lane's values of four rows each
__device__ __forceinline__ uint4 read_rows8(const uint8_t* at, int row_bytes)
{
    typedef short s16x4_t __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4_t lds_s16x4;
    const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at));
    const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 8 * row_bytes));
    return __builtin_bit_cast(uint4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}
// the two values of w added to c
template <typename T>
__device__ __forceinline__ float add2(uint32_t w, float c)
{
    if constexpr (__is_same(T, _Float16)) {
        const f16x2_t one = {static_cast<_Float16>(1.f), static_cast<_Float16>(1.f)};
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, w), one, c, false);
    } else {
        const bf16x2_t one = {static_cast<__bf16>(1.f), static_cast<__bf16>(1.f)};
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w), one, c, false);
    }
}

// a tile's sequence
struct PromptSeq {
    int32_t q0, nq, k0, nk;
    uint32_t local;                             // tile of the sequence
    uint32_t ktile;                             // first key tile of the sequence, of PLANE_KEYS each
};
// what one lane knows of a sequence
struct PromptLane {
    int32_t a, z, ka, kz;
    bool ok;
};
__device__ __forceinline__ PromptLane load_seq(const PromptAttn& p, uint32_t i, int lane)
{
    const uint32_t b = min(i + lane, p.n_seqs - 1);
    PromptLane s{p.q_offsets[b], p.q_offsets[b + 1], p.k_offsets[b], p.k_offsets[b + 1], false};
    s.ok = i + lane < p.n_seqs && s.a >= 0 && s.z >= s.a && static_cast<uint32_t>(s.z) <= p.q_rows && s.ka >= 0 &&
           s.kz >= s.ka && static_cast<uint32_t>(s.kz) <= p.k_rows;
    return s;
}
constexpr int NO_POWER = 200;                   // of V values that are all 0
constexpr int PLANE_KEYS = 32;                  // keys that share a power of two in the f16 planes of f32 rows
// (a sequence without queries has none)
__device__ __forceinline__ uint32_t plane_tiles(const PromptLane& s)
{
    return s.ok && s.z > s.a ? (static_cast<uint32_t>(s.kz - s.ka) + PLANE_KEYS - 1) / PLANE_KEYS : 0;
}
// The sequence of tile `tile`, of ROWS (query, head) rows each or (KEYS) of PLANE_KEYS keys, by the whole wave; false past
// the last one.  Sequences whose offsets point outside their rows have no tiles.  U passes of 64 sequences have their
// loads in flight at once (4000 sequences of 5 tokens: 558 us against 678 with one).
template <int ROWS, bool KEYS, bool PLANES, int U>
__device__ __forceinline__ bool find_tile_by(const PromptAttn& p, uint32_t tile, int lane, bool flag, PromptSeq& s)
{
    uint32_t base = 0, kbase = 0;
    for (uint32_t i = 0; i < p.n_seqs; i += U * WAVE) {
        PromptLane ls[U];
#pragma unroll
        for (int u = 0; u < U; ++u) ls[u] = load_seq(p, i + u * WAVE, lane);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const PromptLane& l = ls[u];
            if (flag && i + u * WAVE + lane < p.n_seqs && !l.ok) flag_range(p.err);
            const uint32_t n = l.ok ? (static_cast<uint32_t>(l.z - l.a) * p.group + ROWS - 1) / ROWS : 0;
            const uint32_t kn = PLANES ? plane_tiles(l) : 0, upto = KEYS ? 0 : base + wave_scan(n),
                           kupto = PLANES ? kbase + wave_scan(kn) : 0;
            const uint64_t past = __ballot((KEYS ? kupto : upto) > tile);
            if (past) {
                const int f = __ffsll(static_cast<unsigned long long>(past)) - 1;
                s.q0 = __builtin_amdgcn_readlane(l.a, f);
                s.nq = __builtin_amdgcn_readlane(l.z, f) - s.q0;
                s.k0 = __builtin_amdgcn_readlane(l.ka, f);
                s.nk = __builtin_amdgcn_readlane(l.kz, f) - s.k0;
                s.ktile = readlane_u32(kupto, f) - readlane_u32(kn, f);
                s.local = tile - (KEYS ? s.ktile : readlane_u32(upto, f) - readlane_u32(n, f));
                return true;
            }
            base = readlane_u32(upto, WAVE - 1);
            kbase = readlane_u32(kupto, WAVE - 1);
        }
    }
    return false;
}
template <int ROWS, bool KEYS, bool PLANES>
__device__ __forceinline__ bool find_tile(const PromptAttn& p, uint32_t tile, int lane, PromptSeq& s)
{
    const bool flag = !KEYS && blockIdx.x == 0;
    return p.n_seqs <= WAVE ? find_tile_by<ROWS, KEYS, PLANES, 1>(p, tile, lane, flag, s)
                            : find_tile_by<ROWS, KEYS, PLANES, 4>(p, tile, lane, flag, s);
}

// ---------------------------------------------------------------------------
// f32 rows of K and V as f16 planes: x 2^e = hi + lo to 22 bits, e the power of two that
// brings the largest finite value of 32 keys (of one KV head, K or V) to 2^13 .. 2^14
// ---------------------------------------------------------------------------
// exponent field of the largest value -> the power that brings it to 2^13
__device__ __forceinline__ int plane_power(uint32_t field) { return 140 - static_cast<int>(min(max(field, 13u), 254u)); }

template <int HD>
__global__ __launch_bounds__(256)
void k_prompt_planes(PromptAttn p)
{
    constexpr int PIECES = PLANE_KEYS * HD / 8, PT = PIECES / 256;   // 8-value pieces of a thread, K or V
    __shared__ uint32_t tops[2][4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t tile = blockIdx.x, kvh = blockIdx.y;
    PromptSeq seq;
    if (!find_tile<1, true, true>(p, tile, lane, seq)) return;
    const uint32_t keys = min(static_cast<uint32_t>(PLANE_KEYS), seq.nk - seq.local * PLANE_KEYS);
    const uint64_t row0 = static_cast<uint64_t>(seq.k0) + seq.local * PLANE_KEYS;
    float x[2][PT][8];
    uint32_t top[2] = {0, 0};
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int i = 0; i < PT; ++i) {
            const uint32_t piece = threadIdx.x + 256 * i, row = piece / (HD / 8), c = piece % (HD / 8);
            const float* src = static_cast<const float*>(v ? p.v : p.k) +
                               (row0 + min(row, keys - 1)) * (v ? p.v_stride : p.k_stride) + kvh * HD + 8 * c;
            load8(src, x[v][i]);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t bits = __float_as_uint(x[v][i][j]) & 0x7FFFFFFFu;
                top[v] = max(top[v], bits < 0x7F800000u ? bits : 0u);
            }
        }
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        top[v] = wave_max_u32(top[v]);
        if (lane == 0) tops[v][wave] = top[v];
    }
    __syncthreads();
    int power[2];
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        const uint32_t t = max(max(tops[v][0], tops[v][1]), max(tops[v][2], tops[v][3]));
        power[v] = plane_power(t >> 23);
        if (v && t == 0) power[v] = NO_POWER;                   // (values of no size set no power for the sum)
    }
    if (threadIdx.x == 0) p.powers[static_cast<size_t>(kvh) * p.plane_tiles + tile] = make_int2(power[0], power[1]);
    const size_t plane = static_cast<size_t>(p.k_rows) * p.num_kv_heads * HD;
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int i = 0; i < PT; ++i) {
            const uint32_t piece = threadIdx.x + 256 * i, row = piece / (HD / 8), c = piece % (HD / 8);
            if (row >= keys) continue;
            float y[8], r[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                y[j] = __builtin_amdgcn_ldexpf(x[v][i][j], power[v] == NO_POWER ? 0 : power[v]);
                r[j] = y[j] - static_cast<float>(static_cast<_Float16>(y[j]));
            }
            const size_t at = 2 * v * plane + ((row0 + row) * p.num_kv_heads + kvh) * HD + 8 * c;
            store8(reinterpret_cast<_Float16*>(p.planes) + at, y);
            store8(reinterpret_cast<_Float16*>(p.planes) + at + plane, r);
        }
}

template <int HD, typename T, int RW, int KG>
__global__ __launch_bounds__(RW * KG * WAVE, (PromptShape<HD, T>::WAVES_PER_SIMD))
void k_attn_prompt(PromptAttn p)
{
    using S = PromptShape<HD, T>;
    constexpr int ROWS = 32 * RW;
    constexpr int KT = S::KT, RB = S::RB, NSUB = KT / 32, ND = HD / 32;
    extern __shared__ __align__(16) uint8_t smem[];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wv = wave % RW, kg = wave / RW;                   // wave of its key group
    const int col = lane & 31, h = lane >> 5;

    // ---- the block's tile, KV head and part ----------------------------------
    // Consecutive blocks go to the eight XCDs in turn: where the KV heads divide them
    // (or they divide the heads), a head's blocks stay on its XCDs and share their L2.
    const uint32_t nkv = p.num_kv_heads;
    uint32_t kvh, tile;
    if (8 % nkv == 0) {
        const uint32_t per = 8 / nkv, x = blockIdx.x & 7;
        kvh = x / per;
        tile = (blockIdx.x >> 3) * per + x % per;
    } else if (nkv % 8 == 0) {
        const uint32_t per = nkv / 8, r = blockIdx.x >> 3;
        kvh = (blockIdx.x & 7) * per + r % per;
        tile = r / per;
    } else {
        kvh = blockIdx.x % nkv;
        tile = blockIdx.x / nkv;
    }
    PromptSeq seq;
    if (!find_tile<ROWS, false, S::F32>(p, tile, lane, seq)) return;
    const int32_t q0 = seq.q0, nq = seq.nq, k0 = seq.k0, nk = seq.nk;
    // (sequences that share keys, around one whose offsets are wrong: more key tiles than the scratch holds)
    if (S::F32 && static_cast<uint64_t>(seq.ktile) + static_cast<uint32_t>(nk + PLANE_KEYS - 1) / PLANE_KEYS > p.plane_tiles)
        return;
    const int32_t before = nk - nq;                             // query i sees keys 0 .. i + before
    const uint32_t G = p.group, rows = static_cast<uint32_t>(nq) * G;
    // the longest tiles of a sequence first: what is left for the end of the launch is short
    const uint32_t tiles = (rows + ROWS - 1) / ROWS;
    const uint32_t r0 = (tiles - 1 - seq.local) * ROWS;
    const uint32_t r = r0 + wv * 32 + col;
    const bool live = r < rows;
    const uint32_t qi = min(r, rows - 1) / G, g = min(r, rows - 1) % G;
    const int32_t limit = live ? static_cast<int32_t>(qi) + before : -1;     // the row's last key
    // last key of the block, first and last key limits of the wave's rows
    const int32_t blk_last = static_cast<int32_t>((min(r0 + ROWS, rows) - 1) / G) + before;
    const uint32_t w0 = min(r0 + wv * 32, rows - 1), w1 = min(r0 + wv * 32 + 31, rows - 1);
    const bool wave_full = r0 + wv * 32 + 31 < rows;
    const int32_t wave_first = wave_full ? static_cast<int32_t>(w0 / G) + before : -1;
    const int32_t wave_last = r0 + wv * 32 < rows ? static_cast<int32_t>(w1 / G) + before : -1;

    int32_t t0 = 0, t1 = blk_last < 0 ? 0 : blk_last / KT + 1;
    if (p.splits > 1) {
        const int32_t part = (t1 + static_cast<int32_t>(p.splits) - 1) / static_cast<int32_t>(p.splits);
        t0 = min(t1, static_cast<int32_t>(blockIdx.y) * part);
        t1 = min(t1, t0 + part);
    }

    // ---- the wave's query rows: B operands --------------------------------------
    using M = std::conditional_t<S::F32, _Float16, T>;          // what the matrix cores take
    const uint32_t head = kvh * G + g;
    const T* qrow = static_cast<const T*>(p.q) + (static_cast<size_t>(q0) + qi) * p.q_stride + head * HD;
    constexpr int QN = HD / 16;
    uint4 qf[S::PLANES][QN];
    float c2 = p.scale_log2;                                    // of the sums: scores in powers of two
    int qpower = 0;
    if constexpr (S::F32) {
        // two f16 at a power of two that brings the row's largest value to 2^13 .. 2^14
        float top = 0.f;
#pragma unroll
        for (int s = 0; s < QN; ++s) {
            float x[8];
            load8(qrow + 16 * s + 8 * h, x);
#pragma unroll
            for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(x[j]));
        }
        top = half_max(top);
        const uint32_t field = (__float_as_uint(top) >> 23) & 0xFFu;
        qpower = field == 255 ? 0 : plane_power(field);
#pragma unroll
        for (int s = 0; s < QN; ++s) {
            float x[8];
            load8(qrow + 16 * s + 8 * h, x);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = __builtin_amdgcn_ldexpf(x[j], qpower);
            split2(x[0], x[1], qf[0][s].x, qf[1][s].x);
            split2(x[2], x[3], qf[0][s].y, qf[1][s].y);
            split2(x[4], x[5], qf[0][s].z, qf[1][s].z);
            split2(x[6], x[7], qf[0][s].w, qf[1][s].w);
        }
    } else {
#pragma unroll
        for (int s = 0; s < QN; ++s) qf[0][s] = load_u4(reinterpret_cast<const uint8_t*>(qrow) + 32 * s + 16 * h);
    }

    // ---- direct loads: K and V tile t into buffer b ----------------------------
    const uint64_t kb = S::F32 ? nkv * RB : p.k_stride * sizeof(M), vb = S::F32 ? nkv * RB : p.v_stride * sizeof(M);
    const uint64_t plane = S::F32 ? static_cast<uint64_t>(p.k_rows) * kb : 0;
    const uint8_t* kbase = (S::F32 ? reinterpret_cast<const uint8_t*>(p.planes) : static_cast<const uint8_t*>(p.k)) +
                           static_cast<uint64_t>(k0) * kb + kvh * RB;
    const uint8_t* vbase = (S::F32 ? reinterpret_cast<const uint8_t*>(p.planes) + 2 * plane
                                   : static_cast<const uint8_t*>(p.v)) +
                           static_cast<uint64_t>(k0) * vb + kvh * RB;
    uint8_t* mine = smem + kg * S::LDS;
    const uint32_t lds0 = static_cast<uint32_t>(
        reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)mine));
    constexpr int NI = S::TILE / 1024 / RW;
    uint32_t koff[NI], voff[NI];                                // of a whole tile, from its first key
#pragma unroll
    for (int u = 0; u < NI; ++u) {
        const int at = (wv * NI + u) * 1024 + lane * 16, row = at / RB, c = at % RB / 16;
        koff[u] = row * static_cast<uint32_t>(kb) + 16 * (c ^ S::kswz(row));
        voff[u] = row * static_cast<uint32_t>(vb) + 16 * (c ^ S::vswz(row));
    }
    auto issue = [&](int32_t t, int b) {
        const uint8_t* kt = kbase + static_cast<uint64_t>(t) * KT * kb;
        const uint8_t* vt = vbase + static_cast<uint64_t>(t) * KT * vb;
        const uint32_t to = lds0 + b * S::BUF + wv * NI * 1024;
        const int32_t last = nk - 1 - t * KT;
#pragma unroll
        for (int pl = 0; pl < S::PLANES; ++pl) {
            const uint32_t kto = to + pl * S::TILE, vto = to + (S::PLANES + pl) * S::TILE;
            if (last >= KT - 1) {
#pragma unroll
                for (int u = 0; u < NI; ++u) {
                    load_to_lds(kt + pl * plane, koff[u], kto + u * 1024);
                    load_to_lds(vt + pl * plane, voff[u], vto + u * 1024);
                }
            } else {
                // keys past the end: the last one again (masked)
#pragma unroll
                for (int u = 0; u < NI; ++u) {
                    const int at = (wv * NI + u) * 1024 + lane * 16, row = at / RB, c = at % RB / 16;
                    const uint32_t src = static_cast<uint32_t>(min(row, last));
                    load_to_lds(kt + pl * plane, src * static_cast<uint32_t>(kb) + 16 * (c ^ S::kswz(row)), kto + u * 1024);
                    load_to_lds(vt + pl * plane, src * static_cast<uint32_t>(vb) + 16 * (c ^ S::vswz(row)), vto + u * 1024);
                }
            }
        }
    };

    f32x16_t acc[ND];
#pragma unroll
    for (int t = 0; t < ND; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[t][i] = 0.f;
    float mx = -INFINITY, sum = 0.f;                            // mx in powers of two
    int vpower = NO_POWER;                                      // f32: acc holds the sum times 2^(PLIFT + vpower)
    const int2* powers = S::F32 ? p.powers + static_cast<size_t>(kvh) * p.plane_tiles + seq.ktile : nullptr;

    // K operands requested ahead, and whether those of V are, as far as registers go
    constexpr int SA = S::F32 ? 2 : 4;
    constexpr bool VAHEAD = !S::F32 || HD < 128;
    // The sums are rescaled when a row's maximum has grown by more than 2^SLACK, not whenever it has: with 32 rows a
    // wave one of them has a new maximum in every other tile.  Weights may then be up to 2^SLACK, which 16-bit types
    // hold as well as 1, and f32 at 2^PLIFT as f16 halves.  f16: weights 2^LIFT times as large, sum and acc with them,
    // or those under 2^-14 would be subnormal and lose bits (thousands of them may make up the sum).
    constexpr float SLACK = S::F32 ? 1.f : 8.f, LIFT = __is_same(T, _Float16) ? 7.f : 0.f;
    constexpr int PLIFT = 14;
    auto tile_step = [&](int32_t t, int b, int2 pw) {
        const uint8_t* kl = mine + b * S::BUF;
        const uint8_t* vl = kl + S::PLANES * S::TILE;
        // ---- S^T = K Q^T ----
        f32x16_t s[NSUB];
#pragma unroll
        for (int u = 0; u < NSUB; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[u][i] = 0.f;
        auto kop = [&](int i, int pl) {
            const int ks = i / NSUB, u = i % NSUB;
            return *reinterpret_cast<const uint4*>(kl + pl * S::TILE + (u * 32 + col) * RB + 16 * ((2 * ks + h) ^ S::kswz(col)));
        };
        // place c of a 16-lane group of a transposing read names row c / 4 and dims 4 (c % 4) .. of 16;
        // the lane receives the rows' values of dim c
        const int c = lane & 15;
        auto vop = [&](int ks, int d, int pl) {
            return read_rows8(vl + pl * S::TILE + (16 * ks + 4 * h + (c >> 2)) * RB + 16 * ((4 * d) ^ S::vswz(c >> 2)) +
                              32 * ((lane >> 4) & 1) + 8 * (c & 3), RB);
        };
        uint4 va[2][ND][S::PLANES];
        constexpr int NK = QN * NSUB;
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            const int ks = i / NSUB, u = i % NSUB;
            const uint4 a = kop(i, 0);
            s[u] = mma16<M>(a, qf[0][ks], s[u]);
            if constexpr (S::F32) {
                s[u] = mma16<M>(a, qf[1][ks], s[u]);
                s[u] = mma16<M>(kop(i, 1), qf[0][ks], s[u]);
            }
        }
        auto ahead = [&](int ks) {
            if constexpr (VAHEAD)
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int pl = 0; pl < S::PLANES; ++pl) va[ks & 1][d][pl] = vop(ks, d, pl);
        };
        ahead(0);
        // the order: SA operands, then one for each that the products have taken, then the first of V
        // (0x100 LDS reads, 0x8 MFMA, 0x402 VALU with the transcendentals)
        __builtin_amdgcn_sched_group_barrier(0x100, SA * S::PLANES, 0);
#pragma unroll
        for (int i = 0; i < NK - SA; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x8, S::F32 ? 3 : 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, S::PLANES, 0);
        }
#pragma unroll
        for (int i = 0; i < SA; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x8, S::F32 ? 3 : 1, 0);
            if (VAHEAD) __builtin_amdgcn_sched_group_barrier(0x100, 2 * ND * S::PLANES / SA, 0);
        }
        float sc = c2;
        if constexpr (S::F32) {
            // (never 0: a hidden key's -inf stays one)
            sc = fmaxf(__builtin_amdgcn_ldexpf(c2, -qpower - pw.x), 0x1p-126f);
        }
        // ---- the causal mask: keys t KT + 32 u + 8 (i / 4) + 4 h + i % 4 ----
        if (t * KT + KT - 1 > wave_first) {
            asm volatile("" : "+v"(s[0]));      // (a branch, not selects in every tile)
            const int32_t room = limit - t * KT - 4 * h;
#pragma unroll
            for (int u = 0; u < NSUB; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    if (32 * u + 8 * (i / 4) + i % 4 > room) s[u][i] = -INFINITY;
                }
        }
        // ---- running maximum and sum ----
        float mt = s[0][0];
#pragma unroll
        for (int u = 0; u < NSUB; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) mt = fmaxf(mt, s[u][i]);
        mt = half_max(mt) * sc;
        if (__ballot(mt > mx + SLACK) || (S::F32 && pw.y < vpower)) {
            const float mn = fmaxf(mx, mt);
            float f = mx > -INFINITY ? __builtin_amdgcn_exp2f(mx - mn) : 0.f;
            sum *= f;
            if constexpr (S::F32) {
                const int vp = min(vpower, pw.y);
                f = __builtin_amdgcn_ldexpf(f, vp - vpower);
                vpower = vp;
            }
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[d][i] *= f;
            mx = mn;
        }
        const float mc = (mx > -INFINITY ? mx : 0.f) - LIFT;    // (no key yet: every weight 0)
        const float pf = S::F32 ? __builtin_amdgcn_ldexpf(1.f, PLIFT + vpower - pw.y) : 1.f;
        // ---- weights of 16 keys, and O^T += V^T P^T of the 16 before ----
        uint4 pb[2], pl[2];
        auto weights = [&](int ks) {
            f32x16_t& sv = s[ks / 2];
            const int o = (ks % 2) * 8;
#pragma unroll
            for (int i = o; i < o + 8; ++i) {
                sv[i] = __builtin_amdgcn_exp2f(fmaf(sv[i], sc, -mc));
                if constexpr (S::F32) {
                    sum += sv[i];
                    sv[i] *= pf;
                }
            }
            uint4& w = pb[ks & 1];
            if constexpr (S::F32) {
                uint4& l = pl[ks & 1];
                split2(sv[o + 0], sv[o + 1], w.x, l.x);
                split2(sv[o + 2], sv[o + 3], w.y, l.y);
                split2(sv[o + 4], sv[o + 5], w.z, l.z);
                split2(sv[o + 6], sv[o + 7], w.w, l.w);
            } else {
                w = make_uint4(pack2<T>(sv[o + 0], sv[o + 1]), pack2<T>(sv[o + 2], sv[o + 3]),
                               pack2<T>(sv[o + 4], sv[o + 5]), pack2<T>(sv[o + 6], sv[o + 7]));
                sum = add2<T>(w.x, add2<T>(w.y, add2<T>(w.z, add2<T>(w.w, sum))));
            }
        };
        weights(0);
        if constexpr (VAHEAD) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int ks = 0; ks < KT / 16; ++ks) {
            if (ks + 1 < KT / 16) {
                ahead(ks + 1);
                weights(ks + 1);
            }
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                const uint4 a = VAHEAD ? va[ks & 1][d][0] : vop(ks, d, 0);
                if constexpr (S::F32) {
                    acc[d] = mma16<M>(a, pl[ks & 1], acc[d]);
                    acc[d] = mma16<M>(VAHEAD ? va[ks & 1][d][S::PLANES - 1] : vop(ks, d, 1), pb[ks & 1], acc[d]);
                }
                acc[d] = mma16<M>(a, pb[ks & 1], acc[d]);
            }
            if constexpr (VAHEAD) {
                if (ks + 1 < KT / 16) {
                    __builtin_amdgcn_sched_group_barrier(0x100, 2 * ND * S::PLANES, 0);
#pragma unroll
                    for (int d = 0; d < ND * (S::F32 ? 3 : 1); ++d) {
                        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x402, 6, 0);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };

    // group kg takes tiles t0 + kg, t0 + kg + KG, ..
    int2 pw = make_int2(0, 0);                                  // of the tile on its way
    auto fetch = [&](int32_t t, int b) {
        issue(t, b);
        if constexpr (S::F32) pw = powers[t];
    };
    if (t0 + kg < t1) fetch(t0 + kg, 0);
    // The query loads end here: the compiler, which does not count the direct loads, would
    // otherwise wait for them at their use in the loop, and so for the next tile on its way.
#pragma unroll
    for (int s = 0; s < S::PLANES * QN; ++s) {
        uint4& w = qf[s / QN][s % QN];
        asm volatile("" : "+v"(w.x), "+v"(w.y), "+v"(w.z), "+v"(w.w));
    }
    int b = 0;
    for (int32_t tt = t0; tt < t1; tt += KG, b ^= 1) {
        const int32_t t = tt + kg;
        // this wave's part of tile t has arrived and its reads of the other buffer are done; after
        // the barrier so are every wave's
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" : "+v"(pw.x), "+v"(pw.y)::"memory");    // (a load of the compiler's, as above)
        const int2 at = pw;
        if (t + KG < t1) fetch(t + KG, b ^ 1);
        if (t * KT <= min(wave_last, t1 * KT - 1)) tile_step(t, b, at);
    }
    sum = half_sum(sum);
    if constexpr (S::F32) {
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[d][i] = __builtin_amdgcn_ldexpf(acc[d][i], -PLIFT - vpower);
    }

    // ---- the second key group's part joins the first's, lane by lane ---------------
    if constexpr (KG == 2) {
        float* other = reinterpret_cast<float*>(smem) + wv * (ND * 16 + 2) * WAVE + lane;
        __syncthreads();                                        // (every tile is read)
        if (kg == 1) {
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) other[(d * 16 + i) * WAVE] = acc[d][i];
            other[ND * 16 * WAVE] = mx;
            other[(ND * 16 + 1) * WAVE] = sum;
        }
        __syncthreads();
        if (kg == 1) return;
        const float m1 = other[ND * 16 * WAVE], mn = fmaxf(mx, m1), m0 = mn > -INFINITY ? mn : 0.f;
        const float f0 = __builtin_amdgcn_exp2f(mx - m0), f1 = __builtin_amdgcn_exp2f(m1 - m0);
        sum = sum * f0 + other[(ND * 16 + 1) * WAVE] * f1;
        mx = mn;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[d][i] = acc[d][i] * f0 + other[(d * 16 + i) * WAVE] * f1;
    }

    // ---- the result -----------------------------------------------------------
    if (!live) return;
    const size_t row_out = static_cast<size_t>(q0) + qi;
    if (p.splits == 1) {
        const float inv = sum == 0.f ? 0.f : 1.0f / sum;
        T* out = static_cast<T*>(p.out) + row_out * p.out_stride + head * HD;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x0 = acc[d][4 * i] * inv, x1 = acc[d][4 * i + 1] * inv, x2 = acc[d][4 * i + 2] * inv,
                            x3 = acc[d][4 * i + 3] * inv;
                T* o = out + 32 * d + 8 * i + 4 * h;
                if constexpr (S::F32) *reinterpret_cast<float4*>(o) = make_float4(x0, x1, x2, x3);
                else *reinterpret_cast<uint2*>(o) = make_uint2(pack2<T>(x0, x1), pack2<T>(x2, x3));
            }
    } else {
        const size_t nrow = static_cast<size_t>(p.q_rows) * nkv * G;
        const size_t at = (row_out * nkv * G + head) * p.splits + blockIdx.y;
        if (h == 0) {
            p.part[2 * at] = mx;
            p.part[2 * at + 1] = sum;
        }
        if (sum == 0.f) return;                                  // (the join reads no such part)
        float* out = p.part + part_acc_at(nrow, p.splits) + at * HD;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<float4*>(out + 32 * d + 8 * i + 4 * h) =
                    make_float4(acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]);
    }
}

// one wave per (query row, head) of the sequences
template <int HD, typename T>
__global__ __launch_bounds__(JOIN_WAVES * WAVE)
void k_prompt_join(PromptAttn p)
{
    const int lane = threadIdx.x & 63;
    const uint32_t heads = p.num_kv_heads * p.group;
    const uint32_t w = blockIdx.x * JOIN_WAVES + (threadIdx.x >> 6), row = w / heads;
    if (row >= p.q_rows) return;
    // (rows outside every sequence, or of one whose offsets are wrong, have no parts)
    bool found = false;
    for (uint32_t i = 0; i < p.n_seqs && !found; i += WAVE) {
        const PromptLane l = load_seq(p, i, lane);
        found = __ballot(l.ok && l.a <= static_cast<int32_t>(row) && static_cast<int32_t>(row) < l.z) != 0;
    }
    if (!found) return;
    const size_t nrow = static_cast<size_t>(p.q_rows) * heads, at = static_cast<size_t>(w) * p.splits;
    float o[HD / WAVE];
    join_parts<HD>(p.part + 2 * at, p.part + part_acc_at(nrow, p.splits) + at * HD, p.splits, 1, lane, o);
    store_row<HD>(static_cast<T*>(p.out) + row * p.out_stride + (w % heads) * HD, o, lane);
}

// Which form, by the blocks that a call gives and the key tiles of its longest sequence (8 query heads a KV
// head, 4 KV heads, head_dim 128, bf16; us of the kernel, and of the join where there is one):
//   2 x 2 waves (64 rows, two key groups: one block a CU, half the chain of tiles) while 64-row blocks leave
//     CUs idle: 512 tokens 11.2 against 15.0 (4 x 2) and 15.1 (4 x 1);
//   4 x 2 (128 rows) up to two such blocks a CU: 1024 tokens 23.3 / 24.8 (4 x 1) / 25.2 (2 x 2), 2048 50.6 / 53.0 /
//     71.8, unless there are few tiles to share out;
//   4 x 1 beyond (two blocks a CU, nothing to merge): 4096 tokens 154 / 161 (4 x 2) / 234 (2 x 2), 64 sequences of
//     64 23 / 39 / 49.
// Keys are split over blocks (each part eight tiles or more) until every CU has one: 64 tokens behind 8000 take
// 89 in one part of 2 x 2 and 19 + 4 in eight; over long parts 4 x 2 is ahead again, in eight or fewer (256
// tokens behind 4000: 28.5 + 6.8 in four against 33.6 + 6.9 in two of 2 x 2; 128 behind 16000 43 against 55, but 64
// behind 16000 41 in sixteen against 30 in eight of 2 x 2).  f32 (tiles of 32) by the same rule: 512 tokens 22.7
// against 27.8 (4 x 2), 24.3 + 4.5 (4 x 1 in two parts); 1024 48.8 / 59.5 (4 x 1); 2048 112 / 130 / 156 (2 x 2).
void prompt_plan(PromptAttn& a, uint32_t head_dim, uint32_t type, uint32_t max_k)
{
    constexpr uint64_t CUS = 256;
    const bool f32 = type == SMOE_TYPE_F32, wide = head_dim == 256;
    const uint32_t kt = f32 || wide ? 32 : 64, keys = max_k / kt + (max_k % kt != 0);
    // full tiles alone: a part-filled one of each sequence may not exist
    const uint64_t rows = static_cast<uint64_t>(a.q_rows) * a.group;
    const uint64_t b64 = (rows + 63) / 64 * a.num_kv_heads, b128 = (rows + 127) / 128 * a.num_kv_heads;
    auto parts = [&](uint64_t blocks) {
        return static_cast<uint32_t>(std::max<uint64_t>(
            1, std::min<uint64_t>({CUS / std::max<uint64_t>(blocks, 1), JOIN_MAX, keys / 8})));
    };
    // (LDS and registers of a CU: head_dim 256 has room for one group of four waves, or in 16 bits two of two)
    if (!(f32 && wide) && b64 <= CUS && (wide || keys <= 24 * parts(b64) || parts(b64) >= 8)) {
        a.row_waves = 2;
        a.key_groups = 2;
        a.splits = parts(b64);
    } else {
        a.row_waves = 4;
        a.key_groups = !wide && keys >= 4 && (b128 <= CUS || (b128 <= 2 * CUS && keys >= 8)) ? 2 : 1;
        a.splits = parts(b128);
    }
    a.tiles = static_cast<uint32_t>(rows / (32 * a.row_waves)) + a.n_seqs;
    a.plane_tiles = f32 ? a.k_rows / PLANE_KEYS + std::min(a.n_seqs, a.k_rows) : 0;
}

// scratch: the f16 planes of f32 rows, their powers, then the parts of split keys
static size_t plane_bytes(const PromptAttn& a, uint32_t head_dim)
{
    return (static_cast<size_t>(a.k_rows) * a.num_kv_heads * head_dim * 8 + 15) & ~size_t(15);
}
static size_t power_bytes(const PromptAttn& a)
{
    return (static_cast<size_t>(a.num_kv_heads) * a.plane_tiles * sizeof(int2) + 15) & ~size_t(15);
}
size_t prompt_scratch_bytes(const PromptAttn& a, uint32_t head_dim)
{
    size_t n = 0;
    if (a.plane_tiles) n += plane_bytes(a, head_dim) + power_bytes(a);
    if (a.splits > 1) n += part_floats(static_cast<size_t>(a.q_rows) * a.num_kv_heads * a.group, a.splits, head_dim) * sizeof(float);
    return n;
}
void prompt_scratch(PromptAttn& a, uint32_t head_dim, void* scratch)
{
    uint8_t* p = static_cast<uint8_t*>(scratch);
    if (a.plane_tiles) {
        a.planes = reinterpret_cast<uint16_t*>(p);
        a.powers = reinterpret_cast<int2*>(p + plane_bytes(a, head_dim));
        p += plane_bytes(a, head_dim) + power_bytes(a);
    }
    a.part = reinterpret_cast<float*>(p);
}

template <int HD, typename T, int RW, int KG>
static hipError_t launch_prompt(const PromptAttn& a, dim3 grid, hipStream_t s)
{
    constexpr uint32_t lds = KG * PromptShape<HD, T>::LDS;
    static_assert(lds <= 160 * 1024, "LDS of a CU");
    if constexpr (lds > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(k_attn_prompt<HD, T, RW, KG>),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return e;
    }
    launch_kernel_lds(k_attn_prompt<HD, T, RW, KG>, grid, dim3(RW * KG * WAVE), lds, s, a);
    return hipGetLastError();
}

hipError_t launch_attention_prompt(const PromptAttn& a, uint32_t head_dim, uint32_t type, hipStream_t s)
{
    return with_type_and_head(type, head_dim, [&](auto t, auto hd) {
        constexpr int HD = decltype(hd)::value;
        using T = decltype(t);
        // every XCD has as many blocks of a tile row where KV heads share or split XCDs
        const uint32_t nkv = a.num_kv_heads;
        const uint32_t per = 8 % nkv == 0 ? 8 / nkv : 1;
        const dim3 grid((a.tiles + per - 1) / per * per * nkv, a.splits);
        hipError_t e;
        if (a.plane_tiles)
            launch_kernel(k_prompt_planes<HD>, dim3(a.plane_tiles, nkv), dim3(256), s, a);
        if (a.key_groups == 1) {
            e = launch_prompt<HD, T, 4, 1>(a, grid, s);
        } else if (a.row_waves == 2) {
            if constexpr (2 * PromptShape<HD, T>::LDS <= 160 * 1024) e = launch_prompt<HD, T, 2, 2>(a, grid, s);
            else e = hipErrorInvalidValue;
        } else {
            if constexpr (PromptShape<HD, T>::WAVES_PER_SIMD == 2) e = launch_prompt<HD, T, 4, 2>(a, grid, s);
            else e = hipErrorInvalidValue;
        }
        if (e != hipSuccess || a.splits == 1) return e;
        const uint32_t waves = a.q_rows * nkv * a.group;
        launch_kernel(k_prompt_join<HD, T>, dim3((waves + JOIN_WAVES - 1) / JOIN_WAVES), dim3(JOIN_WAVES * WAVE), s, a);
        return hipGetLastError();
    });
}

}  // namespace smoe
