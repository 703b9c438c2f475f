// attn_common.hpp -- device helpers of the row, prompt and 4-bit-cache attention kernels.
#pragma once

#include <type_traits>

#include "attention.hpp"
#include "device_common.hpp"
#include "smoe_hip.h"

namespace smoe {

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4v_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));

// two floats rounded to nearest even, in one word (low half first)
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b)
{
    typedef T t2 __attribute__((ext_vector_type(2)));
    const f32x2_t v = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, t2));
}
template <typename T>
__device__ __forceinline__ void unpack2(uint32_t w, float& a, float& b)
{
    typedef T t2 __attribute__((ext_vector_type(2)));
    const f32x2_t v = __builtin_convertvector(__builtin_bit_cast(t2, w), f32x2_t);
    a = v.x;
    b = v.y;
}

// 8 consecutive elements at p (16-byte aligned)
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8])
{
    if constexpr (sizeof(T) == 4) {
        const float4 a = load_f4(p), b = load_f4(p + 4);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
        const uint4 w = load_u4(p);
        unpack2<T>(w.x, x[0], x[1]);
        unpack2<T>(w.y, x[2], x[3]);
        unpack2<T>(w.z, x[4], x[5]);
        unpack2<T>(w.w, x[6], x[7]);
    }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8])
{
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        *reinterpret_cast<uint4*>(p) = make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]),
                                                  pack2<T>(x[6], x[7]));
    }
}

// x = hi + lo in f16, both rounded to nearest: off by 2^-24 of x at most where lo is a normal number
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo)
{
    hi = pack2<_Float16>(a, b);
    const f16x2_t hv = __builtin_bit_cast(f16x2_t, hi);
    lo = pack2<_Float16>(a - static_cast<float>(hv.x), b - static_cast<float>(hv.y));
}

// maximum / sum of the values of lanes l and l ^ 32
__device__ __forceinline__ float half_max(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// inclusive sum over the lanes up to this one
__device__ __forceinline__ uint32_t wave_scan(uint32_t v)
{
    v += dpp_u32<0x111>(0u, v);                 // row_shr 1, 2, 4, 8
    v += dpp_u32<0x112>(0u, v);
    v += dpp_u32<0x114>(0u, v);
    v += dpp_u32<0x118>(0u, v);
    v += dpp_u32<DPP_ROW_BCAST15, 0xA>(0u, v);
    v += dpp_u32<DPP_ROW_BCAST31, 0xC>(0u, v);
    return v;
}

// any lane of a block that finds a bad index says so
__device__ __forceinline__ void flag_range(uint32_t* err)
{
    atomicOr(err, ERR_ATTN_RANGE);
}

// The partial results of one output row, in `splits` parts: out = sum_s f_s o_s /
// sum_s f_s l_s with f_s = 2^(m_s - max m).  Parts without a key (l = 0) hold no o_s.
// One wave per output row: reads its parts, `step` parts apart, and leaves the joined row
// in o, lane l's dims at l * HD / 64.  A pass's loads, of 16 parts, are in flight at once.
template <int HD>
__device__ __forceinline__ void join_parts(const float* ml, const float* acc, uint32_t splits, uint32_t step, int lane,
                                           float (&o)[HD / WAVE])
{
    constexpr int DV = HD / WAVE;
    constexpr uint32_t PASS = 16;
    const bool live = static_cast<uint32_t>(lane) < splits;
    const size_t mine = static_cast<size_t>(lane) * step;
    const float m = live ? ml[2 * mine] : -INFINITY, l = live ? ml[2 * mine + 1] : 0.f;
    const bool used = l != 0.f;                          // (a NaN sum is used)
    const float top = wave_max(used ? m : -INFINITY);
    const float f = used ? exp2f(m - (top > -INFINITY ? top : 0.f)) : 0.f;
    const float sum = wave_sum(used ? f * l : 0.f);
    const uint32_t keep = used ? 0xFFFFFFFFu : 0u;
#pragma unroll
    for (int j = 0; j < DV; ++j) o[j] = 0.f;
    for (uint32_t s0 = 0; s0 < splits; s0 += PASS) {
        float a[PASS][DV], t[DV];
#pragma unroll
        for (uint32_t u = 0; u < PASS; ++u) {
            // (loaded in any case, the last part's again past the end: a branch would keep the loads apart)
            const float* row = acc + static_cast<size_t>(min(s0 + u, splits - 1)) * step * HD + lane * DV;
#pragma unroll
            for (int j = 0; j < DV; ++j) a[u][j] = row[j];
        }
#pragma unroll
        for (int j = 0; j < DV; ++j) t[j] = 0.f;
#pragma unroll
        for (uint32_t u = 0; u < PASS; ++u) {
            // (a part without a key may hold anything, so its bits are cleared: again no branch)
            const float fs = readlane_f32(f, (s0 + u) & 63);
            const uint32_t bits = readlane_u32(keep, (s0 + u) & 63);
#pragma unroll
            for (int j = 0; j < DV; ++j) t[j] = fmaf(fs, __uint_as_float(__float_as_uint(a[u][j]) & bits), t[j]);
        }
#pragma unroll
        for (int j = 0; j < DV; ++j) o[j] += t[j];
    }
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
    for (int j = 0; j < DV; ++j) o[j] *= inv;
}
// the most parts join_parts takes
constexpr uint32_t JOIN_MAX = 64;

template <int HD, typename T>
__device__ __forceinline__ void store_row(T* p, const float (&o)[HD / WAVE], int lane)
{
    constexpr int DV = HD / WAVE;
#pragma unroll
    for (int j = 0; j < DV; ++j) p[lane * DV + j] = static_cast<T>(o[j]);
}

// calls f with a value of the element type and the head size as a constant
template <int HD, typename F>
inline hipError_t with_type(uint32_t type, F&& f)
{
    using hd = std::integral_constant<int, HD>;
    switch (type) {
        case SMOE_TYPE_F32: return f(float{}, hd{});
        case SMOE_TYPE_F16: return f(_Float16{}, hd{});
        case SMOE_TYPE_BF16: return f(__bf16{}, hd{});
    }
    return hipErrorInvalidValue;
}
template <typename F>
inline hipError_t with_type_and_head(uint32_t type, uint32_t head_dim, F&& f)
{
    switch (head_dim) {
        case 64: return with_type<64>(type, f);
        case 128: return with_type<128>(type, f);
        case 256: return with_type<256>(type, f);
    }
    return hipErrorInvalidValue;
}

}  // namespace smoe
