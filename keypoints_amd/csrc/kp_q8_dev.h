// Device helpers of the 8-bit block format (kp_q8.hip, kp_q8_matmul.hip, kp_norm.hip).
//
// A row of elements is cut into blocks of 128 (the last one may be short).  A block stores its elements as e4m3 or e5m2 bytes and ONE
// exponent byte s + 127: element = byte value * 2^s.  s is the smallest whole number >= -127 that brings the block's largest finite
// magnitude to at most the format's largest value 1.75 * 2^TOP, so no finite element saturates; a block of zeros has s = 0.  The scale
// is a power of two for three reasons: x * 2^-s is exact, so the one rounding is the conversion's own (half a step, at most 2^-4 of the
// element for e4m3, 2^-3 for e5m2) and every program that follows the definition gets the same bytes; a byte holds it; and the gfx950
// matrix instructions take exactly such exponent bytes as operands, so a scaled product costs what an unscaled one does.
// Not-a-numbers stay not-a-numbers; infinities stay infinities in e5m2 and become not-a-numbers in e4m3, which has none.
#pragma once
#include "kp_common.h"

namespace {

typedef unsigned int q8_u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int q8_u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 q8_bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 q8_f16x2 __attribute__((ext_vector_type(2)));

constexpr int Q8_BLOCK = 128;
template <int FMT> constexpr int q8_top = FMT == KP_E4M3 ? 8 : 15;

// ---- element access of the three storage types (dtype code as template argument) -------------------------------------------------
template <int DT> constexpr int el_size = DT == KP_F32 ? 4 : 2;
__device__ __forceinline__ float el_bf16(uint32_t w, int hi) { return __uint_as_float(hi ? (w & 0xffff0000u) : (w << 16)); }
template <int DT> __device__ __forceinline__ float el_load(const void* p, long long i) {
    if constexpr (DT == KP_F32) return ((const float*)p)[i];
    else if constexpr (DT == KP_BF16) return __uint_as_float((uint32_t)((const uint16_t*)p)[i] << 16);
    else return (float)((const _Float16*)p)[i];
}
template <int DT> __device__ __forceinline__ void el_store(void* p, long long i, float v) {
    if constexpr (DT == KP_F32) ((float*)p)[i] = v;
    else if constexpr (DT == KP_BF16) ((__bf16*)p)[i] = (__bf16)v;
    else ((_Float16*)p)[i] = (_Float16)v;
}
template <int DT> __device__ __forceinline__ void el_unpack(uint32_t w, float& lo, float& hi) {   // two 16-bit elements
    if constexpr (DT == KP_BF16) {
        lo = el_bf16(w, 0);
        hi = el_bf16(w, 1);
    } else {
        const q8_f16x2 h = __builtin_bit_cast(q8_f16x2, w);
        lo = (float)h[0];
        hi = (float)h[1];
    }
}
template <int DT> __device__ __forceinline__ uint32_t el_pack(float lo, float hi) {
    const kp_f32x2 v = {lo, hi};
    if constexpr (DT == KP_BF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, q8_bf16x2));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, q8_f16x2));
}
// 8 consecutive elements i .. i + 7; the address is a multiple of 16 bytes
template <int DT> __device__ __forceinline__ void el_load8(const void* p, long long i, float (&v)[8]) {
    if constexpr (DT == KP_F32) {
        const float4 a = *reinterpret_cast<const float4*>((const float*)p + i), b = *reinterpret_cast<const float4*>((const float*)p + i + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const q8_u32x4 w = *reinterpret_cast<const q8_u32x4*>((const uint16_t*)p + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) el_unpack<DT>(w[k], v[2 * k], v[2 * k + 1]);
    }
}
template <int DT> __device__ __forceinline__ void el_store8(void* p, long long i, const float (&v)[8]) {
    if constexpr (DT == KP_F32) {
        *reinterpret_cast<float4*>((float*)p + i) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>((float*)p + i + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        const q8_u32x4 w = {el_pack<DT>(v[0], v[1]), el_pack<DT>(v[2], v[3]), el_pack<DT>(v[4], v[5]), el_pack<DT>(v[6], v[7])};
        *reinterpret_cast<q8_u32x4*>((uint16_t*)p + i) = w;
    }
}
// the same with any alignment and only the first `n` elements there (n <= 0: none); the others are zero / not written
template <int DT> __device__ __forceinline__ void el_load8_part(const void* p, long long i, int n, float (&v)[8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = k < n ? el_load<DT>(p, i + k) : 0.f;
}
template <int DT> __device__ __forceinline__ void el_store8_part(void* p, long long i, int n, const float (&v)[8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
        if (k < n) el_store<DT>(p, i + k, v[k]);
}

// ---- the format -------------------------------------------------------------------------------------------------------------------
// magnitude bits of a finite element, 0 for infinities and not-a-numbers: what the block's maximum is taken over (as integers)
__device__ __forceinline__ uint32_t q8_mag(float v) {
    const uint32_t u = __float_as_uint(v) & 0x7fffffffu;
    return u < 0x7f800000u ? u : 0u;
}
__device__ __forceinline__ uint32_t q8_mag8(const float (&v)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) { const uint32_t u = q8_mag(v[k]); m = u > m ? u : m; }
    return m;
}
// exponent byte of a block whose largest finite magnitude has the bits `m`
template <int FMT> __device__ __forceinline__ uint32_t q8_scale_byte(uint32_t m) {
    int b = (int)(m >> 23) - q8_top<FMT> + ((m & 0x7fffffu) > 0x600000u ? 1 : 0);   // (s + 127; 0x600000: mantissa of 1.75)
    b = b < 0 ? 0 : b;
    return m ? (uint32_t)b : 127u;
}
__device__ __forceinline__ float q8_down(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }                   // 2^-s (byte <= 247)
__device__ __forceinline__ float q8_up(uint32_t byte) { return __uint_as_float(byte ? byte << 23 : 0x00400000u); }        // 2^s, 2^-127 subnormal
template <int FMT> __device__ __forceinline__ uint32_t q8_cvt4(float a, float b, float c, float d) {
    uint32_t r;
    if constexpr (FMT == KP_E4M3) {
        r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
        r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
    } else {
        r = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, 0, false);
        r = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, r, true);
    }
    return r;
}
template <int FMT> __device__ __forceinline__ q8_u32x2 q8_cvt8(const float (&v)[8], float down) {
    const q8_u32x2 r = {q8_cvt4<FMT>(v[0] * down, v[1] * down, v[2] * down, v[3] * down),
                        q8_cvt4<FMT>(v[4] * down, v[5] * down, v[6] * down, v[7] * down)};
    return r;
}
template <int FMT> __device__ __forceinline__ void q8_values8(q8_u32x2 q, float up, float (&v)[8]) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        kp_f32x2 lo, hi;
        if constexpr (FMT == KP_E4M3) {
            lo = __builtin_amdgcn_cvt_pk_f32_fp8(q[k], false);
            hi = __builtin_amdgcn_cvt_pk_f32_fp8(q[k], true);
        } else {
            lo = __builtin_amdgcn_cvt_pk_f32_bf8(q[k], false);
            hi = __builtin_amdgcn_cvt_pk_f32_bf8(q[k], true);
        }
        v[4 * k] = lo[0] * up; v[4 * k + 1] = lo[1] * up; v[4 * k + 2] = hi[0] * up; v[4 * k + 3] = hi[1] * up;
    }
}
// 8 bytes with any alignment, the first `n` of them
__device__ __forceinline__ q8_u32x2 q8_load8_part(const uint8_t* p, int n) {
    q8_u32x2 r = {0u, 0u};
#pragma unroll
    for (int k = 0; k < 8; ++k)
        if (k < n) r[k >> 2] |= (uint32_t)p[k] << (8 * (k & 3));
    return r;
}
__device__ __forceinline__ void q8_store8_part(uint8_t* p, int n, q8_u32x2 q) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
        if (k < n) p[k] = (uint8_t)(q[k >> 2] >> (8 * (k & 3)));
}

// ---- reductions over aligned groups of 16 lanes (one DPP row): lane ^ 1, ^ 2, ^ 7, + 8.  All lanes of the wave are active -------------
template <int CTRL> __device__ __forceinline__ uint32_t q8_dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
__device__ __forceinline__ uint32_t q8_umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t q8_max16(uint32_t m) {
    m = q8_umax(m, q8_dpp<0xB1>(m));
    m = q8_umax(m, q8_dpp<0x4E>(m));
    m = q8_umax(m, q8_dpp<0x141>(m));
    return q8_umax(m, q8_dpp<0x128>(m));
}

}  // namespace
