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
// 8 consecutive elements i .. i + 7.  Rows may start anywhere: gfx950 takes wide accesses on any element's address (a row of 1001 elements
// costs what one of 1000 does), so the vector types only promise the element's alignment.
typedef unsigned int q8_u32x4_e2 __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned int q8_u32x4_e4 __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned int q8_u32x2_e1 __attribute__((ext_vector_type(2), aligned(1)));
typedef unsigned int q8_u32x2_e2 __attribute__((ext_vector_type(2), aligned(2)));
template <int DT> struct El8 { q8_u32x4 w[DT == KP_F32 ? 2 : 1]; };   // as loaded
template <int DT> __device__ __forceinline__ El8<DT> el_raw8(const void* p, long long i) {
    El8<DT> r;
    if constexpr (DT == KP_F32) {
        r.w[0] = *reinterpret_cast<const q8_u32x4_e4*>((const float*)p + i);
        r.w[1] = *reinterpret_cast<const q8_u32x4_e4*>((const float*)p + i + 4);
    } else r.w[0] = *reinterpret_cast<const q8_u32x4_e2*>((const uint16_t*)p + i);
    return r;
}
// the first n of them (n <= 0: none), the others zero
template <int DT> __device__ __forceinline__ El8<DT> el_raw8_part(const void* p, long long i, int n) {
    El8<DT> r;
    if constexpr (DT == KP_F32) {
#pragma unroll
        for (int k = 0; k < 8; ++k) r.w[k >> 2][k & 3] = k < n ? ((const uint32_t*)p)[i + k] : 0u;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t lo = 2 * k < n ? ((const uint16_t*)p)[i + 2 * k] : 0u, hi = 2 * k + 1 < n ? ((const uint16_t*)p)[i + 2 * k + 1] : 0u;
            r.w[0][k] = lo | hi << 16;
        }
    }
    return r;
}
template <int DT> __device__ __forceinline__ El8<DT> el_raw8_any(const void* p, long long i, int n) {
    if (n >= 8) return el_raw8<DT>(p, i);
    if (n > 0) return el_raw8_part<DT>(p, i, n);
    El8<DT> none;
#pragma unroll
    for (int k = 0; k < (DT == KP_F32 ? 2 : 1); ++k) none.w[k] = q8_u32x4{0u, 0u, 0u, 0u};
    return none;
}
template <int DT> __device__ __forceinline__ void el_unpack8(const El8<DT>& r, float (&v)[8]) {
    if constexpr (DT == KP_F32) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = __uint_as_float(r.w[k >> 2][k & 3]);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) el_unpack<DT>(r.w[0][k], v[2 * k], v[2 * k + 1]);
    }
}
template <int DT> __device__ __forceinline__ void el_load8(const void* p, long long i, int n, float (&v)[8]) { el_unpack8<DT>(el_raw8_any<DT>(p, i, n), v); }
template <int DT> __device__ __forceinline__ void el_store8(void* p, long long i, int n, const float (&v)[8]) {
    if (n >= 8) {
        if constexpr (DT == KP_F32) {
            *reinterpret_cast<q8_u32x4_e4*>((float*)p + i) = q8_u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
            *reinterpret_cast<q8_u32x4_e4*>((float*)p + i + 4) = q8_u32x4{__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])};
        } else
            *reinterpret_cast<q8_u32x4_e2*>((uint16_t*)p + i) = q8_u32x4{el_pack<DT>(v[0], v[1]), el_pack<DT>(v[2], v[3]), el_pack<DT>(v[4], v[5]), el_pack<DT>(v[6], v[7])};
    } else if (n > 0) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < n) el_store<DT>(p, i + k, v[k]);
    }
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
// 8 bytes anywhere, the first n of them
__device__ __forceinline__ q8_u32x2 q8_load8(const uint8_t* p, int n) {
    if (n >= 8) return *reinterpret_cast<const q8_u32x2_e1*>(p);
    q8_u32x2 r = {0u, 0u};
    if (n > 0)
#pragma unroll
    for (int k = 0; k < 8; ++k)
        if (k < n) r[k >> 2] |= (uint32_t)p[k] << (8 * (k & 3));
    return r;
}
__device__ __forceinline__ void q8_store8(uint8_t* p, int n, q8_u32x2 q) {
    if (n >= 8) *reinterpret_cast<q8_u32x2_e1*>(p) = q;
    else if (n > 0) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < n) p[k] = (uint8_t)(q[k >> 2] >> (8 * (k & 3)));
    }
}

// ---- maxima over aligned groups of G <= 16 lanes: lane ^ 1, ^ 2, ^ 7, + 8 of a DPP row.  All lanes of the wave are active ------------------
template <int CTRL> __device__ __forceinline__ uint32_t q8_dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
__device__ __forceinline__ uint32_t q8_umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
typedef unsigned short q8_u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t q8_umax16(uint32_t a, uint32_t b) {   // two 16-bit maxima
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(q8_u16x2, a), __builtin_bit_cast(q8_u16x2, b)));
}
template <int G, bool PAIRS> __device__ __forceinline__ uint32_t q8_group_max(uint32_t m) {
    auto mx = [](uint32_t a, uint32_t b) { return PAIRS ? q8_umax16(a, b) : q8_umax(a, b); };
    if constexpr (G >= 2) m = mx(m, q8_dpp<0xB1>(m));
    if constexpr (G >= 4) m = mx(m, q8_dpp<0x4E>(m));
    if constexpr (G >= 8) m = mx(m, q8_dpp<0x141>(m));
    if constexpr (G >= 16) m = mx(m, q8_dpp<0x128>(m));
    return m;
}

// ---- a block from its elements as loaded.  The largest magnitude is taken over the type's own bits as integers (two at a time in 16 bits)
// and the elements are converted by the scaling conversions of gfx950, 2 operations an element in all instead of 7.  Blocks that hold an
// infinity or a not-a-number, or whose scale is the smallest one, take the plain sequence: the maximum over finite elements, a
// multiplication and a conversion.
template <int DT> __device__ __forceinline__ uint32_t q8_raw_mag(uint32_t w) { return w & (DT == KP_F32 ? 0x7fffffffu : 0x7fff7fffu); }
template <int DT> __device__ __forceinline__ uint32_t q8_raw_max(uint32_t a, uint32_t b) { return DT == KP_F32 ? q8_umax(a, b) : q8_umax16(a, b); }
// over lanes l, l ^ 16, l ^ 32, l ^ 48 (all lanes of the wave are active): the row swaps of gfx950 instead of two ways through LDS
template <int DT> __device__ __forceinline__ uint32_t q8_raw_max4(uint32_t m) {
    const auto a = __builtin_amdgcn_permlane16_swap(m, m, false, false);
    m = q8_raw_max<DT>(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(m, m, false, false);
    return q8_raw_max<DT>(b[0], b[1]);
}
template <int DT> __device__ __forceinline__ uint32_t q8_raw_peak(const El8<DT>& r) {
    uint32_t m = q8_raw_mag<DT>(r.w[0][0]);
#pragma unroll
    for (int k = 1; k < (DT == KP_F32 ? 8 : 4); ++k) m = q8_raw_max<DT>(m, q8_raw_mag<DT>(r.w[k >> 2][k & 3]));
    return m;
}
// fp32 bits of a magnitude given in the type's own bits
template <int DT> __device__ __forceinline__ uint32_t q8_raw_bits(uint32_t m) {
    if constexpr (DT == KP_F32) return m;
    else if constexpr (DT == KP_BF16) return m << 16;
    else return __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)m));
}
template <int FMT> __device__ __forceinline__ bool q8_plain(uint32_t bits) {   // not for the scaling conversions
    return bits >= 0x7f800000u || bits - 1u < ((uint32_t)(q8_top<FMT> + 1) << 23);
}
// four bytes of four elements, two words of 16-bit pairs or four fp32 words, divided by `up` = 2^s
template <int DT, int FMT> __device__ __forceinline__ uint32_t q8_scaled4(uint32_t a, uint32_t b, uint32_t c, uint32_t d, float up) {
    typedef short s16x2 __attribute__((ext_vector_type(2)));
    s16x2 r = {0, 0};
    if constexpr (DT == KP_F32) {
        if constexpr (FMT == KP_E4M3) {
            r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, __uint_as_float(a), __uint_as_float(b), up, false);
            r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, __uint_as_float(c), __uint_as_float(d), up, true);
        } else {
            r = __builtin_amdgcn_cvt_scalef32_pk_bf8_f32(r, __uint_as_float(a), __uint_as_float(b), up, false);
            r = __builtin_amdgcn_cvt_scalef32_pk_bf8_f32(r, __uint_as_float(c), __uint_as_float(d), up, true);
        }
    } else if constexpr (DT == KP_BF16) {
        const q8_bf16x2 x = __builtin_bit_cast(q8_bf16x2, a), y = __builtin_bit_cast(q8_bf16x2, b);
        if constexpr (FMT == KP_E4M3) {
            r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, x, up, false);
            r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, y, up, true);
        } else {
            r = __builtin_amdgcn_cvt_scalef32_pk_bf8_bf16(r, x, up, false);
            r = __builtin_amdgcn_cvt_scalef32_pk_bf8_bf16(r, y, up, true);
        }
    } else {
        const q8_f16x2 x = __builtin_bit_cast(q8_f16x2, a), y = __builtin_bit_cast(q8_f16x2, b);
        if constexpr (FMT == KP_E4M3) {
            r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, x, up, false);
            r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, y, up, true);
        } else {
            r = __builtin_amdgcn_cvt_scalef32_pk_bf8_f16(r, x, up, false);
            r = __builtin_amdgcn_cvt_scalef32_pk_bf8_f16(r, y, up, true);
        }
    }
    return __builtin_bit_cast(uint32_t, r);
}
template <int DT, int FMT> __device__ __forceinline__ q8_u32x2 q8_scaled8(const El8<DT>& r, float up) {
    if constexpr (DT == KP_F32)
        return q8_u32x2{q8_scaled4<DT, FMT>(r.w[0][0], r.w[0][1], r.w[0][2], r.w[0][3], up), q8_scaled4<DT, FMT>(r.w[1][0], r.w[1][1], r.w[1][2], r.w[1][3], up)};
    else return q8_u32x2{q8_scaled4<DT, FMT>(r.w[0][0], r.w[0][1], 0u, 0u, up), q8_scaled4<DT, FMT>(r.w[0][2], r.w[0][3], 0u, 0u, up)};
}
// This lane's 8 elements of a block that G lanes hold (G <= 16, a power of two): their bytes, and the block's exponent byte.
template <int DT, int FMT, int G> __device__ __forceinline__ uint32_t q8_pack_block(const El8<DT>& r, q8_u32x2& out) {
    uint32_t m = q8_group_max<G, DT != KP_F32>(q8_raw_peak<DT>(r));
    if constexpr (DT != KP_F32) m = q8_umax(m & 0xffffu, m >> 16);
    uint32_t bits = q8_raw_bits<DT>(m), byte;
    if (__any(q8_plain<FMT>(bits))) {
        float v[8];
        el_unpack8<DT>(r, v);
        byte = q8_scale_byte<FMT>(q8_group_max<G, false>(q8_mag8(v)));
        out = q8_cvt8<FMT>(v, q8_down(byte));
        return byte;
    }
    byte = q8_scale_byte<FMT>(bits);
    out = q8_scaled8<DT, FMT>(r, q8_up(byte));
    return byte;
}

// Sums of `parts` partial rows of `width` floats, in a fixed order, in fp64, rounded once: 16 columns x 64 runs of parts a workgroup of 1024;
// column c goes to out0[c], from `cut` on to out1[c - cut] (either may be NULL).
__global__ __launch_bounds__(1024) void q8_join_k(const float* __restrict__ part, long long parts, long long width, float* __restrict__ out0,
                                                  long long cut, float* __restrict__ out1) {
    __shared__ double red[64][17];
    const int col = threadIdx.x & 15, run = threadIdx.x >> 4;
    const long long c = (long long)blockIdx.x * 16 + col;
    double s = 0.0;
    if (c < width) {
        long long p = run;
        for (; p + 7 * 64 < parts; p += 8 * 64) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = part[(p + u * 64) * width + c];
#pragma unroll
            for (int u = 0; u < 8; ++u) s += (double)v[u];
        }
        float v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = p + u * 64 < parts ? part[(p + u * 64) * width + c] : 0.f;
#pragma unroll
        for (int u = 0; u < 8; ++u) s += (double)v[u];
    }
    red[run][col] = s;
    __syncthreads();
    if (run < 4) {   // four groups of 16 runs, then the groups: lanes run * 16 + col of the first wave
        s = 0.0;
        for (int k = 0; k < 16; ++k) s += red[run * 16 + k][col];
        red[run * 16][col] = s;   // (read by this thread only, above)
    }
    __syncthreads();
    if (run == 0 && c < width) {
        s = (red[0][col] + red[16][col]) + (red[32][col] + red[48][col]);
        if (c < cut) { if (out0) out0[c] = (float)s; }
        else if (out1) out1[c - cut] = (float)s;
    }
}

}  // namespace
