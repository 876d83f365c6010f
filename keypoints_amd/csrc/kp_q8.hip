// The 8-bit block format of kp_q8_dev.h: rows to 8 bits, back, and both ways at once (rows and columns) with the column sums.
// All of it is bound by memory: 2 (4) bytes of input and 1 byte per form an element.
#include "kp_q8_dev.h"

namespace {

constexpr int TPB = 256;

// A group of 16 lanes takes a block: 8 consecutive elements a lane, the block's maximum by DPP.  VEC: the rows start on multiples of 16
// bytes; otherwise element loads.  `padded`: the row's last block is written out to its full 128 bytes with zeros.
template <int DT, int FMT, bool VEC>
__global__ __launch_bounds__(TPB) void q8_pack_k(const void* __restrict__ x, long long ldx, uint8_t* __restrict__ q, long long ldq,
                                                 uint8_t* __restrict__ s, long long lds, unsigned nb, unsigned total, long long cols,
                                                 int padded) {
    const int sub = threadIdx.x & 15;
    const unsigned stride = gridDim.x * (TPB / 16);
    for (unsigned b0 = blockIdx.x * (TPB / 16); b0 < total; b0 += stride) {
        const unsigned b = b0 + (threadIdx.x >> 4);
        const bool live = b < total;
        const unsigned row = live ? b / nb : 0, kb = live ? b - row * nb : 0;
        const long long c = (long long)kb * Q8_BLOCK + sub * 8;
        const int n = !live ? 0 : (cols - c >= 8 ? 8 : (cols > c ? (int)(cols - c) : 0));
        float v[8];
        if (VEC && n == 8) el_load8<DT>(x, row * ldx + c, v);
        else el_load8_part<DT>(x, row * ldx + c, n, v);
        const uint32_t byte = q8_scale_byte<FMT>(q8_max16(q8_mag8(v)));
        if (!live) continue;
        const q8_u32x2 r = q8_cvt8<FMT>(v, q8_down(byte));
        uint8_t* dst = q + row * ldq + c;
        if (padded || (VEC && n == 8)) *reinterpret_cast<q8_u32x2*>(dst) = r;
        else q8_store8_part(dst, n, r);
        if (sub == 0) s[row * lds + kb] = (uint8_t)byte;
    }
}

// A finite element that was rounded up to a power of two past the type's range (2^16 in fp16, 2^128) comes back as the type's largest
// number.  Only blocks whose exponent reaches that far look.
template <int DT, int FMT> __device__ __forceinline__ void q8_unpack8(q8_u32x2 q, uint32_t byte, float (&v)[8]) {
    constexpr int RANGE = DT == KP_F16 ? 16 : 128;
    if ((int)byte - 127 + q8_top<FMT> < RANGE) {
        q8_values8<FMT>(q, q8_up(byte), v);
        return;
    }
    const float largest = DT == KP_F16 ? 65504.f : DT == KP_BF16 ? 0x1.fep127f : 0x1.fffffep127f;
    q8_values8<FMT>(q, q8_up(byte - 4), v);   // a 16th
#pragma unroll
    for (int k = 0; k < 8; ++k)
        v[k] = fabsf(v[k]) >= __uint_as_float((uint32_t)(127 + RANGE - 4) << 23) && fabsf(v[k]) < __builtin_inff() ? copysignf(largest, v[k]) : v[k] * 16.f;
}

template <int DT, int FMT, bool VEC>
__global__ __launch_bounds__(TPB) void q8_unpack_k(const uint8_t* __restrict__ q, long long ldq, const uint8_t* __restrict__ s,
                                                   long long lds, void* __restrict__ y, long long ldy, unsigned nb, unsigned total,
                                                   long long cols) {
    const int sub = threadIdx.x & 15;
    const unsigned stride = gridDim.x * (TPB / 16);
    for (unsigned b = blockIdx.x * (TPB / 16) + (threadIdx.x >> 4); b < total; b += stride) {
        const unsigned row = b / nb, kb = b - row * nb;
        const long long c = (long long)kb * Q8_BLOCK + sub * 8;
        const int n = cols - c >= 8 ? 8 : (cols > c ? (int)(cols - c) : 0);
        if (n == 0) continue;
        const uint32_t byte = s[row * lds + kb];
        float v[8];
        if (VEC && n == 8) {
            q8_unpack8<DT, FMT>(*reinterpret_cast<const q8_u32x2*>(q + row * ldq + c), byte, v);
            el_store8<DT>(y, row * ldy + c, v);
        } else {
            q8_unpack8<DT, FMT>(q8_load8_part(q + row * ldq + c, n), byte, v);
            el_store8_part<DT>(y, row * ldy + c, n, v);
        }
    }
}

// Rows and columns at once, a 128 x 128 tile of x a workgroup: a thread holds 8 rows x 8 columns (rows 8 g .. 8 g + 7 with g = thread / 16,
// columns 8 (thread % 16) ..), so that a row's block is a DPP row of lanes and a column's block the 16 values of g: four in the wave, four
// waves through LDS.  The column form leaves through LDS as 16-byte pieces along the rows.  Tiles at the matrix's edge read zeros beyond
// it, and both forms are written to full 128-byte blocks.  With colsum: the tile's column sums, one fp32 row a tile row (summed in a
// fixed order by q8_colsum_k).
template <int DT, int FMT, bool VEC>
__global__ __launch_bounds__(TPB) void q8_pack_both_k(const void* __restrict__ x, long long ldx, uint8_t* __restrict__ q, long long ldq,
                                                      uint8_t* __restrict__ s, long long lds, uint8_t* __restrict__ qt, long long ldqt,
                                                      uint8_t* __restrict__ st, long long ldst, float* __restrict__ colsum,
                                                      long long rows, long long cols) {
    constexpr int PITCH = 144;                      // bytes of an LDS row of the column form (16 more than a block: spread over the banks)
    __shared__ __attribute__((aligned(16))) uint8_t tile[128 * PITCH];
    __shared__ uint32_t wmax[4][128];
    __shared__ float wsum[4][128];
    const int t = threadIdx.x, cv = t & 15, g = t >> 4, wave = t >> 6;
    const long long c0 = (long long)blockIdx.x * 128 + cv * 8, r0 = (long long)blockIdx.y * 128 + g * 8;
    const int n = cols - c0 >= 8 ? 8 : (cols > c0 ? (int)(cols - c0) : 0);
    float v[8][8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const bool in = r0 + j < rows;
        if (VEC && n == 8 && in) el_load8<DT>(x, (r0 + j) * ldx + c0, v[j]);
        else el_load8_part<DT>(x, (r0 + j) * ldx + c0, in ? n : 0, v[j]);
    }
    if (q) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t byte = q8_scale_byte<FMT>(q8_max16(q8_mag8(v[j])));
            if (r0 + j < rows) {
                *reinterpret_cast<q8_u32x2*>(q + (r0 + j) * ldq + c0) = q8_cvt8<FMT>(v[j], q8_down(byte));
                if (cv == 0) s[(r0 + j) * lds + blockIdx.x] = (uint8_t)byte;
            }
        }
    }
    if (!qt && !colsum) return;
    uint32_t m[8];
    float sum[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        m[k] = 0;
        sum[k] = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            m[k] = q8_umax(m[k], q8_mag(v[j][k]));
            sum[k] += v[j][k];
        }
        m[k] = q8_umax(m[k], (uint32_t)__shfl_xor((int)m[k], 16, 64));
        m[k] = q8_umax(m[k], (uint32_t)__shfl_xor((int)m[k], 32, 64));
        sum[k] += __shfl_xor(sum[k], 16, 64);
        sum[k] += __shfl_xor(sum[k], 32, 64);
    }
    if ((t & 63) < 16) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            wmax[wave][cv * 8 + k] = m[k];
            wsum[wave][cv * 8 + k] = sum[k];
        }
    }
    __syncthreads();
    if (colsum && t < 128 && (long long)blockIdx.x * 128 + t < cols)
        colsum[(long long)blockIdx.y * cols + (long long)blockIdx.x * 128 + t] = (wsum[0][t] + wsum[1][t]) + (wsum[2][t] + wsum[3][t]);
    if (!qt) return;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const int c = cv * 8 + k;
        const uint32_t byte = q8_scale_byte<FMT>(q8_umax(q8_umax(wmax[0][c], wmax[1][c]), q8_umax(wmax[2][c], wmax[3][c])));
        float col[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) col[j] = v[j][k];
        *reinterpret_cast<q8_u32x2*>(tile + c * PITCH + g * 8) = q8_cvt8<FMT>(col, q8_down(byte));
        if (g == 0 && c0 + k < cols) st[(c0 + k) * ldst + blockIdx.y] = (uint8_t)byte;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int id = i * TPB + t, c = id >> 3, piece = (id & 7) * 16;
        const long long col = (long long)blockIdx.x * 128 + c;
        if (col < cols)
            *reinterpret_cast<q8_u32x4*>(qt + col * ldqt + (long long)blockIdx.y * 128 + piece) =
                *reinterpret_cast<const q8_u32x4*>(tile + c * PITCH + piece);
    }
}

// column sums of the tile rows' partial sums, in a fixed order, accumulated in fp64 and rounded once
__global__ __launch_bounds__(TPB) void q8_colsum_k(const float* __restrict__ part, float* __restrict__ out, long long parts, long long cols) {
    __shared__ double red[4][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const long long c = (long long)blockIdx.x * 64 + lane;
    double a = 0.0;
    if (c < cols)
        for (long long p = w; p < parts; p += 4) a += (double)part[p * cols + c];
    red[w][lane] = a;
    __syncthreads();
    if (w == 0 && c < cols) out[c] = (float)((red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]));
}

bool q8_aligned(const void* p, unsigned n) { return ((size_t)p % n) == 0; }
unsigned q8_grid(unsigned total) {
    const unsigned g = cdiv(total, TPB / 16);
    return g < 8192 ? g : 8192;
}

template <int DT, int FMT>
int pack_launch(const void* x, long long ldx, uint8_t* q, long long ldq, uint8_t* s, long long lds, unsigned nb, unsigned total,
                long long cols, int padded, hipStream_t st) {
    const bool vec = q8_aligned(x, 16) && ldx % (16 / el_size<DT>) == 0 && ldq % 8 == 0 && q8_aligned(q, 8);
    if (vec) q8_pack_k<DT, FMT, true><<<q8_grid(total), TPB, 0, st>>>(x, ldx, q, ldq, s, lds, nb, total, cols, padded);
    else q8_pack_k<DT, FMT, false><<<q8_grid(total), TPB, 0, st>>>(x, ldx, q, ldq, s, lds, nb, total, cols, padded);
    return kp_check_launch("q8_pack");
}
template <int DT, int FMT>
int unpack_launch(const uint8_t* q, long long ldq, const uint8_t* s, long long lds, void* y, long long ldy, unsigned nb, unsigned total,
                  long long cols, hipStream_t st) {
    const bool vec = q8_aligned(y, 16) && ldy % (16 / el_size<DT>) == 0 && ldq % 8 == 0 && q8_aligned(q, 8);
    if (vec) q8_unpack_k<DT, FMT, true><<<q8_grid(total), TPB, 0, st>>>(q, ldq, s, lds, y, ldy, nb, total, cols);
    else q8_unpack_k<DT, FMT, false><<<q8_grid(total), TPB, 0, st>>>(q, ldq, s, lds, y, ldy, nb, total, cols);
    return kp_check_launch("q8_unpack");
}
template <int DT, int FMT>
int both_launch(const void* x, long long ldx, uint8_t* q, long long ldq, uint8_t* s, long long lds, uint8_t* qt, long long ldqt,
                uint8_t* stq, long long ldst, float* ws, float* colsum, long long rows, long long cols, hipStream_t st) {
    const bool vec = q8_aligned(x, 16) && ldx % (16 / el_size<DT>) == 0;
    const dim3 grid(cdiv(cols, 128), cdiv(rows, 128));
    float* part = colsum ? ws : nullptr;
    if (vec) q8_pack_both_k<DT, FMT, true><<<grid, TPB, 0, st>>>(x, ldx, q, ldq, s, lds, qt, ldqt, stq, ldst, part, rows, cols);
    else q8_pack_both_k<DT, FMT, false><<<grid, TPB, 0, st>>>(x, ldx, q, ldq, s, lds, qt, ldqt, stq, ldst, part, rows, cols);
    if (colsum) q8_colsum_k<<<cdiv(cols, 64), TPB, 0, st>>>(part, colsum, cdiv(rows, 128), cols);
    return kp_check_launch("q8_pack_both");
}

#define Q8_DISPATCH(FN, ...)                                                                                  \
    (dtype == KP_F32 ? (fmt == KP_E4M3 ? FN<KP_F32, KP_E4M3>(__VA_ARGS__) : FN<KP_F32, KP_E5M2>(__VA_ARGS__)) \
     : dtype == KP_BF16 ? (fmt == KP_E4M3 ? FN<KP_BF16, KP_E4M3>(__VA_ARGS__) : FN<KP_BF16, KP_E5M2>(__VA_ARGS__)) \
                        : (fmt == KP_E4M3 ? FN<KP_F16, KP_E4M3>(__VA_ARGS__) : FN<KP_F16, KP_E5M2>(__VA_ARGS__)))

bool types_ok(int dtype, int fmt) {
    return (dtype == KP_F32 || dtype == KP_BF16 || dtype == KP_F16) && (fmt == KP_E4M3 || fmt == KP_E5M2);
}

}  // namespace

extern "C" {

int kp_q8_pack(const void* x, long long ldx, unsigned char* q, long long ldq, unsigned char* s, long long lds, long long rows,
               long long cols, int dtype, int fmt, void* stream) {
    KP_REQUIRE(types_ok(dtype, fmt), "kp_q8_pack: unknown dtype %d or format %d", dtype, fmt);
    KP_REQUIRE(x && q && s && rows > 0 && cols > 0, "kp_q8_pack: bad args (%lld x %lld)", rows, cols);
    const long long nb = (cols + Q8_BLOCK - 1) / Q8_BLOCK;
    KP_REQUIRE((rows == 1 || (ldx >= cols && lds >= nb)) && (ldq >= nb * Q8_BLOCK || ldq == cols), "kp_q8_pack: row strides %lld, %lld, %lld do not fit %lld columns", ldx, ldq, lds, cols);
    KP_REQUIRE(rows * nb < (1LL << 31), "kp_q8_pack: %lld blocks are more than one call takes", rows * nb);
    const int padded = ldq >= nb * Q8_BLOCK;
    KP_REQUIRE(!padded || (q8_aligned(q, 8) && ldq % 8 == 0), "kp_q8_pack: padded rows must start on multiples of 8 bytes");
    kp_count_bytes((double)rows * cols * ((dtype == KP_F32 ? 4 : 2) + 1));
    return Q8_DISPATCH(pack_launch, x, ldx, q, ldq, s, lds, (unsigned)nb, (unsigned)(rows * nb), cols, padded, (hipStream_t)stream);
}

int kp_q8_unpack(const unsigned char* q, long long ldq, const unsigned char* s, long long lds, void* y, long long ldy, long long rows,
                 long long cols, int dtype, int fmt, void* stream) {
    KP_REQUIRE(types_ok(dtype, fmt), "kp_q8_unpack: unknown dtype %d or format %d", dtype, fmt);
    KP_REQUIRE(q && s && y && rows > 0 && cols > 0, "kp_q8_unpack: bad args (%lld x %lld)", rows, cols);
    const long long nb = (cols + Q8_BLOCK - 1) / Q8_BLOCK;
    KP_REQUIRE(rows == 1 || (ldy >= cols && ldq >= cols && lds >= nb), "kp_q8_unpack: row strides %lld, %lld, %lld do not fit %lld columns", ldq, lds, ldy, cols);
    KP_REQUIRE(rows * nb < (1LL << 31), "kp_q8_unpack: %lld blocks are more than one call takes", rows * nb);
    kp_count_bytes((double)rows * cols * ((dtype == KP_F32 ? 4 : 2) + 1));
    return Q8_DISPATCH(unpack_launch, q, ldq, s, lds, y, ldy, (unsigned)nb, (unsigned)(rows * nb), cols, (hipStream_t)stream);
}

long long kp_q8_pack_both_ws_floats(long long rows, long long cols) { return (long long)cdiv(rows, 128) * cols; }

int kp_q8_pack_both(const void* x, long long ldx, unsigned char* q, long long ldq, unsigned char* s, long long lds, unsigned char* qt,
                    long long ldqt, unsigned char* st, long long ldst, float* ws, float* colsum, long long rows, long long cols, int dtype,
                    int fmt, void* stream) {
    KP_REQUIRE(types_ok(dtype, fmt), "kp_q8_pack_both: unknown dtype %d or format %d", dtype, fmt);
    KP_REQUIRE(x && rows > 0 && cols > 0 && (q || qt || colsum), "kp_q8_pack_both: bad args (%lld x %lld)", rows, cols);
    const long long nb = (cols + Q8_BLOCK - 1) / Q8_BLOCK, nbt = (rows + Q8_BLOCK - 1) / Q8_BLOCK;
    KP_REQUIRE(rows == 1 || ldx >= cols, "kp_q8_pack_both: row stride %lld for %lld columns", ldx, cols);
    KP_REQUIRE(!q || (s && ldq >= nb * Q8_BLOCK && lds >= nb && ldq % 8 == 0 && q8_aligned(q, 8)), "kp_q8_pack_both: row form: strides %lld, %lld for %lld columns", ldq, lds, cols);
    KP_REQUIRE(!qt || (st && ldqt >= nbt * Q8_BLOCK && ldst >= nbt && ldqt % 16 == 0 && q8_aligned(qt, 16)), "kp_q8_pack_both: column form: strides %lld, %lld for %lld rows", ldqt, ldst, rows);
    KP_REQUIRE(!colsum || ws, "kp_q8_pack_both: column sums need a workspace");
    KP_REQUIRE(nbt < 65536 && nb < (1LL << 31), "kp_q8_pack_both: %lld rows are more than one call takes", rows);
    kp_count_bytes((double)rows * cols * ((dtype == KP_F32 ? 4 : 2) + (q ? 1 : 0) + (qt ? 1 : 0)));
    return Q8_DISPATCH(both_launch, x, ldx, q, ldq, s, lds, qt, ldqt, st, ldst, ws, colsum, rows, cols, (hipStream_t)stream);
}

}  // extern "C"
