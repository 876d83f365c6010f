// The 8-bit block format of kp_q8_dev.h: rows to 8 bits, back, and both ways at once (rows and columns) with the column sums.
// All of it is bound by memory: 2 (4) bytes of input and 1 byte per form an element.  Measured in bf16 (a large copy: 5.2 TB/s): 2^27 elements
// in memory order 74 us to 8 bits = 5.4 TB/s (88 where the card's memory was slower) and 64 us back = 6.3 TB/s (the bytes come partly out of
// the last cache, just written); both ways at once 16384 x 2048 31 us (both forms), 16384 x 4096 62 us (both forms and column sums) = 4.3 TB/s.
// More blocks of a thread in flight, loads a turn ahead in no branch and fewer operations an element changed none of these.
#include "kp_q8_dev.h"

namespace {

constexpr int TPB = 256;
typedef q8_u32x2 __attribute__((may_alias)) q8_u32x2_a;   // (LDS is written as pairs of words and read as 16-byte pieces)
typedef q8_u32x4 __attribute__((may_alias)) q8_u32x4_a;

// A group of 16 lanes takes a block: 8 consecutive elements a lane, the block's maximum by DPP; UNROLL blocks of a thread in flight.
// `padded`: the row's last block is written out to its full 128 bytes with zeros.
constexpr int UNROLL = 2;
struct BlockAt { unsigned row, kb; long long c; int n; };   // n: elements of this lane's 8 that the row has
// division of block numbers below 2^31 by the blocks of a row: (b * mul) >> (32 + shift), mul = ceil(2^(32 + shift) / nb) with the shift
// that brings it to 32 bits (exact: the error b * (mul nb - 2^(32 + shift)) / (nb 2^(32 + shift)) stays below 1 / nb); mul = 0: one row
struct RowDiv { unsigned mul, shift; };
RowDiv row_div(unsigned nb, unsigned total) {
    if (nb == total) return RowDiv{0, 0};
    if (nb == 1) return RowDiv{1, 0};
    unsigned l = 1;
    while (l < 31 && (1u << l) < nb) ++l;   // 2^(l-1) < nb <= 2^l
    return RowDiv{(unsigned)(((1ull << (31 + l)) + nb - 1) / nb), l - 1};
}
__device__ __forceinline__ BlockAt block_at(unsigned b, unsigned nb, RowDiv div, unsigned total, long long cols, int sub) {
    BlockAt r;
    r.row = nb == 1 ? b : __umulhi(b, div.mul) >> div.shift;
    if (b >= total) r.row = 0;
    r.kb = b < total ? b - r.row * nb : 0;
    r.c = (long long)r.kb * Q8_BLOCK + sub * 8;
    r.n = b >= total ? 0 : (cols - r.c >= 8 ? 8 : (cols > r.c ? (int)(cols - r.c) : 0));
    return r;
}
template <int DT, int FMT>
__global__ __launch_bounds__(TPB) void q8_pack_k(const void* __restrict__ x, long long ldx, uint8_t* __restrict__ q, long long ldq,
                                                 uint8_t* __restrict__ s, long long lds, unsigned nb, RowDiv div, unsigned total,
                                                 long long cols, int padded) {
    const int sub = threadIdx.x & 15;
    const unsigned per = TPB / 16, stride = gridDim.x * per * UNROLL;
    for (unsigned b0 = blockIdx.x * per * UNROLL; b0 < total; b0 += stride) {
        BlockAt at[UNROLL];
        El8<DT> raw[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            at[u] = block_at(b0 + u * per + (threadIdx.x >> 4), nb, div, total, cols, sub);
            raw[u] = el_raw8_any<DT>(x, at[u].row * ldx + at[u].c, at[u].n);
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            q8_u32x2 out;
            const uint32_t byte = q8_pack_block<DT, FMT, 16>(raw[u], out);
            if (b0 + u * per + (threadIdx.x >> 4) < total) {
                q8_store8(q + at[u].row * ldq + at[u].c, padded ? 8 : at[u].n, out);
                if (sub == 0) s[at[u].row * lds + at[u].kb] = (uint8_t)byte;
            }
        }
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

template <int DT, int FMT>
__global__ __launch_bounds__(TPB) void q8_unpack_k(const uint8_t* __restrict__ q, long long ldq, const uint8_t* __restrict__ s,
                                                   long long lds, void* __restrict__ y, long long ldy, unsigned nb, RowDiv div,
                                                   unsigned total, long long cols) {
    const int sub = threadIdx.x & 15;
    const unsigned per = TPB / 16, stride = gridDim.x * per * UNROLL;
    for (unsigned b0 = blockIdx.x * per * UNROLL; b0 < total; b0 += stride) {
        BlockAt at[UNROLL];
        q8_u32x2 raw[UNROLL];
        uint32_t byte[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            at[u] = block_at(b0 + u * per + (threadIdx.x >> 4), nb, div, total, cols, sub);
            raw[u] = q8_load8(q + at[u].row * ldq + at[u].c, at[u].n);
            byte[u] = s[at[u].row * lds + at[u].kb];
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            float v[8];
            q8_unpack8<DT, FMT>(raw[u], byte[u], v);
            el_store8<DT>(y, at[u].row * ldy + at[u].c, at[u].n, v);
        }
    }
}

// Rows and columns at once, a 128 x 128 tile of x a workgroup: a thread holds 8 rows x 8 columns (rows 8 g .. 8 g + 7 with g = thread / 16,
// columns 8 (thread % 16) ..), so that a row's block is a DPP row of lanes and a column's block the 16 values of g: four in the wave, four
// waves through LDS.  The column form leaves through LDS as 16-byte pieces along the rows (rows of 128 bytes, the piece XOR-swizzled by the
// column's octet: the eight columns that differ in it hit different banks).  Tiles at the matrix's edge read zeros beyond it, and both
// forms are written to full 128-byte blocks.  With colsum: the tile's column sums, one fp32 row a tile row (joined by q8_join_k).
template <int DT, int FMT>
__global__ __launch_bounds__(TPB) void q8_pack_both_k(const void* __restrict__ x, long long ldx, uint8_t* __restrict__ q, long long ldq,
                                                      uint8_t* __restrict__ s, long long lds, uint8_t* __restrict__ qt, long long ldqt,
                                                      uint8_t* __restrict__ st, long long ldst, float* __restrict__ colsum,
                                                      long long rows, long long cols) {
    __shared__ __attribute__((aligned(16))) uint8_t tile[128 * 128];
    __shared__ uint32_t wmax[4][128];
    __shared__ float wsum[4][128];
    const int t = threadIdx.x, cv = t & 15, g = t >> 4, wave = t >> 6;
    const long long c0 = (long long)blockIdx.x * 128 + cv * 8, r0 = (long long)blockIdx.y * 128 + g * 8;
    const int n = cols - c0 >= 8 ? 8 : (cols > c0 ? (int)(cols - c0) : 0);
    constexpr int W = DT == KP_F32 ? 8 : 4, PER = 8 / W;   // words of a thread's 8 columns, columns a word
    El8<DT> v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = el_raw8_any<DT>(x, (r0 + j) * ldx + c0, r0 + j < rows ? n : 0);
    if (q) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            q8_u32x2 out;
            const uint32_t byte = q8_pack_block<DT, FMT, 16>(v[j], out);
            if (r0 + j < rows) {
                *reinterpret_cast<q8_u32x2*>(q + (r0 + j) * ldq + c0) = out;
                if (cv == 0) s[(r0 + j) * lds + blockIdx.x] = (uint8_t)byte;
            }
        }
    }
    if (!qt && !colsum) return;
    if (colsum) {
        float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float f[8];
            el_unpack8<DT>(v[j], f);
#pragma unroll
            for (int k = 0; k < 8; ++k) sum[k] += f[k];
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            sum[k] += __shfl_xor(sum[k], 16, 64);
            sum[k] += __shfl_xor(sum[k], 32, 64);
            if ((t & 63) < 16) wsum[wave][cv * 8 + k] = sum[k];
        }
    }
    // the columns' maxima in the type's own bits, two columns a word in 16 bits
#pragma unroll
    for (int k = 0; k < W; ++k) {
        uint32_t m = q8_raw_mag<DT>(v[0].w[k >> 2][k & 3]);
#pragma unroll
        for (int j = 1; j < 8; ++j) m = q8_raw_max<DT>(m, q8_raw_mag<DT>(v[j].w[k >> 2][k & 3]));
        m = q8_raw_max<DT>(m, (uint32_t)__shfl_xor((int)m, 16, 64));
        m = q8_raw_max<DT>(m, (uint32_t)__shfl_xor((int)m, 32, 64));
        if ((t & 63) < 16) wmax[wave][cv * W + k] = m;
    }
    __syncthreads();
    if (colsum && t < 128 && (long long)blockIdx.x * 128 + t < cols)
        colsum[(long long)blockIdx.y * cols + (long long)blockIdx.x * 128 + t] = (wsum[0][t] + wsum[1][t]) + (wsum[2][t] + wsum[3][t]);
    if (!qt) return;
    uint32_t bits[8];
    bool plain = false;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const int w = cv * W + k / PER;
        const uint32_t m = q8_raw_max<DT>(q8_raw_max<DT>(wmax[0][w], wmax[1][w]), q8_raw_max<DT>(wmax[2][w], wmax[3][w]));
        bits[k] = q8_raw_bits<DT>(DT == KP_F32 ? m : (k & 1 ? m >> 16 : m & 0xffffu));
        plain |= q8_plain<FMT>(bits[k]);
    }
    auto leave = [&](int k, uint32_t byte, q8_u32x2 out) {
        const int c = cv * 8 + k;
        *reinterpret_cast<q8_u32x2_a*>(tile + c * 128 + (((g >> 1) ^ (cv & 7)) << 4) + (g & 1) * 8) = out;
        if (g == 0 && c0 + k < cols) st[(c0 + k) * ldst + blockIdx.y] = (uint8_t)byte;
    };
    if (__any(plain)) {   // every wave holds all 128 columns: one answer for the workgroup
        float f[8][8];
#pragma unroll
        for (int j = 0; j < 8; ++j) el_unpack8<DT>(v[j], f[j]);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) m = q8_umax(m, q8_mag(f[j][k]));
            m = q8_umax(m, (uint32_t)__shfl_xor((int)m, 16, 64));
            m = q8_umax(m, (uint32_t)__shfl_xor((int)m, 32, 64));
            if ((t & 63) < 16) wmax[wave][cv * 8 + k] = m;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int c = cv * 8 + k;
            const uint32_t byte = q8_scale_byte<FMT>(q8_umax(q8_umax(wmax[0][c], wmax[1][c]), q8_umax(wmax[2][c], wmax[3][c])));
            float col[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) col[j] = f[j][k];
            leave(k, byte, q8_cvt8<FMT>(col, q8_down(byte)));
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint32_t byte = q8_scale_byte<FMT>(bits[k]);
            const float up = q8_up(byte);
            uint32_t e[8];   // the column's elements: fp32 words, or pairs of rows in the first four
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if constexpr (DT == KP_F32) e[j] = v[j].w[k >> 2][k & 3];
                else if (j < 4) e[j] = __builtin_amdgcn_perm(v[2 * j + 1].w[0][k >> 1], v[2 * j].w[0][k >> 1], k & 1 ? 0x07060302u : 0x05040100u);
            }
            if constexpr (DT == KP_F32) leave(k, byte, q8_u32x2{q8_scaled4<DT, FMT>(e[0], e[1], e[2], e[3], up), q8_scaled4<DT, FMT>(e[4], e[5], e[6], e[7], up)});
            else leave(k, byte, q8_u32x2{q8_scaled4<DT, FMT>(e[0], e[1], 0u, 0u, up), q8_scaled4<DT, FMT>(e[2], e[3], 0u, 0u, up)});
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int id = i * TPB + t, c = id >> 3, piece = id & 7;
        const long long col = (long long)blockIdx.x * 128 + c;
        if (col < cols)
            *reinterpret_cast<q8_u32x4*>(qt + col * ldqt + (long long)blockIdx.y * 128 + piece * 16) =
                *reinterpret_cast<const q8_u32x4_a*>(tile + c * 128 + ((piece ^ ((c >> 3) & 7)) << 4));
    }
}

bool q8_aligned(const void* p, unsigned n) { return ((size_t)p % n) == 0; }
unsigned q8_grid(unsigned total) {
    const unsigned g = cdiv(total, TPB / 16 * UNROLL);
    return g < 8192 ? g : 8192;
}

template <int DT, int FMT>
int pack_launch(const void* x, long long ldx, uint8_t* q, long long ldq, uint8_t* s, long long lds, unsigned nb, unsigned total,
                long long cols, int padded, hipStream_t st) {
    q8_pack_k<DT, FMT><<<q8_grid(total), TPB, 0, st>>>(x, ldx, q, ldq, s, lds, nb, row_div(nb, total), total, cols, padded);
    return kp_check_launch("q8_pack");
}
template <int DT, int FMT>
int unpack_launch(const uint8_t* q, long long ldq, const uint8_t* s, long long lds, void* y, long long ldy, unsigned nb, unsigned total,
                  long long cols, hipStream_t st) {
    q8_unpack_k<DT, FMT><<<q8_grid(total), TPB, 0, st>>>(q, ldq, s, lds, y, ldy, nb, row_div(nb, total), total, cols);
    return kp_check_launch("q8_unpack");
}
template <int DT, int FMT>
int both_launch(const void* x, long long ldx, uint8_t* q, long long ldq, uint8_t* s, long long lds, uint8_t* qt, long long ldqt,
                uint8_t* stq, long long ldst, float* ws, float* colsum, long long rows, long long cols, hipStream_t st) {
    const dim3 grid(cdiv(cols, 128), cdiv(rows, 128));
    q8_pack_both_k<DT, FMT><<<grid, TPB, 0, st>>>(x, ldx, q, ldq, s, lds, qt, ldqt, stq, ldst, colsum ? ws : nullptr, rows, cols);
    if (colsum) q8_join_k<<<cdiv(cols, 16), 1024, 0, st>>>(ws, cdiv(rows, 128), cols, colsum, cols, nullptr);
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
