// The 8-bit block format of kp_q8_dev.h: rows to 8 bits, back, and both ways at once (rows and columns) with the column sums.
// All of it is bound by memory: 2 (4) bytes of input and 1 byte per form an element.
#include "kp_q8_dev.h"

namespace {

constexpr int TPB = 256;
typedef q8_u32x2 __attribute__((may_alias)) q8_u32x2_a;   // (LDS is written as pairs of words and read as 16-byte pieces)
typedef q8_u32x4 __attribute__((may_alias)) q8_u32x4_a;

// A group of 16 lanes takes a block: 8 consecutive elements a lane, the block's maximum by DPP; UNROLL blocks of a thread in flight.
// `padded`: the row's last block is written out to its full 128 bytes with zeros.
constexpr int UNROLL = 2;
struct BlockAt { unsigned row, kb; long long c; int n; };   // n: elements of this lane's 8 that the row has
__device__ __forceinline__ BlockAt block_at(unsigned b, unsigned nb, unsigned total, long long cols, int sub) {
    BlockAt r;
    r.row = b < total ? b / nb : 0;
    r.kb = b < total ? b - r.row * nb : 0;
    r.c = (long long)r.kb * Q8_BLOCK + sub * 8;
    r.n = b >= total ? 0 : (cols - r.c >= 8 ? 8 : (cols > r.c ? (int)(cols - r.c) : 0));
    return r;
}
template <int DT, int FMT>
__global__ __launch_bounds__(TPB) void q8_pack_k(const void* __restrict__ x, long long ldx, uint8_t* __restrict__ q, long long ldq,
                                                 uint8_t* __restrict__ s, long long lds, unsigned nb, unsigned total, long long cols,
                                                 int padded) {
    const int sub = threadIdx.x & 15;
    const unsigned per = TPB / 16, stride = gridDim.x * per * UNROLL;
    for (unsigned b0 = blockIdx.x * per * UNROLL; b0 < total; b0 += stride) {
        BlockAt at[UNROLL];
        El8<DT> raw[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            at[u] = block_at(b0 + u * per + (threadIdx.x >> 4), nb, total, cols, sub);
            raw[u] = el_raw8_any<DT>(x, at[u].row * ldx + at[u].c, at[u].n);
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            float v[8];
            el_unpack8<DT>(raw[u], v);
            const uint32_t byte = q8_scale_byte<FMT>(q8_max16(q8_mag8(v)));
            if (b0 + u * per + (threadIdx.x >> 4) < total) {
                q8_store8(q + at[u].row * ldq + at[u].c, padded ? 8 : at[u].n, q8_cvt8<FMT>(v, q8_down(byte)));
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
                                                   long long lds, void* __restrict__ y, long long ldy, unsigned nb, unsigned total,
                                                   long long cols) {
    const int sub = threadIdx.x & 15;
    const unsigned per = TPB / 16, stride = gridDim.x * per * UNROLL;
    for (unsigned b0 = blockIdx.x * per * UNROLL; b0 < total; b0 += stride) {
        BlockAt at[UNROLL];
        q8_u32x2 raw[UNROLL];
        uint32_t byte[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            at[u] = block_at(b0 + u * per + (threadIdx.x >> 4), nb, total, cols, sub);
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
    float v[8][8];
#pragma unroll
    for (int j = 0; j < 8; ++j) el_load8<DT>(x, (r0 + j) * ldx + c0, r0 + j < rows ? n : 0, v[j]);
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
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        m[k] = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m[k] = q8_umax(m[k], q8_mag(v[j][k]));
        m[k] = q8_umax(m[k], (uint32_t)__shfl_xor((int)m[k], 16, 64));
        m[k] = q8_umax(m[k], (uint32_t)__shfl_xor((int)m[k], 32, 64));
    }
    if ((t & 63) < 16) {
#pragma unroll
        for (int k = 0; k < 8; ++k) wmax[wave][cv * 8 + k] = m[k];
    }
    if (colsum) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) sum += v[j][k];
            sum += __shfl_xor(sum, 16, 64);
            sum += __shfl_xor(sum, 32, 64);
            if ((t & 63) < 16) wsum[wave][cv * 8 + k] = sum;
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
        *reinterpret_cast<q8_u32x2_a*>(tile + c * 128 + (((g >> 1) ^ (cv & 7)) << 4) + (g & 1) * 8) = q8_cvt8<FMT>(col, q8_down(byte));
        if (g == 0 && c0 + k < cols) st[(c0 + k) * ldst + blockIdx.y] = (uint8_t)byte;
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
    q8_pack_k<DT, FMT><<<q8_grid(total), TPB, 0, st>>>(x, ldx, q, ldq, s, lds, nb, total, cols, padded);
    return kp_check_launch("q8_pack");
}
template <int DT, int FMT>
int unpack_launch(const uint8_t* q, long long ldq, const uint8_t* s, long long lds, void* y, long long ldy, unsigned nb, unsigned total,
                  long long cols, hipStream_t st) {
    q8_unpack_k<DT, FMT><<<q8_grid(total), TPB, 0, st>>>(q, ldq, s, lds, y, ldy, nb, total, cols);
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
