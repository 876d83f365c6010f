// Products of two matrices in the 8-bit block format (kp_q8_dev.h): C[m][n] = sum_k A[m][k] B[n][k] (+ bias[n]), both operands in rows
// along k, on the matrix instructions of gfx950.  Two ways to the same numbers:
//
//   16-bit results   the scaled 8-bit instruction.  It takes one exponent byte per operand row and 32 elements; a block of 128 hands the
//                    same byte to its four parts, so scaling costs no arithmetic.  Its accumulator is fp32, but inside the instruction
//                    the products of 8 neighbouring k are aligned to the largest of them and cut off below 2^-13 of it: a result is off
//                    by less than 7 * 2^-13 of the sum of the groups' largest products.  That is no bound against the result itself:
//                    where its products cancel it can be off by more than its own last place.  Taken all the same because the operands
//                    are rounded by up to 2^-4 (e5m2 2^-3) an element, which weighs over a hundred times as much in the same sum, and
//                    because sums of exact products (below) have half the rate; who needs them asks for fp32 results.
//   fp32 results     e4m3 and e5m2 values times a power of two are exact in bfloat16 and so are their products in fp32: the elements are
//                    converted on the way from LDS (exponent and all) and multiplied by the bfloat16 instruction, whose sums are fp32
//                    sums (measured 6e-9 .. 4e-7 of the norm), at half its partner's rate.  Weight gradients go this way.  (Elements
//                    below bfloat16's normal numbers, 2^-126, may be lost; one that was rounded up to 2^128 is an infinity.)
//
// Measured (bf16 / fp32 results; the library's 8-bit product reaches 2.75 PFLOP/s on the first): 8192^3 490 us = 2.25 PFLOP/s / 815 us =
// 1.35 (555 / 840 on the slowest card), 4096^3 67 / 111 us = 2.0 / 1.25, 16384 x 2048 x 4096 119 / 204 us = 2.3 / 1.35, 2048^3 14 / 24 us.  The
// largest are bound by the power cap: at 8192^3 the clock falls to 1.6 GHz with the matrix cores 62 % busy, at 4096^3 it stays at 2.2 GHz with
// 43 %.  Raising the waves' priority around the products changes nothing.
//
// Any order of the elements inside a block serves, as long as A and B agree: the fragments are read as the swizzle likes them.
#include <math.h>
#include "kp_mfma_util.h"
#include "kp_q8_dev.h"

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct MmArgs {
    const uint8_t *a, *sa, *b, *sb;
    long long lda, ldsa, ldb, ldsb;
    const float* bias;
    void* c;
    long long ldc;
    float* part;                 // splits > 1: fp32 partial products [splits][M][N]
    int M, N, nb;                // nb: blocks of 128 along k
    int tiles_m, tiles_n, splits, per_split;   // per_split: blocks of a split, a multiple of 4
    int dtype;
};

// every LDS access goes through types that may alias: the same bytes are written as fp32 or packed pairs and read as 16-byte pieces
typedef u32x4 __attribute__((may_alias)) u32x4_a;
typedef q8_u32x2 __attribute__((may_alias)) u32x2_a;
typedef f32x4 __attribute__((may_alias)) f32x4_a;

union Frag8 {
    i32x8 v;
    u32x4 h[2];
};

// fragment of 64 k-elements, half a row of 32 bytes a lane, and its conversion to bfloat16: 8 elements of piece `i`
template <int F> __device__ __forceinline__ h16x8 q8_bf16x8(const i32x8& v, int i, float up) {
    typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
    u32x4 r;
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            bf2 o;
            if constexpr (F == 0) o = h ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * i + w], up, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * i + w], up, false);
            else o = h ? __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(v[2 * i + w], up, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(v[2 * i + w], up, false);
            r[2 * w + h] = __builtin_bit_cast(uint32_t, o);
        }
    return __builtin_bit_cast(h16x8, r);
}

// One output tile of BM x BN a workgroup, waves in a grid of WGM x WGN.  A step of 128 k-elements is staged through LDS by DMA (two buffers,
// the next step's load in flight during this one); rows of 128 bytes, the 16-byte piece XOR-swizzled by the row pair on the DMA's source and
// on the read, so that 16 lanes of a ds_read_b128 hit 16 different slots.  One barrier a step: fragments of a step's second half are read
// under the first half's products, those of the next step's first half under the second's.  The operands are swapped (the instruction's
// A = rows of B): a lane then holds 4 consecutive n of one m and the epilogue packs them.  Tiles at the far edges are moved back to end with
// the matrix (the rows they share with their neighbours are computed twice, to the same values); EDGE: for matrices smaller than a tile,
// rows past the end repeat the last one and are not stored.  FA, FB: 0 e4m3, 1 e5m2.  F32: the bfloat16 way.
template <int BM, int BN, int WGM, int WGN, int FA, int FB, bool F32, bool EDGE>
__global__ __launch_bounds__(64 * WGM * WGN, 2) void q8_mm_k(const MmArgs P) {
    constexpr int NW = WGM * WGN, WM = BM / WGM, WN = BN / WGN, TM = WM / 32, TN = WN / 32;
    constexpr int ABYTES = BM * 128, BBYTES = BN * 128, BUF = ABYTES + BBYTES;
    constexpr int IA = BM / 8 / NW, IB = BN / 8 / NW;   // DMA instructions of 8 rows a wave and step
    static_assert(NW * 32 * WN * 4 <= 2 * BUF, "epilogue staging");
    __shared__ __attribute__((aligned(16))) uint8_t smem[2 * BUF];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WGN, wn = wave % WGN, fr = lane & 31, fh = lane >> 5;

    // tile of this workgroup: an XCD (blockIdx % 8) takes a contiguous range of tiles, ordered in groups of 8 tile rows, so that the
    // workgroups that share an L2 work on neighbouring tiles
    const int tiles = P.tiles_m * P.tiles_n, total = tiles * P.splits;
    const int xcd = blockIdx.x & 7, q = total >> 3, r = total & 7;
    int id = xcd * q + (xcd < r ? xcd : r) + (blockIdx.x >> 3);
    const int z = id / tiles;
    id -= z * tiles;
    const int per_group = 8 * P.tiles_n, group = id / per_group, first = group * 8;
    const int gm = P.tiles_m - first < 8 ? P.tiles_m - first : 8;
    const int rest = id - group * per_group;
    int m0 = (first + rest % gm) * BM, n0 = (rest / gm) * BN;
    if (!EDGE) {
        m0 = m0 < P.M - BM ? m0 : P.M - BM;
        n0 = n0 < P.N - BN ? n0 : P.N - BN;
    }
    const int kb0 = z * P.per_split, kb1 = kb0 + P.per_split < P.nb ? kb0 + P.per_split : P.nb;

    const auto ra = __builtin_amdgcn_make_buffer_rsrc((void*)(P.a + (long long)m0 * P.lda), 0, 0x7ffffffe, 0x00020000);
    const auto rb = __builtin_amdgcn_make_buffer_rsrc((void*)(P.b + (long long)n0 * P.ldb), 0, 0x7ffffffe, 0x00020000);
    const auto rsa = __builtin_amdgcn_make_buffer_rsrc((void*)(P.sa + (long long)m0 * P.ldsa), 0, 0x7ffffffe, 0x00020000);
    const auto rsb = __builtin_amdgcn_make_buffer_rsrc((void*)(P.sb + (long long)n0 * P.ldsb), 0, 0x7ffffffe, 0x00020000);
    const int lda = (int)P.lda, ldb = (int)P.ldb, ldsa = (int)P.ldsa, ldsb = (int)P.ldsb;
    const int last_m = P.M - 1 - m0, last_n = P.N - 1 - n0;
    auto clamp = [](int row, int last) { return EDGE && row > last ? last : row; };

    // DMA instruction i of this wave fetches rows (i * NW + wave) * 8 .. + 7; its rows are i * NW * 8 below those of instruction 0, with the
    // same swizzle, so one lane offset and a scalar one serve them all (EDGE: the clamped row is per lane)
    const int lrow = lane >> 3, slot = lane & 7;
    constexpr int NA = EDGE ? IA : 1, NB = EDGE ? IB : 1;
    int va[NA], vb[NB];
#pragma unroll
    for (int i = 0; i < NA; ++i) {
        const int row = (i * NW + wave) * 8 + lrow;
        va[i] = clamp(row, last_m) * lda + ((slot ^ ((row >> 1) & 7)) << 4);
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        const int row = (i * NW + wave) * 8 + lrow;
        vb[i] = clamp(row, last_n) * ldb + ((slot ^ ((row >> 1) & 7)) << 4);
    }
    auto issue = [&](int buf, int kb) {   // buf: byte offset of the buffer
        uint8_t* dst = smem + buf + wave * 1024;
#pragma unroll
        for (int i = 0; i < IA; ++i) dma16(ra, dst + i * NW * 1024, va[EDGE ? i : 0], kb * 128 + (EDGE ? 0 : i * NW * 8 * lda));
#pragma unroll
        for (int i = 0; i < IB; ++i) dma16(rb, dst + ABYTES + i * NW * 1024, vb[EDGE ? i : 0], kb * 128 + (EDGE ? 0 : i * NW * 8 * ldb));
    };
    constexpr int NSA = EDGE ? TM : 1, NSB = EDGE ? TN : 1;
    int vsa[NSA], vsb[NSB];
#pragma unroll
    for (int i = 0; i < NSA; ++i) vsa[i] = clamp(wm * WM + i * 32 + fr, last_m) * ldsa;
#pragma unroll
    for (int i = 0; i < NSB; ++i) vsb[i] = clamp(wn * WN + i * 32 + fr, last_n) * ldsb;
    struct Scales { int a[TM], b[TN]; };   // exponent bytes of up to four consecutive blocks of this lane's rows, the current one lowest
    auto load_scales = [&](Scales& s, int kb) {
#pragma unroll
        for (int i = 0; i < TM; ++i) s.a[i] = __builtin_amdgcn_raw_buffer_load_b32(rsa, vsa[EDGE ? i : 0], kb + (EDGE ? 0 : i * 32 * ldsa), 0);
#pragma unroll
        for (int i = 0; i < TN; ++i) s.b[i] = __builtin_amdgcn_raw_buffer_load_b32(rsb, vsb[EDGE ? i : 0], kb + (EDGE ? 0 : i * 32 * ldsb), 0);
    };

    struct Frags { Frag8 a[TM], b[TN]; };
    const int piece0 = (fh ^ ((fr >> 1) & 7)) << 4;
    const int abase = (wm * WM + fr) * 128 + piece0, bbase = ABYTES + (wn * WN + fr) * 128 + piece0;
    auto load_frags = [&](Frags& f, int buf, int kk) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int flip = (kk * 4 + u * 2) << 4;   // (16-byte piece (kk * 4 + u * 2 + fh) ^ swizzle)
            int oa = abase + buf, ob = bbase + buf;
            asm volatile("" : "+v"(oa), "+v"(ob));    // (formed here each time: hoisted, the eight addresses would cost registers)
            const uint8_t* pa = smem + (oa ^ flip);
            const uint8_t* pb = smem + (ob ^ flip);
#pragma unroll
            for (int i = 0; i < TM; ++i) f.a[i].h[u] = *reinterpret_cast<const u32x4_a*>(pa + i * 4096);
#pragma unroll
            for (int i = 0; i < TN; ++i) f.b[i].h[u] = *reinterpret_cast<const u32x4_a*>(pb + i * 4096);
        }
    };
    // accumulators start at the bias of the lane's columns (the join adds it to split sums)
    const bool split = P.splits > 1;
    const int nw = n0 + wn * WN;
    const auto rbias = __builtin_amdgcn_make_buffer_rsrc((void*)P.bias, 0, P.bias && !split ? P.N * 4 : 0, 0x00020000);
    f32x16 acc[TN][TM];
#pragma unroll
    for (int n = 0; n < TN; ++n)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            float v[4];   // (out of the resource's range -- no bias, or columns past the end -- loads give zero)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rbias, (nw + n * 32 + g * 8 + fh * 4 + e) * 4, 0, 0));
#pragma unroll
            for (int m = 0; m < TM; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[n][m][g * 4 + e] = v[e];
        }
    Scales sc, sc_next;
    auto mma = [&](const Frags& f) {
        if constexpr (!F32) {
#pragma unroll
            for (int n = 0; n < TN; ++n)
#pragma unroll
                for (int m = 0; m < TM; ++m)
                    acc[n][m] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(f.b[n].v, f.a[m].v, acc[n][m], FB, FA, 0, sc.b[n], 0, sc.a[m]);
        } else {
            typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
            float ua[TM], ub[TN];
#pragma unroll
            for (int m = 0; m < TM; ++m) ua[m] = q8_up((uint32_t)sc.a[m] & 255u);
#pragma unroll
            for (int n = 0; n < TN; ++n) ub[n] = q8_up((uint32_t)sc.b[n] & 255u);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                bf8 xa[TM];
#pragma unroll
                for (int m = 0; m < TM; ++m) xa[m] = __builtin_bit_cast(bf8, q8_bf16x8<FA>(f.a[m].v, i, ua[m]));
#pragma unroll
                for (int n = 0; n < TN; ++n) {
                    const bf8 xb = __builtin_bit_cast(bf8, q8_bf16x8<FB>(f.b[n].v, i, ub[n]));
#pragma unroll
                    for (int m = 0; m < TM; ++m) acc[n][m] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xb, xa[m], acc[n][m], 0, 0, 0);
                }
            }
        }
    };

    // keeps the products above where they are written, under the reads they cover: the compiler would sink them past the barrier and the
    // branches behind it to the products below (an empty statement that names one register of each accumulator; nothing reads it)
    auto pin = [&]() {
#pragma unroll
        for (int n = 0; n < TN; ++n)
#pragma unroll
            for (int m = 0; m < TM; ++m) asm volatile("" ::"v"(acc[n][m][0]));
        __builtin_amdgcn_sched_barrier(0);
    };

    Frags f0, f1;
    load_scales(sc, kb0);
    sc_next = sc;
    issue(0, kb0);
    if (kb0 + 1 < kb1) {
        issue(BUF, kb0 + 1);
        wait_vm<IA + IB>();
    } else wait_vm<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    load_frags(f0, 0, 0);
    int buf = 0;
#pragma unroll 1
    for (int k = kb0; k < kb1; ++k) {
        if constexpr (!F32) load_frags(f1, buf, 1);
        __builtin_amdgcn_sched_barrier(0);
        mma(f0);
        pin();
        if constexpr (F32) {   // (no registers for a second set beside the converted operands: the other wave of the SIMD covers the reads)
            load_frags(f0, buf, 1);
            mma(f0);
            pin();
        }
        // this wave's reads of the buffer have returned and its part of the next step has arrived: behind the barrier that holds for every
        // wave, and the buffer takes the step after the next.  (After the last step the fragments read here are never used.)
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        // (nothing is in flight here: named at this point, the exponent words cost no wait of their own where they are taken over)
#pragma unroll
        for (int i = 0; i < TM; ++i) asm volatile("" : "+v"(sc_next.a[i]));
#pragma unroll
        for (int i = 0; i < TN; ++i) asm volatile("" : "+v"(sc_next.b[i]));
        if (k + 2 < kb1) issue(buf, k + 2);
        buf ^= BUF;
        load_frags(f0, buf, 0);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (!F32) mma(f1);
        pin();
        if ((k & 3) == 3) sc = sc_next;     // (splits start on multiples of four blocks)
        else {
#pragma unroll
            for (int i = 0; i < TM; ++i) sc.a[i] = (int)((uint32_t)sc.a[i] >> 8);
#pragma unroll
            for (int i = 0; i < TN; ++i) sc.b[i] = (int)((uint32_t)sc.b[i] >> 8);
            if ((k & 3) == 0 && k + 4 < kb1) load_scales(sc_next, k + 4);
        }
    }
    __syncthreads();

    // epilogue: 32 rows of m at a time through a wave's own staging rows in LDS (16-byte pieces XOR-swizzled by the row), then whole rows
    // of WN elements leave
    uint8_t* stage = smem + wave * (32 * WN * 4);
    auto store_rows = [&](auto DTC) {
        constexpr int DT = decltype(DTC)::value, ES = el_size<DT>, ROW = WN * ES, PIECES = ROW / 16, PER = 16 / ES, RPI = 64 / PIECES;
        uint8_t* out = split ? (uint8_t*)(P.part + ((long long)z * P.M) * P.N) : (uint8_t*)P.c;
        const long long ldc = split ? P.N : P.ldc;
        const int prow = lane / PIECES, piece = lane % PIECES;   // this lane's piece of rows prow, prow + RPI, ...
        uint8_t* dst = out + ((m0 + wm * WM + prow) * ldc + nw + piece * PER) * ES;
        const bool whole = !EDGE || (m0 + BM <= P.M && n0 + BN <= P.N);
#pragma unroll
        for (int m = 0; m < TM; ++m) {
#pragma unroll
            for (int n = 0; n < TN; ++n)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int off = (n * 32 + g * 8 + fh * 4) * ES;
                    uint8_t* p = stage + fr * ROW + (((off >> 4) ^ (fr & (PIECES - 1))) << 4) + (off & 15);
                    const f32x16& v = acc[n][m];
                    if constexpr (DT == KP_F32) *reinterpret_cast<f32x4_a*>(p) = f32x4{v[g * 4], v[g * 4 + 1], v[g * 4 + 2], v[g * 4 + 3]};
                    else *reinterpret_cast<u32x2_a*>(p) = q8_u32x2{el_pack<DT>(v[g * 4], v[g * 4 + 1]), el_pack<DT>(v[g * 4 + 2], v[g * 4 + 3])};
                }
            auto piece_at = [&](int i) {
                const int row = i * RPI + prow;
                return *reinterpret_cast<const u32x4_a*>(stage + row * ROW + ((piece ^ (row & (PIECES - 1))) << 4));
            };
            if (whole) {
#pragma unroll
                for (int i = 0; i < 32 / RPI; ++i) *reinterpret_cast<q8_u32x4_e2*>(dst + (long long)(m * 32 + i * RPI) * ldc * ES) = piece_at(i);   // (rows may start anywhere)
            } else {
#pragma unroll 1
                for (int i = 0; i < 32 / RPI; ++i) {
                    const u32x4 w = piece_at(i);
                    uint8_t* d = dst + (long long)(m * 32 + i * RPI) * ldc * ES;
                    const int left = m0 + wm * WM + m * 32 + i * RPI + prow < P.M ? P.N - nw - piece * PER : 0;
#pragma unroll
                    for (int e = 0; e < PER; ++e)
                        if (e < left) {
                            if constexpr (ES == 4) reinterpret_cast<uint32_t*>(d)[e] = w[e];
                            else reinterpret_cast<uint16_t*>(d)[e] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
                        }
                }
            }
        }
    };
    if (split || P.dtype == KP_F32) store_rows(std::integral_constant<int, KP_F32>{});
    else if (P.dtype == KP_BF16) store_rows(std::integral_constant<int, KP_BF16>{});
    else store_rows(std::integral_constant<int, KP_F16>{});
}

// ---- x in its own type against a packed matrix: y[m][n] = P(x)[m] . W[n] (+ bias), one launch, no packed x in memory ---------------------
// A wave packs 16 rows of x in registers, where the 16 x 16 x 128 instruction wants them: lane r16 + 16 quarter holds elements quarter * 16 .. + 15
// and 64 further of row r16's block; the exponent goes straight into the instruction.
template <int DT> struct Raw32 { El8<DT> e[4]; };
template <int DT> __device__ __forceinline__ Raw32<DT> raw_block(const void* x, long long row_at, int k0, int quarter, int K, bool live) {
    Raw32<DT> r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int k = k0 + (i >> 1) * 64 + quarter * 16 + (i & 1) * 8;
        r.e[i] = el_raw8_any<DT>(x, row_at + k, live ? K - k : 0);
    }
    return r;
}
// bytes (into fx) and exponent byte of this lane's row; all lanes of the wave are active
template <int DT, int FMT> __device__ __forceinline__ uint32_t pack_rows16(const Raw32<DT>& raw, Frag8& fx) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = q8_raw_max<DT>(m, q8_raw_peak<DT>(raw.e[i]));
    m = q8_raw_max4<DT>(m);   // the row's four lanes
    if constexpr (DT != KP_F32) m = q8_umax(m & 0xffffu, m >> 16);
    const uint32_t bits = q8_raw_bits<DT>(m);
    if (__any(q8_plain<FMT>(bits))) {
        float v[4][8];
        uint32_t t = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            el_unpack8<DT>(raw.e[i], v[i]);
            t = q8_umax(t, q8_mag8(v[i]));
        }
        t = q8_raw_max4<KP_F32>(t);
        const uint32_t byte = q8_scale_byte<FMT>(t);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const q8_u32x2 o = q8_cvt8<FMT>(v[i], q8_down(byte));
            fx.v[2 * i] = (int)o[0];
            fx.v[2 * i + 1] = (int)o[1];
        }
        return byte;
    }
    const uint32_t byte = q8_scale_byte<FMT>(bits);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const q8_u32x2 o = q8_scaled8<DT, FMT>(raw.e[i], q8_up(byte));
        fx.v[2 * i] = (int)o[0];
        fx.v[2 * i + 1] = (int)o[1];
    }
    return byte;
}
// acc += 16 rows of W (its fragment and exponent byte) times 16 rows of x over a block; F32: exactly, through bfloat16
template <int FW, int FX, bool F32> __device__ __forceinline__ f32x4 mma16(const Frag8& fw, int ew, const Frag8& fx, uint32_t ex, f32x4 acc) {
    if constexpr (!F32) return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fw.v, fx.v, acc, FW, FX, 0, ew, 0, (int)ex);
    else {
        typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
        const float uw = q8_up((uint32_t)ew & 255u), ux = q8_up(ex);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, q8_bf16x8<FW>(fw.v, i, uw)), __builtin_bit_cast(bf8, q8_bf16x8<FX>(fx.v, i, ux)), acc, 0, 0, 0);
        return acc;
    }
}

// Few rows: 16 rows of W a wave stream past the packed rows, 16 x 16 x 128 a block; the 8 waves of a workgroup take every 8th block and join
// through LDS in wave order.  Bound by the bytes of W and, for a few million of them, by the way to memory and back: every wave has U blocks
// of loads in flight before its first product.  NT: groups of 16 rows of W a wave; two once that still gives every CU a workgroup, which
// halves the packing of x.
struct RowArgs {
    const void* x;
    long long ldx;
    const uint8_t *w, *sw;
    long long ldw, ldsw;
    const float* bias;
    void* y;
    long long ldy;
    int M, N, K, nb;
};
template <int DT, int FX, int FW, int NT>
__global__ __launch_bounds__(512) void q8_rows_k(const RowArgs P) {
    constexpr int NW = 8, U = DT == KP_F32 ? 2 : 4;
    __shared__ float red[NW][16][16 * NT + 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, quarter = lane >> 4;
    const int n0 = blockIdx.x * 16 * NT, m0 = blockIdx.y * 16;
    const bool mine = m0 + r16 < P.M;
    const uint8_t *w[NT], *sw[NT];
    f32x4 acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int at = n0 + t * 16 + r16, n = at < P.N ? at : P.N - 1;   // (rows of W past the end repeat the last one and are not stored)
        w[t] = P.w + (long long)n * P.ldw + quarter * 16;
        sw[t] = P.sw + (long long)n * P.ldsw;
        acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const long long xrow = (long long)(m0 + r16) * P.ldx;
    for (int kb0 = wave; kb0 < P.nb; kb0 += NW * U) {
        Frag8 fw[U][NT];
        int es[U][NT];
        Raw32<DT> raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int kb = kb0 + u * NW < P.nb ? kb0 + u * NW : P.nb - 1;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                fw[u][t].h[0] = *reinterpret_cast<const u32x4*>(w[t] + (long long)kb * 128);
                fw[u][t].h[1] = *reinterpret_cast<const u32x4*>(w[t] + (long long)kb * 128 + 64);
                es[u][t] = sw[t][kb];
            }
            raw[u] = raw_block<DT>(P.x, xrow, kb * 128, quarter, P.K, mine && kb0 + u * NW < P.nb);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (kb0 + u * NW >= P.nb) break;
            Frag8 fx;
            const uint32_t byte = pack_rows16<DT, FX + 1>(raw[u], fx);
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[t] = mma16<FW, FX, DT == KP_F32>(fw[u][t], es[u][t], fx, byte, acc[t]);
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) red[wave][r16][t * 16 + quarter * 4 + e] = acc[t][e];   // (a lane: column m = r16, rows n = 4 quarter + e)
    __syncthreads();
    if (threadIdx.x < 256 * NT) {
        const int m = threadIdx.x / (16 * NT), c = threadIdx.x % (16 * NT);
        if (m0 + m < P.M && n0 + c < P.N) {
            float v = P.bias ? P.bias[n0 + c] : 0.f;
#pragma unroll
            for (int k = 0; k < NW; ++k) v += red[k][m][c];
            el_store<DT>(P.y, (long long)(m0 + m) * P.ldy + n0 + c, v);
        }
    }
}

// Few columns (N <= 16 TN), many rows: bound by the bytes of x, which is read once.  A workgroup takes 64 rows, a wave 16 of them; all of W's
// block (N x 128 bytes) goes through LDS once for the four waves.  One barrier a block: while a block's fragments of W come from LDS, the
// next block of W goes there and the next 128 elements of x are packed; two more blocks of both are on their way in registers.  The loads
// stand in no branch (rows past the end repeat the last one, for blocks past the end all lanes read one address): behind a branch that may
// have issued none, the compiler waits for all that are on their way.  A short last block comes after the others.
// Measured (bf16): 32768 x 512 -> 128 12.5 us = 3.4 TB/s, 32768 x 4096 -> 64 46 us = 5.9 TB/s; against loads one block ahead behind branches:
// 8192 x 8192 -> 32 43 us instead of 72, 8192 x 4096 -> 128 28.9 instead of 37, 16384 x 2048 -> 16 12.1 instead of 18.3.
// LDS rows of 128 bytes, the 16-byte piece XOR-swizzled by the row pair as in q8_mm_k; the exponent bytes of rows r16, 16 + r16, ... side by side.
template <int DT, int FX, int FW, int TN>
__global__ __launch_bounds__(256, 2) void q8_narrow_k(const RowArgs P) {
    constexpr int BN = 16 * TN, PIECES = BN * 8, PER = (PIECES + 255) / 256;   // 16-byte pieces of a block of W, a thread's share
    __shared__ __attribute__((aligned(16))) uint8_t tile[2][BN * 128];
    __shared__ __attribute__((aligned(16))) uint8_t exps[2][16 * 8];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r16 = lane & 15, quarter = lane >> 4;
    const int m0 = blockIdx.x * 64 + wave * 16;
    const bool mine = m0 + r16 < P.M;
    const long long xrow = (long long)(mine ? m0 + r16 : P.M - 1) * P.ldx;
    const int erow = tid < P.N ? tid : P.N - 1, full = P.K / Q8_BLOCK;
    struct Ahead { u32x4 w[PER]; uint32_t e; Raw32<DT> x; };   // a thread's part of a block on its way
    auto fetch_w = [&](Ahead& r, int kb, bool in) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int id = i * 256 + tid, row = (id >> 3) < P.N ? id >> 3 : P.N - 1;
            r.w[i] = *reinterpret_cast<const u32x4*>(P.w + (in ? (long long)row * P.ldw + kb * 128LL + (id & 7) * 16 : 0));
        }
        r.e = P.sw[in ? (long long)erow * P.ldsw + kb : 0];
    };
    auto fetch = [&](Ahead& r, int kb) {
        const bool in = kb < full;
        fetch_w(r, kb, in);
#pragma unroll
        for (int i = 0; i < 4; ++i) r.x.e[i] = el_raw8<DT>(P.x, in ? xrow + kb * 128 + (i >> 1) * 64 + quarter * 16 + (i & 1) * 8 : 0);
    };
    auto put = [&](const Ahead& r, int buf) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int id = i * 256 + tid, row = id >> 3;
            if (PIECES % 256 == 0 || id < PIECES) *reinterpret_cast<u32x4_a*>(tile[buf] + row * 128 + (((id & 7) ^ ((row >> 1) & 7)) << 4)) = r.w[i];
        }
        if (tid < BN) exps[buf][(tid & 15) * 8 + (tid >> 4)] = (uint8_t)r.e;
    };
    auto meet = [&]() {   // this wave's reads of a buffer have returned and its part of the other one is written
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    f32x4 acc[TN];
#pragma unroll
    for (int t = 0; t < TN; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    Ahead r0, r1;
    constexpr int TW = TN < 4 ? TN : 4;   // tiles of W whose fragments are held at once
    Frag8 fx, fw[TW];
    uint32_t byte;
    q8_u32x2 ew;
    auto read_w = [&](int buf, int t0) {
#pragma unroll
        for (int t = 0; t < TW; ++t)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int row = (t0 + t) * 16 + r16;
                fw[t].h[u] = *reinterpret_cast<const u32x4_a*>(tile[buf] + row * 128 + (((u * 4 + quarter) ^ ((row >> 1) & 7)) << 4));
            }
        ew = *reinterpret_cast<const u32x2_a*>(exps[buf] + r16 * 8);
    };
    auto products = [&](int buf) {
#pragma unroll
        for (int t0 = 0; t0 < TN; t0 += TW) {
            if (t0) read_w(buf, t0);
#pragma unroll
            for (int t = 0; t < TW; ++t) acc[t0 + t] = mma16<FW, FX, DT == KP_F32>(fw[t], (int)(ew[t0 >> 2] >> (8 * t)), fx, byte, acc[t0 + t]);
        }
    };
    auto step = [&](int kb, Ahead& r) {   // r: block kb + 1
        Frag8 fxn;
        put(r, (kb & 1) ^ 1);
        const uint32_t byten = pack_rows16<DT, FX + 1>(r.x, fxn);
        fetch(r, kb + 3);
        __builtin_amdgcn_sched_barrier(0);
        read_w(kb & 1, 0);
        products(kb & 1);
        fx = fxn;
        byte = byten;
        meet();
    };
    if (full) {
        fetch(r0, 0);
        fetch(r1, 1);
        put(r0, 0);
        byte = pack_rows16<DT, FX + 1>(r0.x, fx);
        fetch(r0, 2);
        meet();
        for (int kb = 0; kb + 1 < full; kb += 2) {
            step(kb, r1);
            step(kb + 1, r0);
        }
        if (full & 1) step(full - 1, r1);
    }
    if (full < P.nb) {
        fetch_w(r0, full, true);
        r0.x = raw_block<DT>(P.x, xrow, full * 128, quarter, P.K, true);
        put(r0, 0);
        byte = pack_rows16<DT, FX + 1>(r0.x, fx);
        meet();
        read_w(0, 0);
        products(0);
    }
    if (!mine) return;
#pragma unroll
    for (int t = 0; t < TN; ++t) {   // a lane: row m = r16, columns t * 16 + quarter * 4 .. + 3
        const int n = t * 16 + quarter * 4;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[t][e] + (P.bias && n + e < P.N ? P.bias[n + e] : 0.f);
        const long long at = (long long)(m0 + r16) * P.ldy + n;
        if (n + 4 <= P.N) {
            if constexpr (DT == KP_F32) *reinterpret_cast<q8_u32x4_e4*>((float*)P.y + at) = q8_u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
            else *reinterpret_cast<q8_u32x2_e2*>((uint16_t*)P.y + at) = q8_u32x2{el_pack<DT>(v[0], v[1]), el_pack<DT>(v[2], v[3])};
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (n + e < P.N) el_store<DT>(P.y, at + e, v[e]);
        }
    }
}

// the splits' partial products, added in order, with the bias, rounded once
template <int DT>
__global__ __launch_bounds__(256) void q8_mm_join_k(const float* __restrict__ part, int splits, const float* __restrict__ bias,
                                                    void* __restrict__ c, long long ldc, int M, int N) {
    const long long total = (long long)M * N;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const long long m = i / N, n = i - m * N;
        float v = part[i];
        for (int z = 1; z < splits; ++z) v += part[z * total + i];
        if (bias) v += bias[n];
        el_store<DT>(c, m * ldc + n, v);
    }
}

struct Plan { int tile, splits, per_split; };

// Tile and split by a model of the time, from the sizes alone.  A step of 128 k-elements of w workgroups on a CU takes (us, fitted to
// measurements of 22 shapes; right: fp32 results):
//     64 x 64    0.15 + 0.18 w   0.23 + 0.29 w   (w <= 4)
//     128 x 128  0.29 + 0.44 w   0.80 + 0.60 w   (w <= 2)
//     256 x 256  1.95            3.2             (w = 1)
// and a split's partial products are written and read once more, at 4 TB/s, by a launch of 3 us.  Against the largest tile that fits, split
// until every CU has one (the first rule here): 777 x 1234 x 1000 18.3 -> 6.4 us, 1024^3 16.6 -> 5.2, 2048^3 36.6 -> 14.6, 512 x 4096 x 4096
// 35.6 -> 19.7, 300 x 300 x 8192 20.3 -> 10.6.
Plan plan_of(long long M, long long N, int nb, bool f32) {
    static const struct { int tile, most; double base[2], each[2]; } T[3] = {
        {64, 4, {0.15, 0.23}, {0.18, 0.29}}, {128, 2, {0.29, 0.80}, {0.44, 0.60}}, {256, 1, {0.0, 0.0}, {1.95, 3.2}}};
    const int groups = (nb + 3) / 4;   // splits start on multiples of four blocks (one word of exponent bytes)
    Plan best = {64, 1, groups * 4};
    double least = 1e30;
    for (const auto& t : T) {
        if (t.tile > 64 && (M < t.tile || N < t.tile)) break;
        const double tiles = (double)((M + t.tile - 1) / t.tile) * (double)((N + t.tile - 1) / t.tile);
        for (int s = 1; s <= 32 && s <= groups; s *= 2) {
            const int per = (groups + s - 1) / s * 4, splits = (nb + per - 1) / per;
            const double work = tiles * splits, slots = 256.0 * t.most, full = floor(work / slots), rest = work - full * slots;
            const double steps = per < nb ? per : nb, w = ceil(rest / 256.0);
            double us = steps * (full * (t.base[f32] + t.each[f32] * t.most) + (w > 0 ? t.base[f32] + t.each[f32] * w : 0.0));
            if (splits > 1) us += 3.0 + (double)M * (double)N * 8.0 * splits / 4e6;
            if (us < least) {
                least = us;
                best = Plan{t.tile, splits, per};
            }
        }
    }
    return best;
}

template <int FA, int FB, bool F32> int mm_launch(const MmArgs& P, const Plan& p, hipStream_t st) {
    const unsigned grid = (unsigned)(P.tiles_m * P.tiles_n * P.splits);
    if (p.tile == 256) q8_mm_k<256, 256, 4, 2, FA, FB, F32, false><<<grid, 512, 0, st>>>(P);
    else if (p.tile == 128) q8_mm_k<128, 128, 2, 2, FA, FB, F32, false><<<grid, 256, 0, st>>>(P);
    else q8_mm_k<64, 64, 2, 2, FA, FB, F32, true><<<grid, 256, 0, st>>>(P);
    return kp_check_launch("q8_matmul");
}

// 1: few rows, 2: few columns, 0: neither -- pack x and take the tiles.
//
// Few rows against that (bf16, us): 4096 x 4096: 1 row 6.7 / 11.8, 16 rows 9.2 / 12.6, 32 rows 16.6 / 13.4; 8192 x 8192: 1 row 17.3 / 23.7,
// 16 rows 20.9 / 24.1; 1024 x 1024, 64 rows 4.4 / 8.1; 4096 x 1000, 32 rows 6.7 / 8.8, 64 rows 12.0 / 9.1; 512 x 8192 (32 workgroups that
// walk 64 blocks each), 4 rows 10.6 / 11.3, 16 rows 14.8 / 12.2.  So: up to 16 rows, unless few workgroups walk far; more where the walk is
// short and two rounds of workgroups are enough.
// Few columns (bf16): a block takes a workgroup 0.9 us (128 columns) or 0.6 (64), whatever the number of workgroups, so it wants many rows, or
// few blocks and not all 128 columns.  128 columns: K = 512: 32768 rows 12.5 / 19.2, 8192 rows 7.9 / 9.3, 4096 rows 7.4 / 7.2; K = 4096: 32768 rows
// 57.8 / 116, 8192 rows 30.3 / 35.5, 4096 rows 28.8 / 24.2; K = 200: 2048 rows 5.5 / 5.7.  64 columns: K = 512: 2048 rows 5.0 / 6.6; K = 2048:
// 2048 rows 12.6 / 14.3; K = 4096: 2048 rows 22.2 / 18.2.  In fp32 a block takes nearly twice as long and packing does not: twice the rows.
int linear_way(long long M, long long N, long long K, bool f32) {
    if (M <= 4) return 1;
    if (M <= 16) return K <= 4096 || N >= 4096 ? 1 : 0;
    if (K <= 1024 && ((N + 15) / 16) * ((M + 15) / 16) <= 512) return 1;
    const long long rows = f32 ? M / 2 : M;
    return N <= 128 && (rows >= 6144 || (N <= 64 && rows >= 2048 && K <= 2048) || K <= 256) ? 2 : 0;
}

template <int DT, int FX, int FW> int narrow_launch(const RowArgs& P, hipStream_t st) {
    const unsigned grid = cdiv(P.M, 64);
    if (P.N <= 16) q8_narrow_k<DT, FX, FW, 1><<<grid, 256, 0, st>>>(P);
    else if (P.N <= 32) q8_narrow_k<DT, FX, FW, 2><<<grid, 256, 0, st>>>(P);
    else if (P.N <= 64) q8_narrow_k<DT, FX, FW, 4><<<grid, 256, 0, st>>>(P);
    else q8_narrow_k<DT, FX, FW, 8><<<grid, 256, 0, st>>>(P);
    return kp_check_launch("q8_linear");
}
template <int DT, int FX> int linear_launch(const RowArgs& P, int fmtw, hipStream_t st) {
    if (P.N <= 128 && linear_way(P.M, P.N, P.K, DT == KP_F32) != 1) return fmtw == KP_E4M3 ? narrow_launch<DT, FX, 0>(P, st) : narrow_launch<DT, FX, 1>(P, st);
    const bool two = P.N >= 32 * 256;
    const dim3 grid(cdiv(P.N, two ? 32 : 16), cdiv(P.M, 16));
    if (two) {
        if (fmtw == KP_E4M3) q8_rows_k<DT, FX, 0, 2><<<grid, 512, 0, st>>>(P);
        else q8_rows_k<DT, FX, 1, 2><<<grid, 512, 0, st>>>(P);
    } else {
        if (fmtw == KP_E4M3) q8_rows_k<DT, FX, 0, 1><<<grid, 512, 0, st>>>(P);
        else q8_rows_k<DT, FX, 1, 1><<<grid, 512, 0, st>>>(P);
    }
    return kp_check_launch("q8_linear");
}

}  // namespace

extern "C" {

static bool mm_sizes_ok(long long M, long long N, long long K) {
    return M > 0 && N > 0 && K > 0 && M <= 0x7fffff00LL && N <= 0x1fffff00LL && K <= (1LL << 23);
}

long long kp_q8_matmul_ws_floats(long long M, long long N, long long K, int dtype) {
    if (!mm_sizes_ok(M, N, K)) return 0;
    const Plan p = plan_of(M, N, (int)((K + Q8_BLOCK - 1) / Q8_BLOCK), dtype == KP_F32);
    return p.splits > 1 ? p.splits * M * N : 0;
}

int kp_q8_matmul_tile(long long M, long long N, long long K, int dtype) {
    return mm_sizes_ok(M, N, K) ? plan_of(M, N, (int)((K + Q8_BLOCK - 1) / Q8_BLOCK), dtype == KP_F32).tile : 0;
}

int kp_q8_matmul(const unsigned char* a, long long lda, const unsigned char* sa, long long ldsa, int fmta, const unsigned char* b,
                 long long ldb, const unsigned char* sb, long long ldsb, int fmtb, const float* bias, void* c, long long ldc, float* ws,
                 long long M, long long N, long long K, int dtype, void* stream) {
    KP_REQUIRE(a && sa && b && sb && c && M > 0 && N > 0 && K > 0, "kp_q8_matmul: bad args (%lld x %lld x %lld)", M, N, K);
    KP_REQUIRE((fmta == KP_E4M3 || fmta == KP_E5M2) && (fmtb == KP_E4M3 || fmtb == KP_E5M2), "kp_q8_matmul: unknown format %d / %d", fmta, fmtb);
    KP_REQUIRE(dtype == KP_F32 || dtype == KP_BF16 || dtype == KP_F16, "kp_q8_matmul: unknown dtype %d", dtype);
    const long long nb = (K + Q8_BLOCK - 1) / Q8_BLOCK, words = (nb + 3) / 4 * 4;
    KP_REQUIRE(mm_sizes_ok(M, N, K) && lda < (1LL << 23) && ldb < (1LL << 23) && ldsa < (1LL << 23) && ldsb < (1LL << 23),
               "kp_q8_matmul: %lld x %lld x %lld is more than one call takes (2^23 along the product, 2^31 and 2^29 rows)", M, N, K);
    KP_REQUIRE(lda >= nb * Q8_BLOCK && ldb >= nb * Q8_BLOCK && lda % 16 == 0 && ldb % 16 == 0 && ((size_t)a & 15) == 0 && ((size_t)b & 15) == 0,
               "kp_q8_matmul: operand rows must be padded to whole blocks and start on multiples of 16 bytes (strides %lld, %lld)", lda, ldb);
    KP_REQUIRE(ldsa >= words && ldsb >= words && ldsa % 4 == 0 && ldsb % 4 == 0 && ((size_t)sa & 3) == 0 && ((size_t)sb & 3) == 0,
               "kp_q8_matmul: rows of exponent bytes must be padded to words (strides %lld, %lld)", ldsa, ldsb);
    KP_REQUIRE(ldc >= N, "kp_q8_matmul: output row stride %lld for %lld columns", ldc, N);
    const Plan p = plan_of(M, N, (int)nb, dtype == KP_F32);
    KP_REQUIRE(p.splits == 1 || ws, "kp_q8_matmul: this shape needs a workspace (kp_q8_matmul_ws_floats)");
    MmArgs P;
    P.a = a; P.sa = sa; P.b = b; P.sb = sb; P.lda = lda; P.ldsa = ldsa; P.ldb = ldb; P.ldsb = ldsb; P.bias = bias; P.c = c; P.ldc = ldc;
    P.part = ws; P.M = (int)M; P.N = (int)N; P.nb = (int)nb; P.dtype = dtype;
    P.tiles_m = (int)cdiv(M, p.tile); P.tiles_n = (int)cdiv(N, p.tile); P.splits = p.splits; P.per_split = p.per_split;
    KP_REQUIRE((long long)P.tiles_m * P.tiles_n * P.splits < (1LL << 31), "kp_q8_matmul: %lld x %lld is more than one call takes", M, N);
    kp_count_bytes((double)(M + N) * K + (double)M * N * (dtype == KP_F32 ? 4 : 2));
    const hipStream_t st = (hipStream_t)stream;
    int rc;
    const int f = (fmta == KP_E5M2 ? 2 : 0) | (fmtb == KP_E5M2 ? 1 : 0);
    if (dtype == KP_F32) rc = f == 0 ? mm_launch<0, 0, true>(P, p, st) : f == 1 ? mm_launch<0, 1, true>(P, p, st) : f == 2 ? mm_launch<1, 0, true>(P, p, st) : mm_launch<1, 1, true>(P, p, st);
    else rc = f == 0 ? mm_launch<0, 0, false>(P, p, st) : f == 1 ? mm_launch<0, 1, false>(P, p, st) : f == 2 ? mm_launch<1, 0, false>(P, p, st) : mm_launch<1, 1, false>(P, p, st);
    if (rc != KP_OK || p.splits == 1) return rc;
    const unsigned grid = M * N > 256LL * 2048 ? 2048 : cdiv((size_t)(M * N), 256);
    if (dtype == KP_F32) q8_mm_join_k<KP_F32><<<grid, 256, 0, st>>>(ws, p.splits, bias, c, ldc, (int)M, (int)N);
    else if (dtype == KP_BF16) q8_mm_join_k<KP_BF16><<<grid, 256, 0, st>>>(ws, p.splits, bias, c, ldc, (int)M, (int)N);
    else q8_mm_join_k<KP_F16><<<grid, 256, 0, st>>>(ws, p.splits, bias, c, ldc, (int)M, (int)N);
    return kp_check_launch("q8_matmul join");
}

int kp_q8_linear_suits(long long M, long long N, long long K, int dtype) { return linear_way(M, N, K, dtype == KP_F32) != 0; }

int kp_q8_linear(const void* x, long long ldx, int fmtx, const unsigned char* w, long long ldw, const unsigned char* sw, long long ldsw,
                 int fmtw, const float* bias, void* y, long long ldy, long long M, long long N, long long K, int dtype, void* stream) {
    KP_REQUIRE(x && w && sw && y && M > 0 && N > 0 && K > 0, "kp_q8_linear: bad args (%lld x %lld x %lld)", M, N, K);
    KP_REQUIRE((fmtx == KP_E4M3 || fmtx == KP_E5M2) && (fmtw == KP_E4M3 || fmtw == KP_E5M2), "kp_q8_linear: unknown format %d / %d", fmtx, fmtw);
    KP_REQUIRE(dtype == KP_F32 || dtype == KP_BF16 || dtype == KP_F16, "kp_q8_linear: unknown dtype %d", dtype);
    const long long nb = (K + Q8_BLOCK - 1) / Q8_BLOCK;
    KP_REQUIRE(M < (1LL << 31) - 64 && (N <= 128 || M <= 65535LL * 16) && N <= 0x7fffff00LL && K < (1LL << 30), "kp_q8_linear: %lld x %lld x %lld is more than one call takes", M, N, K);
    KP_REQUIRE(ldw >= nb * Q8_BLOCK && ldw % 16 == 0 && ((size_t)w & 15) == 0 && ldsw >= nb, "kp_q8_linear: the weight's rows must be padded to whole blocks and start on multiples of 16 bytes (strides %lld, %lld)", ldw, ldsw);
    KP_REQUIRE((M == 1 || ldx >= K) && ldy >= N, "kp_q8_linear: row strides %lld, %lld for %lld and %lld columns", ldx, ldy, K, N);
    RowArgs P{x, ldx, w, sw, ldw, ldsw, bias, y, ldy, (int)M, (int)N, (int)K, (int)nb};
    const hipStream_t st = (hipStream_t)stream;
    kp_count_bytes((double)N * K + (double)(M * K + M * N) * (dtype == KP_F32 ? 4 : 2));
    if (dtype == KP_F32) return fmtx == KP_E4M3 ? linear_launch<KP_F32, 0>(P, fmtw, st) : linear_launch<KP_F32, 1>(P, fmtw, st);
    if (dtype == KP_BF16) return fmtx == KP_E4M3 ? linear_launch<KP_BF16, 0>(P, fmtw, st) : linear_launch<KP_BF16, 1>(P, fmtw, st);
    return fmtx == KP_E4M3 ? linear_launch<KP_F16, 0>(P, fmtw, st) : linear_launch<KP_F16, 1>(P, fmtw, st);
}

}  // extern "C"
