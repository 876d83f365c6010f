// Layer norm over the last dimension: y = (x - mean) * rstd * w + b per row of C elements, forward and backward, with the reduction of the
// weight's and bias's gradients.  Statistics and sums in fp32, over registers: a row is read once, its variance is the mean of the squared
// distances from its mean (no difference of large squares).
//
//   forward   reads x, writes y (and, for a backward, mean and rstd; with keep the row in the 8-bit block format of kp_q8_dev.h, taken from
//             the registers the row is in anyway)
//   backward  g = dy w, xh = (x - mean) rstd, dx = rstd (g - mean(g) - xh mean(g xh)); a thread's columns are the same for every row it
//             meets, so dw += dy xh and db += dy stay in its registers; one partial row a workgroup, joined by a second launch in a fixed
//             order (fp64), so equal calls give equal bits
//
// Both are bound by memory.  Measured (a large copy reaches 5.2 TB/s here): 2097152 rows of 64 in bf16: forward 112 us = 4.8 TB/s, backward with
// join 157 us = 5.1 TB/s; 8192 rows of 4096 in fp16: forward 25.7 us = 5.2 TB/s, backward 43.7 us = 4.6 TB/s, with an 8-bit copy 38.4 and 38.1 us
// = 4.4 TB/s (a pass of 170 MB: its start and end count); 4096 x 16384 in bf16 51 and 98 us = 5.3 and 4.1 TB/s.
// A row is spread over G lanes, 8 consecutive elements (16 bytes of a 16-bit type) each, NJ times: the smallest
// power of two that holds it up to a wave (rows of 64 elements: eight rows a wave; a wave takes up to 1024), then 4, 8 or 16 waves with
// sums through LDS, and beyond 16384 elements a workgroup that walks the row and reads it again.
#include "kp_q8_dev.h"

namespace {

// ---- sums and maxima over a row's G lanes (G <= 64: lanes of a wave, aligned; more: the whole workgroup) ---------------------------------
template <int CTRL> __device__ __forceinline__ float ln_dpp(float v) { return __uint_as_float(q8_dpp<CTRL>(__float_as_uint(v))); }
template <int G> __device__ __forceinline__ float ln_wave_sum(float v) {
    if constexpr (G >= 2) v += ln_dpp<0xB1>(v);      // lane ^ 1
    if constexpr (G >= 4) v += ln_dpp<0x4E>(v);      // lane ^ 2
    if constexpr (G >= 8) v += ln_dpp<0x141>(v);     // lane ^ 7
    if constexpr (G >= 16) v += ln_dpp<0x128>(v);    // lane + 8 of 16
    if constexpr (G >= 32) v += __shfl_xor(v, 16, 64);
    if constexpr (G >= 64) v += __shfl_xor(v, 32, 64);
    return v;
}
// sums of N values at once; `red`: N * (G / 64) * (rows a workgroup takes at once) floats that the workgroup's previous sum did not use
// (every thread calls it; one barrier)
template <int G, int N> __device__ __forceinline__ void ln_sums(float (&v)[N], float* red) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = ln_wave_sum<(G < 64 ? G : 64)>(v[i]);
    if constexpr (G > 64) {
        constexpr int W = G / 64;
        const int wave = threadIdx.x >> 6, base = wave / W * W * N;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) red[base + i * W + wave % W] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) v[i] += red[base + i * W + w];
        }
    }
}

struct LnFwd {
    const void* x; const float *w, *b; void* y; float *mean, *rstd; uint8_t *q, *s;
    long long ldx, ldy, rows; int C, nb; float eps;
};
struct LnBwd {
    const void *dy, *x; const uint8_t *q, *s; const float *w, *mean, *rstd; void* dx; float* part;
    long long lddy, ldx, lddx, rows; int C, nb;
};

// How a row's last chunks are read.  FULL: rows of exactly 8 G NJ elements.  OVERLAP: a chunk that would reach past the end starts 8 elements
// before it and counts those that no other lane has counted (it computes and stores the others as their lanes do): loads and stores stand in
// no branch, behind which the compiler would wait for everything on its way, stores too.  Against PARTS, element by element, the backward
// takes (bf16, us): 8192 x 4096 43.7 / 50.3, 32768 x 1024 45.6 / 53.1, 8192 x 8192 86.1 / 95.4, 2097152 x 64 157 / 159; the forward 32768 x 1024
// 26.2 / 28.6, 32768 x 1000 27.9 / 30.5, 4096 x 16384 51.0 / 57.1, with an 8-bit copy 2097152 x 64 144 / 151.
// PARTS stays for rows of less than 8 elements, and for kept rows whose overlapping chunk could lie in two blocks.
enum LnEnds { LN_FULL, LN_OVERLAP, LN_PARTS };

// A row's lanes: sub = thread % G, chunk j of 8 columns at (j * G + sub) * 8.  The next row's loads are in flight during this row's sums
// (not in the backward of the widest rows, two chunks a lane in workgroups of 1024: the 128 registers a lane has there go to the sums).
// A workgroup has 256 threads; past a wave, G in the forward and 1024 in the backward, so that the four rows of 256 lanes that are taken at
// once share one partial row of the weight's gradient.
template <int G> constexpr int ln_tpb = G > 64 ? 1024 : 256;
template <int G> constexpr int ln_fwd_tpb = G > 64 ? G : 256;

// KEEP: 0, or KP_E4M3 / KP_E5M2: the row leaves in 8 bits too
template <int DT, int G, int NJ, int KEEP, int ENDS>
__global__ __launch_bounds__(ln_fwd_tpb<G>) void ln_fwd_k(const LnFwd P) {
    constexpr int TPB = ln_fwd_tpb<G>, R = TPB / G;
    __shared__ float red[G > 64 ? 64 : 1];   // four sets of 16: two sums a row, alternating rows
    const int sub = threadIdx.x & (G - 1);
    const float inv = 1.f / (float)P.C;
    int col[NJ], n[NJ], skip[NJ];   // as in the backward; lanes past the last block of 128 do what the last block's lanes do
    float w[NJ][8], b[NJ][8];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        int c = (j * G + sub) * 8;
        const int left = P.C - c;
        if (ENDS == LN_OVERLAP && KEEP != 0 && c >= P.nb * Q8_BLOCK) c = (P.nb - 1) * Q8_BLOCK + (c & (Q8_BLOCK - 1));
        col[j] = ENDS == LN_OVERLAP && c > P.C - 8 ? P.C - 8 : c;
        n[j] = ENDS != LN_PARTS || left >= 8 ? 8 : (left < 0 ? 0 : left);
        skip[j] = ENDS == LN_OVERLAP && left < 8 ? (left < 0 ? 8 : 8 - left) : 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) { w[j][k] = 1.f; b[j][k] = 0.f; }
        if (P.w) el_load8<KP_F32>(P.w, col[j], n[j], w[j]);
        if (P.b) el_load8<KP_F32>(P.b, col[j], n[j], b[j]);
    }
    El8<DT> next[NJ];
    auto fetch = [&](long long row) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            if constexpr (ENDS != LN_PARTS) next[j] = el_raw8<DT>(P.x, row < P.rows ? row * P.ldx + col[j] : 0);
            else next[j] = el_raw8_any<DT>(P.x, row * P.ldx + col[j], row < P.rows ? n[j] : 0);
        }
    };
    const long long step = (long long)gridDim.x * R;
    long long row = (long long)blockIdx.x * R + threadIdx.x / G, r0 = (long long)blockIdx.x * R, odd = 0;
    float mean = 0.f, rstd = 0.f;
    auto stats = [&](long long at) {
        if (P.mean && sub == 0 && at >= 0 && at < P.rows) {
            P.mean[at] = mean;
            P.rstd[at] = rstd;
        }
    };
    fetch(row);
    auto turn = [&](auto ALL) {   // ALL: every row of the workgroup's turn is there
        const bool live = decltype(ALL)::value || row < P.rows;
        float v[NJ][8];
        float sum[1] = {0.f}, sq[1] = {0.f};
        El8<DT> raw[KEEP ? NJ : 1];
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            if constexpr (KEEP != 0) raw[j] = next[j];
            el_unpack8<DT>(next[j], v[j]);
#pragma unroll
            for (int k = 0; k < 8; ++k) sum[0] += ENDS != LN_OVERLAP || k >= skip[j] ? v[j][k] : 0.f;
        }
        stats(row - step);   // (the row before's: behind the loads, these stores in a branch would make the next turn wait for this turn's)
        fetch(row + step);
        float* slot = red + (G > 64 ? (odd ? 32 : 0) : 0);
        ln_sums<G, 1>(sum, slot);
        mean = sum[0] * inv;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                v[j][k] = ENDS != LN_PARTS || k < n[j] ? v[j][k] - mean : 0.f;
                const float once = ENDS != LN_OVERLAP || k >= skip[j] ? v[j][k] : 0.f;
                sq[0] = __builtin_fmaf(once, once, sq[0]);
            }
        ln_sums<G, 1>(sq, slot + (G > 64 ? 16 : 0));
        rstd = 1.f / sqrtf(sq[0] * inv + P.eps);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            if constexpr (KEEP != 0) {
                q8_u32x2 out;
                const uint32_t byte = q8_pack_block<DT, KEEP, (G < 16 ? G : 16)>(raw[j], out);
                if (live && n[j] > 0) {
                    q8_store8(P.q + row * P.C + col[j], n[j], out);
                    if (ENDS != LN_PARTS || (col[j] & (Q8_BLOCK - 1)) == 0) P.s[row * P.nb + col[j] / Q8_BLOCK] = (uint8_t)byte;   // (all of a block's lanes: no branch)
                }
            }
            float o[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) o[k] = __builtin_fmaf(v[j][k] * rstd, w[j][k], b[j][k]);
            if (live) el_store8<DT>(P.y, row * P.ldy + col[j], n[j], o);
        }
        r0 += step;
        row += step;
        odd ^= 1;
    };
    if constexpr (ENDS != LN_PARTS) {
        while (r0 + R <= P.rows) turn(std::true_type{});
        if (r0 < P.rows) turn(std::false_type{});
    } else
        while (r0 < P.rows) turn(std::false_type{});
    stats(row - step);
}

template <int DT, int G, int NJ, int KEEP, int ENDS>
__global__ __launch_bounds__(ln_tpb<G>) void ln_bwd_k(const LnBwd P) {
    constexpr int TPB = ln_tpb<G>, R = TPB / G, W = G < 64 ? G : 64;
    __shared__ float red[G > 64 ? 64 : 1];                                     // two sets of 32: two sums at once, alternating rows
    __shared__ float join[G == 1024 ? 1 : (G > 64 ? R * G * 8 : 4 * W * 8)];
    const int sub = threadIdx.x & (G - 1);
    const float inv = 1.f / (float)P.C;
    int col[NJ], n[NJ], skip[NJ];   // a chunk's first column, its elements that the row has, those that another lane counts
    float w[NJ][8], dw[NJ][8], db[NJ][8];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        const int c = (j * G + sub) * 8, left = P.C - c;
        col[j] = ENDS == LN_OVERLAP && left < 8 ? P.C - 8 : c;
        n[j] = ENDS != LN_PARTS || left >= 8 ? 8 : (left < 0 ? 0 : left);
        skip[j] = ENDS == LN_OVERLAP && left < 8 ? (left < 0 ? 8 : 8 - left) : 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) { w[j][k] = 1.f; dw[j][k] = db[j][k] = 0.f; }
        if (P.w) el_load8<KP_F32>(P.w, col[j], n[j], w[j]);
    }
    constexpr bool PRE = !(G == 1024 && NJ == 2);
    struct Row { El8<DT> dy[NJ], x[KEEP ? 1 : NJ]; q8_u32x2 q[KEEP ? NJ : 1]; uint32_t s[KEEP ? NJ : 1]; float mean, rstd; };
    auto fetch = [&](Row& r, long long row) {
        const bool live = row < P.rows;
        if constexpr (ENDS != LN_PARTS) {
            r.mean = P.mean[live ? row : 0];
            r.rstd = P.rstd[live ? row : 0];
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int c = col[j];
                if constexpr (KEEP != 0) {
                    r.s[j] = P.s[live ? row * P.nb + c / Q8_BLOCK : 0];
                    r.q[j] = q8_load8(P.q + (live ? row * P.C + c : 0), 8);
                } else r.x[j] = el_raw8<DT>(P.x, live ? row * P.ldx + c : 0);
                r.dy[j] = el_raw8<DT>(P.dy, live ? row * P.lddy + c : 0);
            }
            return;
        }
        r.mean = live ? P.mean[row] : 0.f;
        r.rstd = live ? P.rstd[row] : 0.f;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int c = col[j], m = live ? n[j] : 0;
            if constexpr (KEEP != 0) {
                r.s[j] = m > 0 ? P.s[row * P.nb + c / Q8_BLOCK] : 127u;
                r.q[j] = q8_load8(P.q + row * P.C + c, m);
            } else r.x[j] = el_raw8_any<DT>(P.x, row * P.ldx + c, m);
            r.dy[j] = el_raw8_any<DT>(P.dy, row * P.lddy + c, m);
        }
    };
    const long long step = (long long)gridDim.x * R;
    long long row = (long long)blockIdx.x * R + threadIdx.x / G;
    Row next;
    long long r0 = (long long)blockIdx.x * R, odd = 0;
    if constexpr (PRE) fetch(next, row);
    auto turn = [&](auto ALL) {   // ALL: every row of the workgroup's turn is there
        constexpr bool all = decltype(ALL)::value;
        if constexpr (!PRE) fetch(next, row);
        float g[NJ][8], xh[NJ][8];
        const bool here = all || row < P.rows;   // (rows past the end were read at the first one's start)
        const float mean = here ? next.mean : 0.f, rstd = here ? next.rstd : 0.f;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            if constexpr (KEEP != 0) q8_values8<KEEP>(next.q[j], q8_up(next.s[j]), xh[j]);
            else el_unpack8<DT>(next.x[j], xh[j]);
            el_unpack8<DT>(next.dy[j], g[j]);
            if constexpr (ENDS != LN_PARTS && !all)
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    g[j][k] = here ? g[j][k] : 0.f;
                    xh[j][k] = here ? xh[j][k] : 0.f;
                }
        }
        if constexpr (PRE) fetch(next, row + step);
        float ab[2] = {0.f, 0.f};   // sums of g and of g xh; past the row's end g is zero
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            if constexpr (!PRE)
                if (P.w) el_load8<KP_F32>(P.w, col[j], n[j], w[0]);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                xh[j][k] = (xh[j][k] - mean) * rstd;
                db[j][k] += g[j][k];
                dw[j][k] = __builtin_fmaf(g[j][k], xh[j][k], dw[j][k]);
                g[j][k] *= w[PRE ? j : 0][k];
                const float once = ENDS != LN_OVERLAP || k >= skip[j] ? g[j][k] : 0.f;
                ab[0] += once;
                ab[1] = __builtin_fmaf(once, xh[j][k], ab[1]);
            }
        }
        if (P.dx) {
            ln_sums<G, 2>(ab, red + (G > 64 ? (odd ? 32 : 0) : 0));
            const float a = ab[0] * inv, b = ab[1] * inv;
            if (here) {
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    float o[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) o[k] = rstd * (g[j][k] - a - xh[j][k] * b);
                    el_store8<DT>(P.dx, row * P.lddx + col[j], n[j], o);
                }
            }
        }
        r0 += step;
        row += step;
        odd ^= 1;
    };
    if constexpr (ENDS != LN_PARTS) {
        while (r0 + R <= P.rows) turn(std::true_type{});
        if (r0 < P.rows) turn(std::false_type{});
    } else
        while (r0 < P.rows) turn(std::false_type{});
    if (!P.part) return;
    // the workgroup's partial row [2][C]: lanes of a wave with the same columns first, then the waves (or rows) that share them
    float* prow = P.part + (long long)blockIdx.x * 2 * P.C;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float (&acc)[NJ][8] = which ? db : dw;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            float* dst = prow + which * P.C + col[j];
            if constexpr (G == 1024) {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (k < n[j] && k >= skip[j]) dst[k] = acc[j][k];
            } else {
                constexpr int GL = G > 64 ? G : W, SETS = G > 64 ? R : 4;   // columns' lanes, copies of them in LDS
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    float s = acc[j][k];
#pragma unroll
                    for (int o = W; o < 64; o <<= 1) s += __shfl_xor(s, o, 64);
                    if (G > 64 || (threadIdx.x & 63) < W) join[((G > 64 ? threadIdx.x / G : threadIdx.x >> 6) * GL + sub) * 8 + k] = s;
                }
                __syncthreads();
                if (threadIdx.x < GL)
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        if (k < n[j] && k >= skip[j]) {
                            float s = 0.f;
#pragma unroll
                            for (int t = 0; t < SETS; ++t) s += join[(t * GL + sub) * 8 + k];
                            dst[k] = s;
                        }
                __syncthreads();
            }
        }
    }
}

__device__ __forceinline__ float ln_total(float v, float* red) {   // over a workgroup of 1024
    float t[1] = {v};
    ln_sums<1024, 1>(t, red);
    return t[0];
}

// Rows past 16384 elements: a workgroup walks the row, element by element and thread, and reads it again for each pass (three times forward;
// twice backward and once more for the columns).  Right for any length, not made fast: 4096 x 20000 in bf16 174 us forward and 311 backward,
// 2.7 and 3.3 times what their bytes take (4096 x 16384 above: 1.0 and 1.3).
template <int DT, int KEEP>
__global__ __launch_bounds__(1024) void ln_fwd_long_k(const LnFwd P) {
    __shared__ float red[32];
    const float inv = 1.f / (float)P.C;
    for (long long row = blockIdx.x; row < P.rows; row += gridDim.x) {
        float sum = 0.f;
        for (int c = threadIdx.x; c < P.C; c += 1024) sum += el_load<DT>(P.x, row * P.ldx + c);
        const float mean = ln_total(sum, red) * inv;
        float sq = 0.f;
        for (int c = threadIdx.x; c < P.C; c += 1024) {
            const float d = el_load<DT>(P.x, row * P.ldx + c) - mean;
            sq = __builtin_fmaf(d, d, sq);
        }
        const float rstd = 1.f / sqrtf(ln_total(sq, red + 16) * inv + P.eps);
        for (int c = threadIdx.x; c < P.C; c += 1024) {
            float o = (el_load<DT>(P.x, row * P.ldx + c) - mean) * rstd;
            if (P.w) o *= P.w[c];
            if (P.b) o += P.b[c];
            el_store<DT>(P.y, row * P.ldy + c, o);
        }
        if (P.mean && threadIdx.x == 0) {
            P.mean[row] = mean;
            P.rstd[row] = rstd;
        }
        if constexpr (KEEP != 0) {   // 16 lanes a block, as in q8_pack_k
            const int sub = threadIdx.x & 15;
            for (int b0 = 0; b0 < P.nb; b0 += 64) {
                const int kb = b0 + (int)(threadIdx.x >> 4), c = kb * Q8_BLOCK + sub * 8;
                const int n = P.C - c >= 8 ? 8 : (P.C > c ? P.C - c : 0);
                q8_u32x2 out;
                const uint32_t byte = q8_pack_block<DT, KEEP, 16>(el_raw8_any<DT>(P.x, row * P.ldx + c, n), out);
                q8_store8(P.q + row * P.C + c, n, out);
                if (sub == 0 && kb < P.nb) P.s[row * P.nb + kb] = (uint8_t)byte;
            }
        }
        __syncthreads();
    }
}
template <int DT, int KEEP> __device__ __forceinline__ float ln_kept(const LnBwd& P, long long row, int c) {
    if constexpr (KEEP == 0) return el_load<DT>(P.x, row * P.ldx + c);
    else {
        float v[8];
        q8_values8<KEEP>(q8_u32x2{P.q[row * P.C + c], 0u}, q8_up(P.s[row * P.nb + c / Q8_BLOCK]), v);
        return v[0];
    }
}
template <int DT, int KEEP>
__global__ __launch_bounds__(1024) void ln_bwd_long_k(const LnBwd P) {
    __shared__ float red[32];
    const float inv = 1.f / (float)P.C;
    for (long long row = blockIdx.x; row < P.rows; row += gridDim.x) {
        const float mean = P.mean[row], rstd = P.rstd[row];
        float a = 0.f, b = 0.f;
        for (int c = threadIdx.x; c < P.C; c += 1024) {
            const float g = el_load<DT>(P.dy, row * P.lddy + c) * (P.w ? P.w[c] : 1.f);
            a += g;
            b = __builtin_fmaf(g, (ln_kept<DT, KEEP>(P, row, c) - mean) * rstd, b);
        }
        a = ln_total(a, red) * inv;
        b = ln_total(b, red + 16) * inv;
        for (int c = threadIdx.x; c < P.C; c += 1024) {
            const float g = el_load<DT>(P.dy, row * P.lddy + c) * (P.w ? P.w[c] : 1.f);
            el_store<DT>(P.dx, row * P.lddx + c, rstd * (g - a - (ln_kept<DT, KEEP>(P, row, c) - mean) * rstd * b));
        }
        __syncthreads();
    }
}
template <int DT, int KEEP>
__global__ __launch_bounds__(256) void ln_cols_long_k(const LnBwd P) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= P.C) return;
    float dw = 0.f, db = 0.f;
    for (long long row = blockIdx.y; row < P.rows; row += gridDim.y) {
        const float g = el_load<DT>(P.dy, row * P.lddy + c);
        db += g;
        dw = __builtin_fmaf(g, (ln_kept<DT, KEEP>(P, row, c) - P.mean[row]) * P.rstd[row], dw);
    }
    float* prow = P.part + (long long)blockIdx.y * 2 * P.C;
    prow[c] = dw;
    prow[P.C + c] = db;
}

// ---- which kernel -----------------------------------------------------------------------------------------------------------------
constexpr int LONG = 16384;
constexpr long long MOST = 1LL << 30;   // columns are counted in 32 bits, a partial row of 2 C floats and a walk's last step past its end included
int ln_group(int C) {   // lanes of a row
    if (C > 1024) return C > 4096 ? 1024 : C > 2048 ? 512 : 256;
    int g = 1;
    while (g < 64 && g * 8 < C) g <<= 1;
    return g;
}
int ln_rows(int C) { const int g = ln_group(C); return C > LONG ? 1 : (g > 64 ? 1024 : 256) / g; }   // rows a workgroup takes at once
// workgroups of the backward: every one leaves a partial row of 2 C floats, which the join reads back.  Rows within a wave: 16 waves a CU,
// short partial rows; wider ones: one workgroup of 16 waves a CU.
int ln_parts(long long rows, int C) {
    const int per = ln_rows(C);
    const long long want = (rows + per - 1) / per, cap = C > LONG ? 64 : (ln_group(C) > 64 ? 256 : 1024);
    return (int)(want < cap ? want : cap);
}

template <int DT, int KEEP> int fwd_launch(const LnFwd& P, hipStream_t st) {
    if (P.C > LONG) {
        ln_fwd_long_k<DT, KEEP><<<(unsigned)(P.rows < 1024 ? P.rows : 1024), 1024, 0, st>>>(P);
        return kp_check_launch("layer_norm_fwd");
    }
    const int g = ln_group(P.C), per = g > 64 ? 1 : 256 / g;
    const long long want = (P.rows + per - 1) / per, cap = g > 64 ? 1024 * 512 / g : 2048;
    const unsigned grid = (unsigned)(want < cap ? want : cap);
#define LN_FWD(G, NJ)                                                                                                    \
    do {                                                                                                                 \
        if (P.C == 8 * G * NJ) ln_fwd_k<DT, G, NJ, KEEP, LN_FULL><<<grid, ln_fwd_tpb<G>, 0, st>>>(P);                    \
        else if (KEEP ? P.C % 8 == 0 : G > 1) ln_fwd_k<DT, G, NJ, KEEP, LN_OVERLAP><<<grid, ln_fwd_tpb<G>, 0, st>>>(P);  \
        else ln_fwd_k<DT, KEEP ? G : 1, KEEP ? NJ : 1, KEEP, LN_PARTS><<<grid, ln_fwd_tpb<KEEP ? G : 1>, 0, st>>>(P);    \
    } while (0)
    switch (g) {
        case 1: LN_FWD(1, 1); break;
        case 2: LN_FWD(2, 1); break;
        case 4: LN_FWD(4, 1); break;
        case 8: LN_FWD(8, 1); break;
        case 16: LN_FWD(16, 1); break;
        case 32: LN_FWD(32, 1); break;
        case 64: if (P.C <= 512) LN_FWD(64, 1); else LN_FWD(64, 2); break;
        case 256: LN_FWD(256, 1); break;
        case 512: LN_FWD(512, 1); break;
        default: if (P.C <= 8192) LN_FWD(1024, 1); else LN_FWD(1024, 2); break;
    }
#undef LN_FWD
    return kp_check_launch("layer_norm_fwd");
}
template <int DT, int KEEP> int bwd_launch(const LnBwd& P, int parts, hipStream_t st) {
    if (P.C > LONG) {
        if (P.dx) ln_bwd_long_k<DT, KEEP><<<(unsigned)(P.rows < 1024 ? P.rows : 1024), 1024, 0, st>>>(P);
        if (P.part) ln_cols_long_k<DT, KEEP><<<dim3(cdiv(P.C, 256), parts), 256, 0, st>>>(P);
        return kp_check_launch("layer_norm_bwd");
    }
#define LN_BWD(G, NJ)                                                                                              \
    do {                                                                                                           \
        if (P.C == 8 * G * NJ) ln_bwd_k<DT, G, NJ, KEEP, LN_FULL><<<parts, ln_tpb<G>, 0, st>>>(P);                 \
        else if (KEEP ? P.C % 8 == 0 : G > 1) ln_bwd_k<DT, G, NJ, KEEP, LN_OVERLAP><<<parts, ln_tpb<G>, 0, st>>>(P); \
        else ln_bwd_k<DT, KEEP ? G : 1, KEEP ? NJ : 1, KEEP, LN_PARTS><<<parts, ln_tpb<G>, 0, st>>>(P);              \
    } while (0)
    switch (ln_group(P.C)) {
        case 1: LN_BWD(1, 1); break;
        case 2: LN_BWD(2, 1); break;
        case 4: LN_BWD(4, 1); break;
        case 8: LN_BWD(8, 1); break;
        case 16: LN_BWD(16, 1); break;
        case 32: LN_BWD(32, 1); break;
        case 64: if (P.C <= 512) LN_BWD(64, 1); else LN_BWD(64, 2); break;
        case 256: LN_BWD(256, 1); break;
        case 512: LN_BWD(512, 1); break;
        default: if (P.C <= 8192) LN_BWD(1024, 1); else LN_BWD(1024, 2); break;
    }
#undef LN_BWD
    return kp_check_launch("layer_norm_bwd");
}
template <int DT> int fwd_type(const LnFwd& P, int fmt, hipStream_t st) {
    if (!P.q) return fwd_launch<DT, 0>(P, st);
    if (fmt == KP_E4M3) return fwd_launch<DT, KP_E4M3>(P, st);
    return fwd_launch<DT, KP_E5M2>(P, st);
}
template <int DT> int bwd_type(const LnBwd& P, int fmt, int parts, hipStream_t st) {
    if (!P.q) return bwd_launch<DT, 0>(P, parts, st);
    if (fmt == KP_E4M3) return bwd_launch<DT, KP_E4M3>(P, parts, st);
    return bwd_launch<DT, KP_E5M2>(P, parts, st);
}

}  // namespace

extern "C" {

int kp_layer_norm_fwd(const void* x, long long ldx, const float* w, const float* b, float eps, void* y, long long ldy, float* mean,
                      float* rstd, unsigned char* q, unsigned char* s, int fmt, long long rows, long long C, int dtype, void* stream) {
    KP_REQUIRE(dtype == KP_F32 || dtype == KP_BF16 || dtype == KP_F16, "kp_layer_norm_fwd: unknown dtype %d", dtype);
    KP_REQUIRE(x && y && rows > 0 && C > 0 && (rows == 1 || (ldx >= C && ldy >= C)), "kp_layer_norm_fwd: bad args (%lld x %lld, strides %lld, %lld)", rows, C, ldx, ldy);
    KP_REQUIRE(C <= MOST, "kp_layer_norm_fwd: %lld columns are more than one call takes (2^30)", C);
    KP_REQUIRE(eps >= 0.f && !mean == !rstd && !q == !s && (!q || fmt == KP_E4M3 || fmt == KP_E5M2), "kp_layer_norm_fwd: mean with rstd, q with s, a known format, eps >= 0");
    LnFwd P{x, w, b, y, mean, rstd, q, s, ldx, ldy, rows, (int)C, (int)((C + Q8_BLOCK - 1) / Q8_BLOCK), eps};
    const hipStream_t st = (hipStream_t)stream;
    kp_count_bytes((double)rows * C * (2 * (dtype == KP_F32 ? 4 : 2) + (q ? 1 : 0)));
    return dtype == KP_F32 ? fwd_type<KP_F32>(P, fmt, st) : dtype == KP_BF16 ? fwd_type<KP_BF16>(P, fmt, st) : fwd_type<KP_F16>(P, fmt, st);
}

long long kp_layer_norm_bwd_ws_floats(long long rows, long long C) {
    return rows > 0 && C > 0 && C <= MOST ? ln_parts(rows, (int)C) * 2 * C : 0;
}

int kp_layer_norm_bwd(const void* dy, long long lddy, const void* x, long long ldx, const unsigned char* q, const unsigned char* s, int fmt,
                      const float* w, const float* mean, const float* rstd, void* dx, long long lddx, float* ws, float* dw, float* db,
                      long long rows, long long C, int dtype, void* stream) {
    KP_REQUIRE(dtype == KP_F32 || dtype == KP_BF16 || dtype == KP_F16, "kp_layer_norm_bwd: unknown dtype %d", dtype);
    KP_REQUIRE(dy && mean && rstd && (dx || dw || db) && rows > 0 && C > 0, "kp_layer_norm_bwd: bad args (%lld x %lld)", rows, C);
    KP_REQUIRE(C <= MOST, "kp_layer_norm_bwd: %lld columns are more than one call takes (2^30)", C);
    KP_REQUIRE(rows == 1 || (lddy >= C && (!dx || lddx >= C) && (!x || ldx >= C)), "kp_layer_norm_bwd: row strides %lld, %lld, %lld for %lld columns", lddy, ldx, lddx, C);
    KP_REQUIRE((x != nullptr) != (q != nullptr) && !q == !s && (!q || fmt == KP_E4M3 || fmt == KP_E5M2), "kp_layer_norm_bwd: either x or its 8-bit form");
    KP_REQUIRE(ws || !(dw || db), "kp_layer_norm_bwd: the weight's gradient needs a workspace (kp_layer_norm_bwd_ws_floats)");
    const int parts = ln_parts(rows, (int)C);
    LnBwd P{dy, x, q, s, w, mean, rstd, dx, (dw || db) ? ws : nullptr, lddy, ldx, lddx, rows, (int)C, (int)((C + Q8_BLOCK - 1) / Q8_BLOCK)};
    const hipStream_t st = (hipStream_t)stream;
    kp_count_bytes((double)rows * C * (2 * (dtype == KP_F32 ? 4 : 2) + (q ? 1 : (dtype == KP_F32 ? 4 : 2))));
    const int rc = dtype == KP_F32 ? bwd_type<KP_F32>(P, fmt, parts, st) : dtype == KP_BF16 ? bwd_type<KP_BF16>(P, fmt, parts, st) : bwd_type<KP_F16>(P, fmt, parts, st);
    if (rc != KP_OK || !(dw || db)) return rc;
    q8_join_k<<<cdiv(2 * C, 16), 1024, 0, st>>>(ws, parts, 2 * C, dw, C, db);
    return kp_check_launch("layer_norm_bwd join");
}

}  // extern "C"
