// Linear + softmax cross entropy over many classes, the logits not kept (but for few of them: lce_keeps), with its gradient.
//
//   z = x W^T + b  (T,V)     m_t = max_v z     s_t = sum_v exp(z - m_t)     lse_t = m_t + log s_t
//   loss_t = lse_t - (1 - e) z[t, y_t] - e mean_v z          (0 where y_t = ignore_index)
//   g = c_t (exp(z - m_t) / s_t - (1 - e) [v = y_t] - e / V),   c_t = dL/dloss_t        (0 where ignored)
//   dx = g W      dW = g^T x      db = sum_t g
//
// Forward: every tile of z reduces in registers to (max, sum of exponentials, sum) of its rows; a second launch joins the
// tiles of a row.  Backward: z is computed again, a piece of the vocabulary at a time; the piece's g (rounded once to the
// inputs' type, as the operand of the matrix instructions has to be) lives in a workspace of bounded size, and two products
// turn it into the piece's dW and its share of dx.  db sums g in float32, where it is made, before that rounding (a second
// walk over it took 28 us more of a piece of 6550 rows by 16,384 classes).  8 T D V operations for both directions
// where keeping T V logits takes 6: the price of not keeping them, which pays for 16 bits; float32's matrix rate makes keeping
// them the better way, up to 1 GB.
// Bound by the matrix cores for T in the hundreds and above, by reading W below.
// Rows whose target is ignored are left out of the products (from LCE_ROWS rows on): a list of the kept ones is made on
// the device, and the workgroups past them leave.
// float16 holds g times 2^15 (|g| <= 1: below 65504, and its normal range then reaches down to 2e-9, under 1/V); the
// coefficients c_t are scaled to at most 1 the same way; both factors come back in float32 on the way out.
// Measured (bf16; a large library product reaches 1250 TFLOP/s on this card): 6,550 kept rows of 8192, D 1024, V 100,000:
// statistics 1.33 ms = 1010 TFLOP/s; of each of 6 pieces g 268 us = 840, dx's product 279 us = 805, dW's 221 us (and 98 for
// the classes past its rounds) = 940, db 5 us: 5.75 - 5.9 ms by card.  float16 takes 4 % longer (1024 rows, D 1024, 50,000
// classes: 535 and 514 us).  No LDS bank conflict; of the statistics' time the epilogue is 17 %; rows of x or W other than a
// power of two apart change nothing (1480 us at 1024 and at 1088 elements, all rows).  64 rows, D 256, V 6500, float32: eight
// launches of 3 to 13 us.
#include <algorithm>

#include "pngpd_lce_gemm.h"

#define LCE_PIECE_BYTES (256ll << 20)      // a piece's g
#define LCE_PIECE_MOST (1ll << 30)         // where a round of dW's large tiles over the CUs takes more

#define LCE_ROWS 512                       // below, dropping rows does not drop enough tiles to pay for the list's launch
#define LOG2E 1.44269504088896340736f

// Where the kept rows lie: [0] how many, [1 ..] their row, [1 + T ..] a row's place among them or -1.  NULL: all, in order.
struct LceRows {
    const int *p;
    int T;
    __device__ __forceinline__ int count() const { return p ? p[0] : T; }
    __device__ __forceinline__ const int *list() const { return p ? p + 1 : nullptr; }
    __device__ __forceinline__ int row(int k) const { return p ? p[1 + k] : k; }
    __device__ __forceinline__ int place(int t) const { return p ? p[1 + T + t] : t; }
};

struct LceArgs {
    LceOperand x, w;                       // rows of 16-byte multiples
    LceRows rows;
    int packed;                            // x holds the kept rows only
    const void *bias;
    int bf32;
    const long long *target;
    long long ignore;
    int T, D, V, mt, mt0;                  // mt: tiles of classes of a launch (lce_join_kernel: of all), mt0: those before
    float smooth;
    float *pm, *ps, *zt;                   // forward: (mt,T,2) max / sum, (mt,T) sum of z, (T) z at the target
    const float *stat, *coef;              // backward: (T,2) max / sum, (T)
    float *z;                              // (T, ldz) the logits kept for the backward pass, or NULL
    int ldz;
    void *g;
    float *db;                             // (tiles of rows, ldg): column sums of g's rows, before it is rounded, or NULL
    int v0, vc, ldg;                       // the launch's classes (g and db start at the first one)
};                                         // (T above, but for target: by place among the kept rows)

// The kept rows in order: 8 targets a thread and round, the places by a scan over the workgroup.
__global__ __launch_bounds__(1024) void lce_rows_kernel(const long long *__restrict__ target, long long ignore, int T,
                                                        int *__restrict__ rows) {
    __shared__ int sh[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int base = 0;
    for (int t0 = 0; t0 < T; t0 += 8192) {
        const int t = t0 + threadIdx.x * 8;
        unsigned keep = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) if (t + e < T && target[t + e] != ignore) keep |= 1u << e;
        const int n = __popc(keep);
        int at = n;
#pragma unroll
        for (int k = 1; k < 64; k <<= 1) { const int u = __shfl_up(at, k); if (lane >= k) at += u; }
        __syncthreads();
        if (lane == 63) sh[wave] = at;
        __syncthreads();
        int before = base, all = 0;
        for (int w = 0; w < 16; ++w) { if (w < wave) before += sh[w]; all += sh[w]; }
        int k = before + at - n;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (t + e < T) {
                const bool on = keep >> e & 1;
                rows[1 + T + t + e] = on ? k : -1;
                if (on) rows[1 + k++] = t + e;
            }
        }
        base += all;
    }
    if (threadIdx.x == 0) rows[0] = base;
}

// four values of column pairs q, q + 1 of a lane and of its partner in the other half: the lane of half h is given the
// eight consecutive ones of q + h
__device__ __forceinline__ uint4 lce_pair(uint2 x, uint2 y) {
    const auto a = __builtin_amdgcn_permlane32_swap(x.x, y.x, false, false);
    const auto b = __builtin_amdgcn_permlane32_swap(x.y, y.y, false, false);
    return make_uint4(a[0], b[0], a[1], b[1]);
}
template <int DT> __device__ __forceinline__ uint2 lce_half4(float a, float b, float c, float d) {
    return make_uint2(pk_half<DT>(a, b), pk_half<DT>(c, d));
}

// 2^((z - m) log2 e) is one FMA, z log2 e - (m log2 e), where the rounding of the product in brackets is small: an error of
// 2^-24 |m| in the exponent, so for maxima up to 64 (2^-18) and 16-bit inputs; otherwise the difference is taken first
// (a row of classes masked by the type's lowest value, large logits, float32).
template <int DT> __device__ __forceinline__ bool lce_far(float m) { return DT == PNGPD_F32 || fabsf(m) > 64.f; }

// (max, sum) of two parts of a row; a part without values is (-inf, 0)
__device__ __forceinline__ void lce_join(float &m, float &s, float m2, float s2) {
    const float M = fmaxf(m, m2), ref = M == -INFINITY ? 0.f : M;
    s = s * __expf(m - ref) + s2 * __expf(m2 - ref);
    m = M;
}

// What the epilogue of a tile needs beside the accumulators, fetched ahead of its loads and kept in LDS: a load issued
// behind the next tile's would wait for those.  v: bias (both); n: target's place among the tile's classes or -1, and
// for the gradient m log2 e, c/s, c e/V, c (or -m, where the difference is taken first: lce_far).
template <int BM, int BN> struct LceSide {
    float bias[BM];
    int rel[BN];
    float m[BN], ks[BN], kf[BN], co[BN];
};

template <int DT, int BM, int BN, int THREADS>
__device__ __forceinline__ void lce_side(const LceArgs &a, LceSide<BM, BN> *s, int v0, int m0, int n0, int T, bool grad) {
    typedef typename elem<DT>::t E;
    for (int i = threadIdx.x; i < BM; i += THREADS) {
        const int v = min(v0 + m0 + i, a.V - 1);
        s->bias[i] = !a.bias ? 0.f : a.bf32 ? ((const float *)a.bias)[v] : ld_elem<DT>((const E *)a.bias + v);
    }
    for (int i = threadIdx.x; i < BN; i += THREADS) {
        const int k = n0 + i;
        int rel = -2;                                             // -2: no row, or an ignored one
        float m = 0.f, sum = 1.f, co = 0.f;
        if (k < T) {
            const long long y = a.target[a.rows.row(k)];
            if (y != a.ignore) rel = y >= (long long)v0 + m0 && y < (long long)v0 + m0 + BM && y < a.V ? (int)(y - v0 - m0) : -1;
            if (grad) { m = a.stat[2 * (size_t)k]; sum = a.stat[2 * (size_t)k + 1]; co = a.coef[k]; }
        }
        s->rel[i] = rel;
        if (grad) { s->m[i] = m; s->ks[i] = co / sum; s->kf[i] = co * (a.smooth / (float)a.V); s->co[i] = co; }
    }
}

// The epilogues cost vector instructions that the matrix pipe waits for (128 values a lane of the large tile): what only
// some tiles need (the target's logit, classes past V, smoothing) is asked once a wave, and an exponential is one FMA and
// one v_exp_f32.  A workgroup walks over tiles: the next one's loads run under the epilogue.
template <int DT, int BM, int BN, int WGM, int WGN, int PIPE>
__global__ __launch_bounds__(WGM * WGN * 64, 2) void lce_stats_kernel(const LceArgs a) {
    typedef LceCore<DT, false, false, BM, BN, WGM, WGN, PIPE> Core;
    typedef LceSide<BM, BN> Side;
    extern __shared__ __align__(16) char smem[];
    Side *side = (Side *)(smem + Core::LDS);
    float *sh = (float *)(side + 2);                              // [WGM][BN][3]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int wm = (wave % WGM) * Core::WM, wn = (wave / WGM) * Core::WN;
    const int T = a.rows.count(), nt = (T + BN - 1) / BN, total = a.mt * nt;
    const int *list = a.packed ? nullptr : a.rows.list();
    int at = blockIdx.x, tm, tn, flip = 0;
    if (at >= total) return;
    LceOperand w = a.w;
    w.p = (const typename elem<DT>::t *)a.w.p + (long long)a.v0 * a.w.ld;
    Core c;
    lce_tile_of(at, a.mt, nt, tm, tn);
    lce_side<DT, BM, BN, Core::THREADS>(a, side, a.v0, tm * BM, tn * BN, T, false);
    c.start(smem, w, a.x, list, tm * BM, a.vc, tn * BN, T, 0, a.D);
    while (true) {
        const int m0 = tm * BM, n0 = tn * BN, here = a.mt0 + tm;
        c.finish(smem, w.ld, a.x.ld);
        const Side *s = side + flip;
        at += gridDim.x; flip ^= 1;
        if (at < total) {
            lce_tile_of(at, a.mt, nt, tm, tn);
            lce_side<DT, BM, BN, Core::THREADS>(a, side + flip, a.v0, tm * BM, tn * BN, T, false);
            c.start(smem, w, a.x, list, tm * BM, a.vc, tn * BN, T, 0, a.D);
        }
        const int vl = wm + 4 * half;                             // the lane's row 0 in the tile
        if (a.bias) {
#pragma unroll
            for (int i = 0; i < Core::FM; ++i) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const f32x4 b = *(const f32x4 *)(s->bias + vl + 32 * i + 8 * q);
#pragma unroll
                    for (int j = 0; j < Core::FN; ++j) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) c.acc[i][j][4 * q + e] += b[e];
                    }
                }
            }
        }
        const bool whole = m0 + BM <= a.vc;
#pragma unroll
        for (int j = 0; j < Core::FN; ++j) {
            const int col = wn + 32 * j + (lane & 31), k = n0 + col, rel = s->rel[col], mine = rel - vl;
            if constexpr (DT == PNGPD_F32 || BM < 256) {          // (lce_keeps: of 16 bits not with the large tile)
                if (a.z && k < T) {
                    float *z = a.z + (size_t)k * a.ldz + a.v0 + m0 + vl;
#pragma unroll
                    for (int i = 0; i < Core::FM; ++i) {
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            *(f32x4 *)(z + 32 * i + 8 * q) = f32x4{c.acc[i][j][4 * q], c.acc[i][j][4 * q + 1],
                                                                   c.acc[i][j][4 * q + 2], c.acc[i][j][4 * q + 3]};
                    }
                }
            }
            if (__any(mine >= 0 && mine < Core::WM)) {
                float z = 0.f;
                bool found = false;                               // (the other half has the other rows of four)
#pragma unroll
                for (int i = 0; i < Core::FM; ++i) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const bool it = mine == 32 * i + (r & 3) + 8 * (r >> 2);
                        z = it ? c.acc[i][j][r] : z;
                        found |= it;
                    }
                }
                if (found) a.zt[k] = z;
            }
            float sz = 0.f;
            if (whole) {
                if (a.smooth != 0.f) {
#pragma unroll
                    for (int i = 0; i < Core::FM; ++i) {
#pragma unroll
                        for (int r = 0; r < 16; ++r) sz += c.acc[i][j][r];
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < Core::FM; ++i) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const bool past = m0 + vl + 32 * i + (r & 3) + 8 * (r >> 2) >= a.vc;
                        sz += past ? 0.f : c.acc[i][j][r];
                        c.acc[i][j][r] = past ? -INFINITY : c.acc[i][j][r];
                    }
                }
            }
            sz = half_sum(sz);
            float m = -INFINITY, e = 0.f;
#pragma unroll
            for (int i = 0; i < Core::FM; ++i) {
#pragma unroll
                for (int r = 0; r < 16; r += 2) m = max3f(m, c.acc[i][j][r], c.acc[i][j][r + 1]);
            }
            float lo, hi;
            half_pair(m, lo, hi);
            m = fmaxf(lo, hi);
            const float mf = m == -INFINITY ? 0.f : m;
            if (__any(lce_far<DT>(m) && rel != -2)) {             // (not for what an ignored row holds: the others' bits stay)
#pragma unroll
                for (int i = 0; i < Core::FM; ++i) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) e += __builtin_amdgcn_exp2f((c.acc[i][j][r] - mf) * LOG2E);
                }
            } else {
                const float ref = mf * LOG2E;
#pragma unroll
                for (int i = 0; i < Core::FM; ++i) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) e += __builtin_amdgcn_exp2f(fmaf(c.acc[i][j][r], LOG2E, -ref));
                }
            }
            e = half_sum(e);
            if (half == 0) {
                float *o = sh + ((wave % WGM) * BN + col) * 3;
                o[0] = m; o[1] = e; o[2] = sz;
            }
        }
        lce_lds_barrier();
        for (int col = threadIdx.x; col < BN; col += Core::THREADS) {
            const int k = n0 + col;
            if (k >= T) continue;
            float m = sh[col * 3], e = sh[col * 3 + 1], sz = sh[col * 3 + 2];
#pragma unroll
            for (int w = 1; w < WGM; ++w) {
                const float *o = sh + (w * BN + col) * 3;
                lce_join(m, e, o[0], o[1]);
                sz += o[2];
            }
            const size_t to = (size_t)here * a.T + k;
            *(f32x2 *)(a.pm + 2 * to) = f32x2{m, e};
            if (a.smooth != 0.f) a.ps[to] = sz;
        }
        if (at >= total) return;
    }
}

// One row a group of 32 lanes: joins its tiles, in fp64; stat (T,2) = max, sum of the kept rows; row (T) = every row's loss.
// A grid of one workgroup (few rows) walks over all of them and goes on to the loss.
#define LCE_FEW 64
__device__ __forceinline__ double lce_block_sum(double v, double *sh) {
    for (int k = 32; k >= 1; k >>= 1) v += __shfl_xor(v, k);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0.0;
    for (int k = 0; k < (int)(blockDim.x >> 6); ++k) s += sh[k];
    return s;
}

// kept rows; loss = their sum or mean (a mean over none is NaN)
__device__ __forceinline__ void lce_loss(const float *row, const LceArgs &a, int reduction, float *loss, float *kept) {
    __shared__ double sh[16];
    double s = 0.0, n = 0.0;
#pragma unroll 4
    for (int t = threadIdx.x; t < a.T; t += blockDim.x) {
        if (a.target[t] != a.ignore) n += 1.0;
        s += (double)row[t];
    }
    s = lce_block_sum(s, sh);
    n = lce_block_sum(n, sh);
    if (threadIdx.x == 0) {
        *kept = (float)n;
        if (reduction == PNGPD_REDUCE_MEAN) *loss = (float)(s / n);
        if (reduction == PNGPD_REDUCE_SUM) *loss = (float)s;
    }
}
__global__ __launch_bounds__(1024) void lce_loss_kernel(const LceArgs a, const float *row, int reduction, float *loss, float *kept) {
    lce_loss(row, a, reduction, loss, kept);
}

// ROWS rows a workgroup and turn
template <int ROWS>
__global__ __launch_bounds__(ROWS * 32) void lce_join_kernel(const LceArgs a, float *stat, float *row, int reduction, float *loss,
                                                             float *kept) {
    __shared__ double sh[32][ROWS][2];
    __shared__ float shm[32][ROWS];
    const int tx = threadIdx.x % ROWS, ty = threadIdx.x / ROWS;
    for (int t0 = blockIdx.x * ROWS; t0 < a.T; t0 += gridDim.x * ROWS) {
        const int t = t0 + tx, place = t < a.T ? a.rows.place(t) : -1;
        float m = -INFINITY;
        double s = 0.0, sz = 0.0;
        if (place >= 0) {
#pragma unroll 4
            for (int k = ty; k < a.mt; k += 32) {
                const size_t at = (size_t)k * a.T + place;
                const f32x2 p = *(const f32x2 *)(a.pm + 2 * at);
                const float M = fmaxf(m, p[0]), ref = M == -INFINITY ? 0.f : M;
                s = s * (double)expf(m - ref) + (double)p[1] * (double)expf(p[0] - ref);
                m = M;
                if (a.smooth != 0.f) sz += (double)a.ps[at];
            }
        }
        __syncthreads();                                          // (the turn before has read its parts)
        shm[ty][tx] = m; sh[ty][tx][0] = s; sh[ty][tx][1] = sz;
        __syncthreads();
        // the other way round: a row's 32 parts in 32 lanes
        const int lane = threadIdx.x & 31, u = t0 + threadIdx.x / 32, at = u < a.T ? a.rows.place(u) : -1;
        m = shm[lane][threadIdx.x / 32]; s = sh[lane][threadIdx.x / 32][0]; sz = sh[lane][threadIdx.x / 32][1];
        float M = m;
#pragma unroll
        for (int k = 16; k >= 1; k >>= 1) M = fmaxf(M, __shfl_xor(M, k));
        s *= (double)expf(m - (M == -INFINITY ? 0.f : M));
#pragma unroll
        for (int k = 16; k >= 1; k >>= 1) { s += __shfl_xor(s, k); sz += __shfl_xor(sz, k); }
        if (lane || u >= a.T) continue;
        if (at < 0) { row[u] = 0.f; continue; }
        stat[2 * (size_t)at] = M; stat[2 * (size_t)at + 1] = (float)s;
        const long long y = a.target[u];
        double l = 0.0;
        if (y != a.ignore) {
            if (y < 0 || y >= a.V) l = NAN;                        // a class that does not exist: as loud as a value can be
            else {
                // differences from the maximum first: beside a maximum of 1e30 the logarithm would be lost
                l = log(s) + (1.0 - (double)a.smooth) * ((double)M - (double)a.zt[at]);
                if (a.smooth != 0.f) l += (double)a.smooth * ((double)M - sz / a.V);
            }
        }
        row[u] = (float)l;
    }
    if (gridDim.x == 1) {
        __threadfence_block();
        __syncthreads();
        lce_loss(row, a, reduction, loss, kept);
    }
}

struct LceCoef {
    const float *dloss, *kept;
    const long long *target;
    long long ignore;
    LceRows rows;
    int V, reduction;
    float up;
    float *coef, *scale;
};
// coef (T) = c_t over the largest finite |c_t| (times up, the factor of the type's range), scale = what gives c_t back.  One
// workgroup of 256.
__device__ __forceinline__ void lce_coef(const LceCoef &a) {
    __shared__ float sh[4];
    const int T = a.rows.T;
    float top = 1.f;
    if (a.reduction == PNGPD_REDUCE_NONE) {
        top = 0.f;
#pragma unroll 8
        for (int t = threadIdx.x; t < T; t += 256) {
            const float c = fabsf(a.dloss[t]);
            if (c < INFINITY && a.target[t] != a.ignore) top = fmaxf(top, c);
        }
        for (int k = 32; k >= 1; k >>= 1) top = fmaxf(top, __shfl_xor(top, k));
        if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = top;
        __syncthreads();
        top = fmaxf(fmaxf(sh[0], sh[1]), fmaxf(sh[2], sh[3]));
        if (top == 0.f) top = 1.f;
    }
    for (int t0 = threadIdx.x; t0 < T; t0 += 8 * 256) {           // eight rows' loads at a time: one workgroup has all of them
        long long y[8];
        float c[8];
        int k[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int t = min(t0 + 256 * i, T - 1);
            y[i] = a.target[t]; k[i] = a.rows.place(t);
            c[i] = a.reduction == PNGPD_REDUCE_NONE ? a.dloss[t] : 1.f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float v = y[i] == a.ignore ? 0.f : y[i] < 0 || y[i] >= a.V ? NAN : c[i] / top * a.up;
            if (t0 + 256 * i < T && k[i] >= 0) a.coef[k[i]] = v;
        }
    }
    if (threadIdx.x == 0) {
        float s = top / a.up;
        if (a.reduction == PNGPD_REDUCE_SUM) s = *a.dloss / a.up;
        if (a.reduction == PNGPD_REDUCE_MEAN) s = *a.kept > 0.f ? *a.dloss / *a.kept / a.up : 0.f;    // no row, no gradient
        *a.scale = s;
    }
}

// one step of a sum over lanes that spreads the values over them: of N values a lane keeps half, and adds its partner's
template <int N> __device__ __forceinline__ void lce_spread(float (&v)[16], int lane, int k) {
    const bool up = lane & k;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        const float keep = up ? v[N / 2 + i] : v[i], send = up ? v[i] : v[N / 2 + i];
        v[i] = keep + __shfl_xor(send, k);
    }
}

template <int DT, int BM, int BN, int WGM, int WGN, int PIPE>
__global__ __launch_bounds__(WGM * WGN * 64, 2) void lce_grad_kernel(const LceArgs a) {
    typedef LceCore<DT, false, false, BM, BN, WGM, WGN, PIPE> Core;
    typedef LceSide<BM, BN> Side;
    typedef typename elem<DT>::t E;
    extern __shared__ __align__(16) char smem[];
    Side *side = (Side *)(smem + Core::LDS);
    float *sh = (float *)(side + 2);                              // [WGN][BM]
    static_assert(WGN * BM * 4 <= WGM * BN * 12, "the room that lce_z_shape allows for");
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int wm = (wave % WGM) * Core::WM, wn = (wave / WGM) * Core::WN;
    const int T = a.rows.count(), nt = (T + BN - 1) / BN, total = a.mt * nt;
    LceOperand w = a.w;
    w.p = (const E *)a.w.p + (long long)a.v0 * a.w.ld;
    int at = blockIdx.x, tm, tn, flip = 0;
    if (at >= total) return;
    Core c;
    lce_tile_of(at, a.mt, nt, tm, tn);
    lce_side<DT, BM, BN, Core::THREADS>(a, side, a.v0, tm * BM, tn * BN, T, true);
    c.start(smem, w, a.x, nullptr, tm * BM, a.vc, tn * BN, T, 0, a.D);
    while (true) {
        const int m0 = tm * BM, n0 = tn * BN;
        c.finish(smem, w.ld, a.x.ld);
        const Side *s = side + flip;
        at += gridDim.x; flip ^= 1;
        if (at < total) {
            lce_tile_of(at, a.mt, nt, tm, tn);
            lce_side<DT, BM, BN, Core::THREADS>(a, side + flip, a.v0, tm * BM, tn * BN, T, true);
            c.start(smem, w, a.x, nullptr, tm * BM, a.vc, tn * BN, T, 0, a.D);
        }
        const int vl = wm + 4 * half;                             // the lane's row 0 in the tile
        if (a.bias) {
#pragma unroll
            for (int i = 0; i < Core::FM; ++i) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const f32x4 b = *(const f32x4 *)(s->bias + vl + 32 * i + 8 * q);
#pragma unroll
                    for (int j = 0; j < Core::FN; ++j) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) c.acc[i][j][4 * q + e] += b[e];
                    }
                }
            }
        }
        const bool whole = m0 + BM <= a.vc;
#pragma unroll
        for (int j = 0; j < Core::FN; ++j) {
            const int col = wn + 32 * j + (lane & 31), k = n0 + col, mine = s->rel[col] - vl;
            const float m = s->m[col], ks = s->ks[col], kf = s->kf[col], co = s->co[col];
            float ref = m * LOG2E;
            if (__any(lce_far<DT>(m) && co != 0.f)) {
                ref = 0.f;
#pragma unroll
                for (int i = 0; i < Core::FM; ++i) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) c.acc[i][j][r] -= m;
                }
            }
#pragma unroll
            for (int i = 0; i < Core::FM; ++i) {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    c.acc[i][j][r] = fmaf(__builtin_amdgcn_exp2f(fmaf(c.acc[i][j][r], LOG2E, -ref)), ks, -kf);
            }
            if (__any(mine >= 0 && mine < Core::WM)) {
                const float hit = co * (1.f - a.smooth);
#pragma unroll
                for (int i = 0; i < Core::FM; ++i) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) c.acc[i][j][r] -= mine == 32 * i + (r & 3) + 8 * (r >> 2) ? hit : 0.f;
                }
            }
            // rows without a weight (ignored ones that are still here among them) have no gradient, whatever they hold
            const bool none = co == 0.f;
            if (__any(none) || !whole) {
#pragma unroll
                for (int i = 0; i < Core::FM; ++i) {
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        c.acc[i][j][r] = none || m0 + vl + 32 * i + (r & 3) + 8 * (r >> 2) >= a.vc ? 0.f : c.acc[i][j][r];
                }
            }
            if (k < T) {                                          // (alike in both halves: lce_pair's lanes stay together)
                E *g = (E *)a.g + (size_t)k * a.ldg + m0 + wm;
#pragma unroll
                for (int i = 0; i < Core::FM; ++i) {
                    const f32x16 &v = c.acc[i][j];
                    if constexpr (DT == PNGPD_F32) {
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            *(f32x4 *)(g + 32 * i + 8 * q + 4 * half) = f32x4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
                    } else {
#pragma unroll
                        for (int q = 0; q < 4; q += 2)
                            *(uint4 *)(g + 32 * i + 8 * (q + half)) =
                                lce_pair(lce_half4<DT>(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]),
                                         lce_half4<DT>(v[4 * q + 4], v[4 * q + 5], v[4 * q + 6], v[4 * q + 7]));
                    }
                }
            }
        }
        // db's share of the tile, in float32 whatever g is stored in: a row's 16 values of 32 lanes end up one a lane pair
        if (a.db) {
#pragma unroll
            for (int i = 0; i < Core::FM; ++i) {
                float v[16];
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    v[r] = c.acc[i][0][r];
#pragma unroll
                    for (int j = 1; j < Core::FN; ++j) v[r] += c.acc[i][j][r];
                }
                lce_spread<16>(v, lane, 16); lce_spread<8>(v, lane, 8); lce_spread<4>(v, lane, 4); lce_spread<2>(v, lane, 2);
                const float u = v[0] + __shfl_xor(v[0], 1);
                const int r = (lane & 31) >> 1;
                if (!(lane & 1)) sh[(wave / WGM) * BM + vl + 32 * i + (r & 3) + 8 * (r >> 2)] = u;
            }
            lce_lds_barrier();
            for (int m = threadIdx.x; m < BM; m += Core::THREADS) {
                float u = sh[m];
#pragma unroll
                for (int k = 1; k < WGN; ++k) u += sh[k * BM + m];
                a.db[(size_t)(n0 / BN) * a.ldg + m0 + m] = u;
            }
        }
        if (at >= total) return;
    }
}

// lce_grad_kernel's epilogue on kept logits: four classes a thread, 1024 of `share` rows a workgroup.
template <int DT>
__global__ __launch_bounds__(256) void lce_kept_grad_kernel(const LceArgs a, int cols, int share) {
    typedef typename elem<DT>::t E;
    const int per = (cols + 1023) / 1024, part = blockIdx.x / per, v = (blockIdx.x - part * per) * 1024 + threadIdx.x * 4;
    const int k0 = part * share, k1 = min(a.rows.count(), k0 + share);
    if (k0 >= k1 || v >= cols) return;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
    for (int k = k0; k < k1; ++k) {
        const float m = a.stat[2 * (size_t)k], co = a.coef[k], ks = co / a.stat[2 * (size_t)k + 1], kf = co * (a.smooth / (float)a.V);
        const long long y = a.target[a.rows.row(k)] - a.v0;       // (an ignored row's co is 0)
        const f32x4 z = *(const f32x4 *)(a.z + (size_t)k * a.ldz + a.v0 + v);
        f32x4 g;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float p = __builtin_amdgcn_exp2f(lce_far<DT>(m) ? (z[e] - m) * LOG2E : fmaf(z[e], LOG2E, -(m * LOG2E)));
            g[e] = fmaf(p, ks, -kf) - (y == v + e ? co * (1.f - a.smooth) : 0.f);
            if (co == 0.f || v + e >= a.vc) g[e] = 0.f;
        }
        E *o = (E *)a.g + (size_t)k * a.ldg + v;
        if constexpr (DT == PNGPD_F32) *(f32x4 *)o = g;
        else *(uint2 *)o = lce_half4<DT>(g[0], g[1], g[2], g[3]);
        sum += g;
    }
    if (a.db) *(f32x4 *)(a.db + (size_t)part * a.ldg + v) = sum;
}

// db of a piece: the sums (S, ldg) joined in fp64, 32 classes by 8 of the S a workgroup.  A sum is of `rows0` kept rows, from
// class `cut` on of `rows1`.
template <int DT>
__global__ __launch_bounds__(256) void lce_db_join_kernel(const float *__restrict__ part, LceRows rows, int rows0, int cut, int rows1,
                                                          int ldg, int vc, const float *__restrict__ scale, void *__restrict__ db,
                                                          int f32) {
    __shared__ double sh[8][32];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, v = blockIdx.x * 32 + tx, per = v < cut ? rows0 : rows1;
    const int S = (rows.count() + per - 1) / per;
    double s = 0.0;
    if (v < vc) {
#pragma unroll 8
        for (int k = ty; k < S; k += 8) s += (double)part[(size_t)k * ldg + v];
    }
    sh[ty][tx] = s;
    __syncthreads();
    if (ty || v >= vc) return;
    for (int k = 1; k < 8; ++k) s += sh[k][tx];
    const float o = (float)(s * (double)*scale);
    if (f32) ((float *)db)[v] = o;
    else st_elem<DT>((typename elem<DT>::t *)db + v, o);
}

struct LceOut {
    LceOperand a, b;
    LceRows rows;                          // counts N (dx) or K (dW)
    int M, N, mt, nt;                      // M: m that exist in a's rows (padded); N likewise, -1: the kept rows
    int mo, no;                            // outputs stored (no: N = -1's are the kept rows)
    long long K, kper;                     // k (-1: the kept rows), k of a split
    int splits;
    void *out;                             // typed: out[n * ldo + m] = scale * sum
    long long ldo;
    float *part;                           // or fp32 partial sums (splits, pn, M), added to what is there
    int pn;
    int add;
    const float *scale;
    int vec;                               // out's rows are whole 16-byte chunks
};

template <int DT, bool BMC, int BM, int BN, int WGM, int WGN, int PIPE>
__global__ __launch_bounds__(WGM * WGN * 64, 2) void lce_out_kernel(const LceOut a) {
    typedef LceCore<DT, true, BMC, BM, BN, WGM, WGN, PIPE> Core;
    typedef typename elem<DT>::t E;
    extern __shared__ __align__(16) char smem[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int wm = (wave % WGM) * Core::WM, wn = (wave / WGM) * Core::WN;
    const int N = a.N < 0 ? a.rows.count() : a.N, no = a.N < 0 ? N : a.no, nt = a.N < 0 ? (N + BN - 1) / BN : a.nt;
    const long long K = a.K < 0 ? a.rows.count() : a.K;
    const int tiles = a.mt * nt;
    if ((int)blockIdx.x >= tiles * a.splits) return;
    const int split = blockIdx.x / tiles;
    int tm, tn;
    lce_tile_of(blockIdx.x - split * tiles, a.mt, nt, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;
    const long long k0 = split * a.kper, k1 = k0 + a.kper < K ? k0 + a.kper : K;
    Core c;
    c.start(smem, a.a, a.b, nullptr, m0, a.M, n0, N, k0, k1);
    c.finish(smem, a.a.ld, a.b.ld);
    const float sc = a.part ? 1.f : *a.scale;
#pragma unroll
    for (int j = 0; j < Core::FN; ++j) {
        const int n = n0 + wn + 32 * j + (lane & 31);
        if (n >= no) continue;
#pragma unroll
        for (int i = 0; i < Core::FM; ++i) {
            f32x16 v = c.acc[i][j];
            const int mb = m0 + wm + 32 * i;
            if (a.part) {
                float *o = a.part + ((size_t)split * a.pn + n) * a.M + mb + 4 * half;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    if (mb + 8 * q + 4 * half < a.M) {
                        const f32x4 u = {v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
                        f32x4 *at = (f32x4 *)(o + 8 * q);
                        *at = a.add ? *at + u : u;
                    }
                }
                continue;
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) v[r] *= sc;
            E *o = (E *)a.out + n * a.ldo + mb;
            if (a.vec && mb + 32 <= a.mo) {
                if constexpr (DT == PNGPD_F32) {
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        *(f32x4 *)(o + 8 * q + 4 * half) = f32x4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
                } else {
#pragma unroll
                    for (int q = 0; q < 4; q += 2)
                        *(uint4 *)(o + 8 * (q + half)) = lce_pair(lce_half4<DT>(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]),
                                                                  lce_half4<DT>(v[4 * q + 4], v[4 * q + 5], v[4 * q + 6], v[4 * q + 7]));
                }
            } else {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int m = (r & 3) + 8 * (r >> 2) + 4 * half;
                    if (mb + m < a.mo) st_elem<DT>(o + m, v[r]);
                }
            }
        }
    }
}

// dx (or dW) = scale * sum of the splits' partial sums (rows of Dp, a multiple of 4); 0 where a row is not among the kept
template <int DT>
__global__ __launch_bounds__(256) void lce_dx_kernel(const float *__restrict__ part, int splits, LceRows rows, int D, int Dp,
                                                     const float *__restrict__ scale, void *__restrict__ dx) {
    typedef typename elem<DT>::t E;
    const int per = Dp / 4;
    const long long q = (long long)blockIdx.x * 256 + threadIdx.x;
    if (q >= (long long)rows.T * per) return;
    const long long t = q / per;
    const int d = (int)(q - t * per) * 4, k = rows.place((int)t);
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (k >= 0) {
#pragma unroll 8
        for (int s = 0; s < splits; ++s) v += *(const f32x4 *)(part + ((size_t)s * rows.T + k) * Dp + d);
    }
    const float sc = *scale;
    E *o = (E *)dx + t * D + d;
#pragma unroll
    for (int e = 0; e < 4; ++e) if (d + e < D) st_elem<DT>(o + e, k < 0 ? 0.f : v[e] * sc);
}

// dst (R,Dp) = src (R,D) with zeros behind; with `mask` the kept rows only, in their places (all of them, in order: a row
// of zeros where the target is ignored — what such a row holds is nobody's, a NaN there must not meet g's zeros in a
// product).  One 16-byte chunk of dst a thread.  coef.coef: the first workgroup makes the coefficients in its place.
template <int DT>
__global__ __launch_bounds__(256) void lce_copy_kernel(const void *__restrict__ src, long long ld, int D, int Dp, long long R,
                                                       int mask, LceRows rows, const long long *__restrict__ target,
                                                       long long ignore, void *__restrict__ dst, const LceCoef coef) {
    typedef typename elem<DT>::t E;
    constexpr int EPC = 16 / (int)sizeof(E);
    const int per = Dp / EPC, first = coef.coef ? 1 : 0;
    if (first && blockIdx.x == 0) { lce_coef(coef); return; }
    const long long q = (long long)(blockIdx.x - first) * 256 + threadIdx.x;
    if (q >= R * per) return;
    const long long k = q / per;
    const int d = (int)(q - k * per) * EPC;
    if (mask && k >= rows.count()) return;
    const long long r = mask ? rows.row((int)k) : k;
    const E *s = (const E *)src + r * ld + d;
    __align__(16) E v[EPC];
#pragma unroll
    for (int e = 0; e < EPC; ++e) v[e] = (E)0;
    if (!mask || rows.p || target[r] != ignore) {
        if (d + EPC <= D) __builtin_memcpy(v, s, 16);
        else {
#pragma unroll
            for (int e = 0; e < EPC; ++e) if (d + e < D) v[e] = s[e];
        }
    }
    *(uint4 *)((E *)dst + k * Dp + d) = *(const uint4 *)v;
}

// ---------------------------------------------------------------------------------------------------- host
typedef pngpd_lce_t Lce;
static inline size_t lce_up(size_t n) { return (n + 255) & ~(size_t)255; }
static inline int lce_esize(int dt) { return dt == PNGPD_F32 ? 4 : 2; }
static inline int lce_dp(const Lce *a) { const int c = 16 / lce_esize(a->dtype); return (a->D + c - 1) / c * c; }
// rows that the loads can take as they are: 16-byte aligned, D a whole number of chunks, and `reach` of them within the
// 4 GiB of a lane's offset (a tile's 256, or all where the kept rows are picked out of them; copied, they are packed, and
// LCE_MOST_D keeps a tile's within)
#define LCE_MOST_D (1 << 22)
static inline bool lce_plain(const Lce *a, const void *p, long long ld, long long reach) {
    const int es = lce_esize(a->dtype);
    return lce_dp(a) == a->D && !((uintptr_t)p & 15) && (ld * es) % 16 == 0 && (double)ld * es * (double)reach < 4e9;
}

// tile shapes: 0 = 256 x 256, 1 = 64 x 64, 2 = 64 x 32, 3 = 128 x 128
static const int LCE_BM[4] = {256, 64, 64, 128}, LCE_BN[4] = {256, 64, 32, 128};
#define LCE_SHAPE0 256, 256, 2, 4, 2
#define LCE_SHAPE1 64, 64, 2, 2, 4
#define LCE_SHAPE2 64, 32, 2, 1, 5
#define LCE_SHAPE3 128, 128, 2, 2, 2
static inline int lce_cdiv(long long a, int b) { return (int)((a + b - 1) / b); }
// An operation takes 0.4 of the 64 x 64 tile's time in 256 x 256 tiles and 0.75 in 128 x 128 ones, where they fill their rounds of
// the 256 CUs and are not mostly padding (forward + backward of 1024 rows, D 2048, 12,000 classes, bf16: 296 us in 128 x 128
// tiles, 381 in 64 x 64; 1024 rows, D 1024, 5000 classes, float32, 320 tiles of 128 or 1264 of 64: 536 and 443).  least: large
// tiles at least.  The narrow tile is for rows that would leave half of 64 unused.
static int lce_shape(long long M, long long N, int least = 256) {
    if (N <= 32) return 2;
    const auto tiles = [&](int n) { return (long long)lce_cdiv(M, n) * lce_cdiv(N, n); };
    const auto whole = [&](int n) { return (tiles(n) + 255) / 256 * 256; };
    const long long large = 32 * whole(256), mid = 15 * whole(128), small = 5 * tiles(64);
    if (tiles(256) >= least && large <= mid && large <= small) return 0;
    return mid <= small ? 3 : 1;
}

// Of `n` classes, those that the large tile takes: whole rounds of 256 workgroups (one a CU) of `other` tiles each.  What is
// left of a round goes to the 64 x 64 tile where it is less than 0.4 of one: that tile is 2.5 times slower an operation but
// spreads over all CUs (1024 rows, 50,000 classes: 3.06 rounds take 3.2 tiles' time in place of 4).
static int lce_cut(int n, int other) {
    const long long tiles = (long long)lce_cdiv(n, 256) * other, rounds = tiles / 256;
    if (!rounds || tiles % 256 == 0 || tiles % 256 >= 102) return n;
    const long long cut = rounds * 256 / other * 256;
    return cut > 0 && cut < n ? (int)cut : n;
}

struct LcePlan {
    int Dp, fshape, fmt, fcut, padx, padw;
    int piece, large, ldg, xshape, splits; // classes of a piece, at most of the last one
    int wsplits;                           // dW: cuts of the rows
    int share;                             // kept logits: rows of a workgroup (and of a sum of db)
    size_t o_part, o_ps, o_zt, o_row, o_x, o_w, o_coef, o_scale, o_g, o_dx, o_dw, o_db, bytes;
};

static LcePlan lce_plan(const Lce *a, bool bwd) {
    LcePlan p = {};
    const int es = lce_esize(a->dtype);
    p.Dp = lce_dp(a);
    p.padw = !lce_plain(a, a->w, a->ldw, 256);
    size_t at = 0;
    auto take = [&](size_t n) { const size_t o = at; at += lce_up(n); return o; };
    if (p.padw) p.o_w = take((size_t)a->V * p.Dp * es);
    if (!bwd) {
        p.padx = !lce_plain(a, a->x, a->ldx, a->rows ? a->T : 256);
        if (p.padx) p.o_x = take((size_t)a->T * p.Dp * es);
        p.fshape = lce_shape(a->V, a->T);
        p.fcut = p.fshape ? a->V : lce_cut(a->V, lce_cdiv(a->T, 256));
        p.fmt = lce_cdiv(p.fcut, LCE_BM[p.fshape]) + lce_cdiv(a->V - p.fcut, LCE_BM[1]);
        p.o_part = take((size_t)p.fmt * a->T * 8);
        if (a->smoothing != 0.f) p.o_ps = take((size_t)p.fmt * a->T * 4);
        p.o_zt = take((size_t)a->T * 4);
        p.o_row = take((size_t)a->T * 4);
    } else {
        p.padx = 1;
        p.o_x = take((size_t)a->T * p.Dp * es);
        p.o_coef = take((size_t)a->T * 4);
        p.o_scale = take(4);
        // a piece: g of at most LCE_PIECE_BYTES, at least 256 classes; pieces whose dW is whole rounds of the large tile over
        // the CUs (up to a quarter of one more in the last), or of one size where not even one round fits (forward + backward
        // of 8192 rows, D 1024, 33,000 classes, bf16: 2.42 ms, and 3.66 in pieces of one size; D 512, 60,000 classes: 2.38 and
        // 3.71)
        long long most = LCE_PIECE_BYTES / ((long long)a->T * es) / 256;
        if (most < 1) most = 1;
        const long long across_d = lce_cdiv(p.Dp, 256), fit = 256 / across_d;
        if (most < fit && (long long)a->T * fit * 256 * es <= LCE_PIECE_MOST) most = fit;
        const long long rounds = most * across_d / 256;
        const long long tiles_v = lce_cdiv(a->V, 256), n = (tiles_v + most - 1) / most;
        p.piece = (int)(n == 1 || !rounds ? (tiles_v + n - 1) / n : std::max(1ll, 256 * rounds / across_d)) * 256;
        const int rest = a->V % p.piece;
        p.large = a->V > p.piece && rest < p.piece / 4 ? p.piece + (rest + 255) / 256 * 256 : p.piece;
        p.ldg = p.large + (es == 2 ? 128 : 64);
        p.o_g = take((size_t)a->T * p.ldg * es);
        // dx: few tiles and a long k: cut k until there are about 512 workgroups, of at least 256 classes
        p.xshape = a->T <= 32 ? 2 : a->T >= 128 && p.Dp >= 256 ? 0 : 1;
        const long long tiles = (long long)lce_cdiv(p.Dp, LCE_BM[p.xshape]) * lce_cdiv(a->T, LCE_BN[p.xshape]);
        long long s = (p.xshape == 0 ? 256 : 512) / tiles;
        if (s > p.piece / 256) s = p.piece / 256;
        p.splits = s < 1 ? 1 : (int)s;
        p.o_dx = take((size_t)p.splits * a->T * p.Dp * 4);
        // dW: few tiles and many rows: cut the rows until there are about 256 workgroups, of at least 512 rows
        // (forward + backward of 200,000 rows, D 256, 2 classes, float32: 1.1 ms, and 6.1 in four workgroups)
        const long long vmost = std::min(a->V, p.large), small = (long long)lce_cdiv(p.Dp, 64) * lce_cdiv(vmost, 64);
        p.wsplits = (int)std::max(1ll, small < 128 ? std::min(256 / small, (long long)a->T / 512) : 1);
        if (p.wsplits > 1) p.o_dw = take((size_t)p.wsplits * vmost * p.Dp * 4);
        // kept logits: about 1024 workgroups;  db: a sum a workgroup there, a tile of rows otherwise (the small tile's: 64 of them,
        // or all that there are)
        p.share = (int)std::max(1ll, (long long)a->T * lce_cdiv(p.piece, 1024) / 1024);
        if (a->bias) p.o_db = take((size_t)lce_cdiv(a->T, a->z ? p.share : 64) * p.ldg * 4);
    }
    p.bytes = at;
    return p;
}

static bool lce_bad(const Lce *a) {
    return !a || !a->x || !a->w || !a->target || a->T <= 0 || a->D <= 0 || a->V <= 0 || a->dtype < PNGPD_F32 || a->dtype > PNGPD_F16 ||
           a->ldx < (a->T > 1 ? a->D : 0) || a->ldw < (a->V > 1 ? a->D : 0) || (a->bias_dtype != PNGPD_F32 && a->bias_dtype != a->dtype) ||
           a->reduction < PNGPD_REDUCE_NONE || a->reduction > PNGPD_REDUCE_SUM || !(a->smoothing >= 0.f && a->smoothing <= 1.f) ||
           !a->stat || !a->kept || !a->rows != !pngpd_lce_rows_ints(a->T) ||
           (a->z && (((uintptr_t)a->z & 15) || !pngpd_lce_z_bytes(a->T, a->D, a->V, a->dtype)));
}

template <class K, class A> static int lce_launch(K kernel, int lds, long long grid, int threads, const A &a, hipStream_t st) {
    if (grid > 0x7fffffffll) return PNGPD_ERR_UNSUPPORTED;
    const int rc = pngpd_allow_lds((const void *)kernel, lds);
    if (rc) return rc;
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(threads), lds, st, a);
    return pngpd_launch_status();
}
template <int DT, bool GRAD, int BM, int BN, int WGM, int WGN, int PIPE> static int lce_z_shape(LceArgs &a, hipStream_t st) {
    constexpr int lds = LceCore<DT, false, false, BM, BN, WGM, WGN, PIPE>::LDS + 2 * (int)sizeof(LceSide<BM, BN>) + WGM * BN * 12;
    static_assert(lds <= 160 * 1024, "LDS of a CU");
    a.mt = lce_cdiv(a.vc, BM);
    // as many workgroups as run at once (256 CUs), walking over the tiles
    const long long tiles = (long long)a.mt * lce_cdiv(a.T, BN), most = 256ll * (160 * 1024 / lds < 4 ? 160 * 1024 / lds : 4);
    if (tiles > 0x7fffffffll - most) return PNGPD_ERR_UNSUPPORTED;
    const long long grid = tiles < most ? tiles : most;
    if constexpr (GRAD) return lce_launch(lce_grad_kernel<DT, BM, BN, WGM, WGN, PIPE>, lds, grid, WGM * WGN * 64, a, st);
    else return lce_launch(lce_stats_kernel<DT, BM, BN, WGM, WGN, PIPE>, lds, grid, WGM * WGN * 64, a, st);
}
template <int DT, bool GRAD> static int lce_z(LceArgs &a, int shape, hipStream_t st) {
    return shape == 0 ? lce_z_shape<DT, GRAD, LCE_SHAPE0>(a, st) : shape == 1 ? lce_z_shape<DT, GRAD, LCE_SHAPE1>(a, st)
         : shape == 2 ? lce_z_shape<DT, GRAD, LCE_SHAPE2>(a, st) : lce_z_shape<DT, GRAD, LCE_SHAPE3>(a, st);
}
template <int DT, bool BMC, int BM, int BN, int WGM, int WGN, int PIPE> static int lce_out_shape(LceOut &a, hipStream_t st) {
    a.mt = lce_cdiv(a.M, BM); a.nt = lce_cdiv(a.no, BN);
    return lce_launch(lce_out_kernel<DT, BMC, BM, BN, WGM, WGN, PIPE>, LceCore<DT, true, BMC, BM, BN, WGM, WGN, PIPE>::LDS,
                      (long long)a.mt * a.nt * a.splits, WGM * WGN * 64, a, st);
}
template <int DT, bool BMC> static int lce_out(LceOut &a, int shape, hipStream_t st) {
    if (shape == 0) return lce_out_shape<DT, BMC, LCE_SHAPE0>(a, st);
    if constexpr (BMC) if (shape == 3) return lce_out_shape<DT, BMC, LCE_SHAPE3>(a, st);
    if constexpr (!BMC) if (shape == 2) return lce_out_shape<DT, BMC, LCE_SHAPE2>(a, st);
    return lce_out_shape<DT, BMC, LCE_SHAPE1>(a, st);
}

template <int DT>
static void lce_copy(const Lce *a, const void *src, long long ld, long long R, int mask, LceRows rows, void *dst, hipStream_t st,
                     const LceCoef &coef = LceCoef{}) {
    const int Dp = lce_dp(a);
    const long long n = R * (Dp * lce_esize(DT) / 16);
    hipLaunchKernelGGL(lce_copy_kernel<DT>, dim3((unsigned)((n + 255) / 256 + (coef.coef != nullptr))), dim3(256), 0, st, src, ld, a->D, Dp, R,
                       mask, rows, (const long long *)a->target, (long long)a->ignore_index, dst, coef);
}

static inline int lce_ldz(int V) { return (V + 255) / 256 * 256; }
// Whether the logits are kept, in float32, where they are few: written and read they are 8 bytes a logit at the memory's rate
// (1.6 ps); computed again 2 D operations at the matrix cores' float32 rate (0.014 ps D), or, for few rows of 16 bits, W read again
// (2 D bytes a class, against 8 T of the logits).  Forward + backward on the GPU alone, kept and computed again: float32, 64 x 256 x
// 6500 55 and 61 us, 256 x 128 x 20,000 92 and 102, 1024 x 2048 x 12,000 1375 and 1745; bf16, 1 x 64 x 100,000 77 and 86, 64 x 256 x
// 40,000 (T = D / 4) 76 and 79, 256 x 1024 x 40,000 174 and 189, 500 x 2048 x 30,000 317 and 349.  More rows of 16 bits are computed
// again, also of a D past 800 where 2 D operations cost more than 1.6 ps: their large tile does not store them (not measured).
static bool lce_keeps(int T, int D, int V, int dt) {
    if (V < 128) return false;                                    // (rows are padded to whole 256 classes)
    const long long bytes = (long long)T * lce_ldz(V) * 4;
    return dt == PNGPD_F32 ? D >= 128 && bytes <= LCE_PIECE_MOST : 4ll * T <= D && bytes <= LCE_PIECE_BYTES && lce_shape(V, T) != 0;
}
static LceArgs lce_args(const Lce *a) {
    LceArgs k = {};
    k.x = LceOperand{a->x, a->ldx}; k.w = LceOperand{a->w, a->ldw}; k.rows = LceRows{a->rows, a->T};
    k.bias = a->bias; k.bf32 = a->bias_dtype == PNGPD_F32; k.target = (const long long *)a->target; k.ignore = a->ignore_index;
    k.T = a->T; k.D = a->D; k.V = a->V; k.smooth = a->smoothing;
    k.z = a->z; k.ldz = lce_ldz(a->V);
    return k;
}

template <int DT> static int lce_forward(const Lce *a, const LcePlan &p, hipStream_t st) {
    char *ws = (char *)a->workspace;
    LceArgs k = lce_args(a);
    if (a->rows) hipLaunchKernelGGL(lce_rows_kernel, dim3(1), dim3(1024), 0, st, k.target, k.ignore, a->T, a->rows);
    if (p.padx) {
        lce_copy<DT>(a, a->x, a->ldx, a->T, 1, k.rows, ws + p.o_x, st);
        k.x = LceOperand{ws + p.o_x, p.Dp};
        k.packed = 1;
    }
    if (p.padw) { lce_copy<DT>(a, a->w, a->ldw, a->V, 0, k.rows, ws + p.o_w, st); k.w = LceOperand{ws + p.o_w, p.Dp}; }
    k.D = p.Dp;
    k.pm = (float *)(ws + p.o_part); k.ps = (float *)(ws + p.o_ps); k.zt = (float *)(ws + p.o_zt);
    k.vc = p.fcut;
    int rc = lce_z<DT, false>(k, p.fshape, st);
    if (rc) return rc;
    if (p.fcut < a->V) {
        k.v0 = p.fcut; k.vc = a->V - p.fcut; k.mt0 = k.mt;
        if ((rc = lce_z<DT, false>(k, 1, st))) return rc;
    }
    k.mt = p.fmt;
    float *row = a->reduction == PNGPD_REDUCE_NONE ? a->loss : (float *)(ws + p.o_row);
    if (a->T <= LCE_FEW) {
        hipLaunchKernelGGL(lce_join_kernel<32>, dim3(1), dim3(1024), 0, st, k, a->stat, row, a->reduction, a->loss, a->kept);
        return pngpd_launch_status();
    }
    hipLaunchKernelGGL(lce_join_kernel<8>, dim3((unsigned)((a->T + 7) / 8)), dim3(256), 0, st, k, a->stat, row, a->reduction, a->loss, a->kept);
    if (a->reduction != PNGPD_REDUCE_NONE)
        hipLaunchKernelGGL(lce_loss_kernel, dim3(1), dim3(1024), 0, st, k, row, a->reduction, a->loss, a->kept);
    return pngpd_launch_status();
}

template <int DT> static int lce_backward(const Lce *a, const LcePlan &p, hipStream_t st) {
    typedef typename elem<DT>::t E;
    char *ws = (char *)a->workspace;
    LceArgs k = lce_args(a);
    float *coef = (float *)(ws + p.o_coef), *scale = (float *)(ws + p.o_scale), *part = (float *)(ws + p.o_dx);
    lce_copy<DT>(a, a->x, a->ldx, a->T, 1, k.rows, ws + p.o_x, st,
                 LceCoef{a->dloss, a->kept, k.target, k.ignore, k.rows, a->V, a->reduction, DT == PNGPD_F16 ? 32768.f : 1.f, coef, scale});
    k.x = LceOperand{ws + p.o_x, p.Dp};
    k.packed = 1;
    if (p.padw) { lce_copy<DT>(a, a->w, a->ldw, a->V, 0, k.rows, ws + p.o_w, st); k.w = LceOperand{ws + p.o_w, p.Dp}; }
    k.D = p.Dp;
    k.stat = a->stat; k.coef = coef; k.ldg = p.ldg;
    for (int v0 = 0, vc; v0 < a->V; v0 += vc) {
        vc = a->V - v0 <= p.large ? a->V - v0 : p.piece;
        const int gshape = lce_shape(vc, a->T), wide = lce_shape(p.Dp, vc, 192), wshape = wide == 2 ? 1 : wide;
        const int cols = (vc + 63) / 64 * 64;                      // columns of g that are written (zeros past vc)
        const int gcut = gshape ? vc : lce_cut(vc, lce_cdiv(a->T, 256));
        float *sums = (float *)(ws + p.o_db);
        k.v0 = v0; k.vc = gcut; k.g = ws + p.o_g; k.db = a->db ? sums : nullptr;
        int rc;
        if (a->z) {
            k.vc = vc;
            const long long grid = (long long)lce_cdiv(a->T, p.share) * ((cols + 1023) / 1024);
            if (grid > 0x7fffffffll) return PNGPD_ERR_UNSUPPORTED;
            hipLaunchKernelGGL(lce_kept_grad_kernel<DT>, dim3((unsigned)grid), dim3(256), 0, st, k, cols, p.share);
            rc = pngpd_launch_status();
        } else rc = lce_z<DT, true>(k, gshape, st);
        if (rc) return rc;
        if (!a->z && gcut < vc) {
            k.v0 = v0 + gcut; k.vc = vc - gcut; k.g = (E *)(ws + p.o_g) + gcut; k.db = a->db ? sums + gcut : nullptr;
            if ((rc = lce_z<DT, true>(k, 1, st))) return rc;
        }
        const E *g = (const E *)(ws + p.o_g);
        const E *w = (const E *)k.w.p + (long long)v0 * k.w.ld;
        if (a->db) {
            void *db = a->bias_dtype == PNGPD_F32 ? (void *)((float *)a->db + v0) : (void *)((E *)a->db + v0);
            hipLaunchKernelGGL(lce_db_join_kernel<DT>, dim3((unsigned)lce_cdiv(vc, 32)), dim3(256), 0, st, sums, k.rows,
                               a->z ? p.share : LCE_BN[gshape], a->z ? vc : gcut, LCE_BN[1], p.ldg, vc, scale, db,
                               (int)(a->bias_dtype == PNGPD_F32));
        }
        if (a->dx) {
            LceOut o = {};
            o.a = LceOperand{w, k.w.ld}; o.b = LceOperand{g, p.ldg}; o.rows = k.rows;
            o.M = p.Dp; o.N = -1; o.mo = a->D; o.no = a->T; o.K = vc; o.splits = p.splits;
            o.kper = ((long long)vc + 64 * p.splits - 1) / (64 * p.splits) * 64;
            o.part = part; o.pn = a->T; o.add = v0 > 0; o.scale = scale;
            if ((rc = lce_out<DT, false>(o, p.xshape, st))) return rc;
        }
        if (a->dw && p.wsplits > 1) {
            LceOut o = {};
            o.a = LceOperand{k.x.p, p.Dp}; o.b = LceOperand{g, p.ldg}; o.rows = k.rows;
            o.M = p.Dp; o.N = cols; o.mo = a->D; o.no = vc; o.K = -1; o.splits = p.wsplits;
            o.kper = ((long long)a->T + 64 * p.wsplits - 1) / (64 * p.wsplits) * 64;
            o.part = (float *)(ws + p.o_dw); o.pn = vc; o.scale = scale;
            if ((rc = lce_out<DT, true>(o, 1, st))) return rc;
            const long long n = (long long)vc * (p.Dp / 4);
            hipLaunchKernelGGL(lce_dx_kernel<DT>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, o.part, p.wsplits,
                               LceRows{nullptr, vc}, a->D, p.Dp, scale, (void *)((E *)a->dw + (long long)v0 * a->D));
        } else if (a->dw) {
            const int wcut = wshape ? vc : lce_cut(vc, lce_cdiv(p.Dp, 256));
            for (int c0 = 0; c0 < vc; c0 = c0 ? vc : wcut) {       // the large tile's classes, then the rest
                const int c1 = c0 ? vc : wcut;
                LceOut o = {};
                o.a = LceOperand{k.x.p, p.Dp}; o.b = LceOperand{g + c0, p.ldg}; o.rows = k.rows;
                o.M = p.Dp; o.N = (c1 == vc ? cols : c1) - c0; o.mo = a->D; o.no = c1 - c0; o.K = -1; o.kper = a->T; o.splits = 1;
                o.out = (E *)a->dw + (long long)(v0 + c0) * a->D; o.ldo = a->D; o.scale = scale;
                o.vec = (a->D * (long long)sizeof(E)) % 16 == 0 && !((uintptr_t)a->dw & 15);
                if ((rc = lce_out<DT, true>(o, c0 ? 1 : wshape, st))) return rc;
            }
        }
    }
    if (a->dx) {
        const long long n = (long long)a->T * (p.Dp / 4);
        hipLaunchKernelGGL(lce_dx_kernel<DT>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, part, p.splits, k.rows, a->D, p.Dp,
                           scale, a->dx);
    }
    return pngpd_launch_status();
}

extern "C" {

size_t pngpd_lce_rows_ints(int T) { return T < LCE_ROWS ? 0 : 2 * (size_t)T + 1; }

size_t pngpd_lce_z_bytes(int T, int D, int V, int dtype) {
    if (T <= 0 || D <= 0 || V <= 0 || V >= 1 << 30 || dtype < PNGPD_F32 || dtype > PNGPD_F16 || !lce_keeps(T, D, V, dtype)) return 0;
    return (size_t)T * lce_ldz(V) * 4;
}

size_t pngpd_lce_workspace_bytes(const pngpd_lce_t *a, int backward) {
    return lce_bad(a) ? 0 : lce_plan(a, backward != 0).bytes;
}

// row numbers and places of the kept rows are ints behind one another: 1 + 2 T of them
static bool lce_too_many(const Lce *a) { return a->D > LCE_MOST_D || a->T >= 1 << 30 || a->V >= 1 << 30; }

int pngpd_lce_fwd(const pngpd_lce_t *a, void *stream) {
    if (lce_bad(a) || !a->loss) return PNGPD_ERR_INVALID_ARG;
    if (lce_too_many(a)) return PNGPD_ERR_UNSUPPORTED;
    const LcePlan p = lce_plan(a, false);
    if (!a->workspace || ((uintptr_t)a->workspace & 255) || a->workspace_bytes < p.bytes) return PNGPD_ERR_WORKSPACE;
    hipStream_t st = (hipStream_t)stream;
    if (a->dtype == PNGPD_F32) return lce_forward<PNGPD_F32>(a, p, st);
    if (a->dtype == PNGPD_BF16) return lce_forward<PNGPD_BF16>(a, p, st);
    return lce_forward<PNGPD_F16>(a, p, st);
}

int pngpd_lce_bwd(const pngpd_lce_t *a, void *stream) {
    if (lce_bad(a) || !a->dloss || (a->db && !a->bias)) return PNGPD_ERR_INVALID_ARG;
    if (lce_too_many(a)) return PNGPD_ERR_UNSUPPORTED;
    if (!a->dx && !a->dw && !a->db) return PNGPD_OK;
    const LcePlan p = lce_plan(a, true);
    if (!a->workspace || ((uintptr_t)a->workspace & 255) || a->workspace_bytes < p.bytes) return PNGPD_ERR_WORKSPACE;
    hipStream_t st = (hipStream_t)stream;
    if (a->dtype == PNGPD_F32) return lce_backward<PNGPD_F32>(a, p, st);
    if (a->dtype == PNGPD_BF16) return lce_backward<PNGPD_BF16>(a, p, st);
    return lce_backward<PNGPD_F16>(a, p, st);
}

}  // extern "C"
