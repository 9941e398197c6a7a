// Linear + softmax cross entropy over many classes, the logits never kept, with its gradient.
//
//   z = x W^T + b  (T,V)     m_t = max_v z     s_t = sum_v exp(z - m_t)     lse_t = m_t + log s_t
//   loss_t = lse_t - (1 - e) z[t, y_t] - e mean_v z          (0 where y_t = ignore_index)
//   g = c_t (exp(z - m_t) / s_t - (1 - e) [v = y_t] - e / V),   c_t = dL/dloss_t        (0 where ignored)
//   dx = g W      dW = g^T x      db = sum_t g
//
// Forward: every tile of z reduces in registers to (max, sum of exponentials, sum) of its rows; a second launch joins the
// tiles of a row.  Backward: z is computed again, a piece of the vocabulary at a time; the piece's g (rounded once to the
// inputs' type, as the operand of the matrix instructions has to be) lives in a workspace of bounded size, and two products
// turn it into the piece's dW and its share of dx.  8 T D V operations for both directions where keeping T V logits takes
// 6: the price of not keeping them.  Bound by the matrix cores for T in the hundreds and above, by reading W below.
// float16 holds g times 2^15 (|g| <= 1: below 65504, and its normal range then reaches down to 2e-9, under 1/V); the
// coefficients c_t are scaled to at most 1 the same way; both factors come back in float32 on the way out.
#include "pngpd_lce_gemm.h"

#define LCE_PIECE_BYTES (256ll << 20)      // a piece's g

struct LceArgs {
    LceOperand x, w;                       // rows of 16-byte multiples
    const void *bias;
    int bf32;
    const long long *target;
    long long ignore;
    int T, D, V, mt, nt;
    float smooth;
    float *pm, *ps, *zt;                   // forward: (mt,T,2) max / sum, (mt,T) sum of z, (T) z at the target
    const float *stat, *coef;              // backward: (T,2) max / sum, (T)
    void *g;
    int v0, vc, ldg;                       // the piece
};

template <int DT> __device__ __forceinline__ void lce_bias4(const LceArgs &a, int v, float (&b)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
        b[e] = !a.bias || v + e >= a.V ? 0.f
             : a.bf32 ? ((const float *)a.bias)[v + e] : ld_elem<DT>((const typename elem<DT>::t *)a.bias + v + e);
}

// (max, sum) of two parts of a row; a part without values is (-inf, 0)
__device__ __forceinline__ void lce_join(float &m, float &s, float m2, float s2) {
    const float M = fmaxf(m, m2), ref = M == -INFINITY ? 0.f : M;
    s = s * __expf(m - ref) + s2 * __expf(m2 - ref);
    m = M;
}

template <int DT, int BM, int BN, int WGM, int WGN>
__global__ __launch_bounds__(WGM * WGN * 64, 2) void lce_stats_kernel(const LceArgs a) {
    typedef LceCore<DT, false, false, BM, BN, WGM, WGN> Core;
    extern __shared__ __align__(16) char smem[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int wm = (wave % WGM) * Core::WM, wn = (wave / WGM) * Core::WN;
    int tm, tn;
    lce_tile_of(blockIdx.x, a.mt * a.nt, a.mt, a.nt, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;
    Core c;
    c.run(smem, a.w, a.x, m0, a.V, n0, a.T, 0, a.D);
    float *sh = (float *)smem;                                    // [WGM][BN][3]
    const bool ragged = m0 + BM > a.V;
#pragma unroll
    for (int i = 0; i < Core::FM; ++i) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int v = m0 + wm + 32 * i + 8 * q + 4 * half;
            float b[4];
            lce_bias4<DT>(a, v, b);
#pragma unroll
            for (int j = 0; j < Core::FN; ++j) {
#pragma unroll
                for (int e = 0; e < 4; ++e) c.acc[i][j][4 * q + e] += b[e];
            }
        }
    }
#pragma unroll
    for (int j = 0; j < Core::FN; ++j) {
        const int col = wn + 32 * j + (lane & 31), t = n0 + col;
        float m = -INFINITY, s = 0.f, sz = 0.f;
        const long long y = t < a.T ? a.target[t] : -1;
        const long long rel = y - (m0 + wm + 4 * half);
        const bool here = rel >= 0 && rel < Core::WM && y < a.V;
#pragma unroll
        for (int i = 0; i < Core::FM; ++i) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int off = 32 * i + (r & 3) + 8 * (r >> 2);
                float z = c.acc[i][j][r];
                if (here && rel == off) a.zt[t] = z;
                if (ragged && m0 + wm + 4 * half + off >= a.V) z = -INFINITY;
                else if (a.smooth != 0.f) sz += z;
                c.acc[i][j][r] = z;
                m = fmaxf(m, z);
            }
        }
        float lo, hi;
        half_pair(m, lo, hi);
        m = fmaxf(lo, hi);
        const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int i = 0; i < Core::FM; ++i) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s += __expf(c.acc[i][j][r] - ref);
        }
        s = half_sum(s);
        if (a.smooth != 0.f) sz = half_sum(sz);
        if (half == 0) {
            float *o = sh + ((wave % WGM) * BN + col) * 3;
            o[0] = m; o[1] = s; o[2] = sz;
        }
    }
    __syncthreads();
    for (int col = threadIdx.x; col < BN; col += Core::THREADS) {
        const int t = n0 + col;
        if (t >= a.T) continue;
        float m = sh[col * 3], s = sh[col * 3 + 1], sz = sh[col * 3 + 2];
#pragma unroll
        for (int k = 1; k < WGM; ++k) {
            const float *o = sh + (k * BN + col) * 3;
            lce_join(m, s, o[0], o[1]);
            sz += o[2];
        }
        const size_t at = (size_t)tm * a.T + t;
        *(f32x2 *)(a.pm + 2 * at) = f32x2{m, s};
        if (a.smooth != 0.f) a.ps[at] = sz;
    }
}

// One row a group of 8 lanes: joins its tiles, in fp64; stat (T,2) = max, sum; row (T) = the row's loss.
__global__ __launch_bounds__(256) void lce_join_kernel(const LceArgs a, float *__restrict__ stat, float *__restrict__ row) {
    __shared__ double sh[8][32][2];
    __shared__ float shm[8][32];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, t = blockIdx.x * 32 + tx;
    float m = -INFINITY;
    double s = 0.0, sz = 0.0;
    if (t < a.T) {
        for (int k = ty; k < a.mt; k += 8) {
            const size_t at = (size_t)k * a.T + t;
            const f32x2 p = *(const f32x2 *)(a.pm + 2 * at);
            const float M = fmaxf(m, p[0]), ref = M == -INFINITY ? 0.f : M;
            s = s * (double)expf(m - ref) + (double)p[1] * (double)expf(p[0] - ref);
            m = M;
            if (a.smooth != 0.f) sz += (double)a.ps[at];
        }
    }
    shm[ty][tx] = m; sh[ty][tx][0] = s; sh[ty][tx][1] = sz;
    __syncthreads();
    if (ty || t >= a.T) return;
    float M = m;
    for (int k = 1; k < 8; ++k) M = fmaxf(M, shm[k][tx]);
    const float ref = M == -INFINITY ? 0.f : M;
    s = sz = 0.0;
    for (int k = 0; k < 8; ++k) { s += sh[k][tx][0] * (double)expf(shm[k][tx] - ref); sz += sh[k][tx][1]; }
    stat[2 * (size_t)t] = M; stat[2 * (size_t)t + 1] = (float)s;
    const long long y = a.target[t];
    double l = 0.0;
    if (y != a.ignore) {
        if (y < 0 || y >= a.V) l = NAN;                            // a class that does not exist: as loud as a value can be
        else {
            l = (double)M + log(s) - (1.0 - (double)a.smooth) * (double)a.zt[t];
            if (a.smooth != 0.f) l -= (double)a.smooth * sz / a.V;
        }
    }
    row[t] = (float)l;
}

__device__ __forceinline__ double lce_block_sum(double v, double *sh) {
    for (int k = 32; k >= 1; k >>= 1) v += __shfl_xor(v, k);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0.0;
    for (int k = 0; k < 16; ++k) s += sh[k];
    return s;
}

// kept rows; loss = their sum or mean (a mean over none is NaN)
__global__ __launch_bounds__(1024) void lce_loss_kernel(const float *__restrict__ row, const long long *__restrict__ target,
                                                        long long ignore, int T, int reduction, float *__restrict__ loss,
                                                        float *__restrict__ kept) {
    __shared__ double sh[16];
    double s = 0.0, n = 0.0;
    for (int t = threadIdx.x; t < T; t += 1024) {
        if (target[t] != ignore) n += 1.0;
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

// coef (T) = c_t over the largest finite |c_t| (times up, the factor of the type's range), scale = what gives c_t back
__global__ __launch_bounds__(1024) void lce_coef_kernel(const float *__restrict__ dloss, const float *__restrict__ kept,
                                                        const long long *__restrict__ target, long long ignore, int T, int V,
                                                        int reduction, float up, float *__restrict__ coef,
                                                        float *__restrict__ scale) {
    __shared__ float sh[16];
    float top = 1.f;
    if (reduction == PNGPD_REDUCE_NONE) {
        top = 0.f;
        for (int t = threadIdx.x; t < T; t += 1024) {
            const float c = fabsf(dloss[t]);
            if (c < INFINITY && target[t] != ignore) top = fmaxf(top, c);
        }
        for (int k = 32; k >= 1; k >>= 1) top = fmaxf(top, __shfl_xor(top, k));
        if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = top;
        __syncthreads();
        for (int k = 0; k < 16; ++k) top = fmaxf(top, sh[k]);
        if (top == 0.f) top = 1.f;
    }
    for (int t = threadIdx.x; t < T; t += 1024) {
        const long long y = target[t];
        float c = reduction == PNGPD_REDUCE_NONE ? dloss[t] / top * up : up;
        if (y == ignore) c = 0.f;
        else if (y < 0 || y >= V) c = NAN;
        coef[t] = c;
    }
    if (threadIdx.x == 0) {
        float s = top / up;
        if (reduction == PNGPD_REDUCE_SUM) s = *dloss / up;
        if (reduction == PNGPD_REDUCE_MEAN) s = *kept > 0.f ? *dloss / *kept / up : 0.f;     // no row, no gradient
        *scale = s;
    }
}

template <int DT, int BM, int BN, int WGM, int WGN>
__global__ __launch_bounds__(WGM * WGN * 64, 2) void lce_grad_kernel(const LceArgs a) {
    typedef LceCore<DT, false, false, BM, BN, WGM, WGN> Core;
    typedef typename elem<DT>::t E;
    extern __shared__ __align__(16) char smem[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int wm = (wave % WGM) * Core::WM, wn = (wave / WGM) * Core::WN;
    int tm, tn;
    lce_tile_of(blockIdx.x, a.mt * a.nt, a.mt, a.nt, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;
    LceOperand w = a.w;
    w.p = (const E *)a.w.p + (long long)a.v0 * a.w.ld;
    Core c;
    c.run(smem, w, a.x, m0, a.vc, n0, a.T, 0, a.D);
    const float flat = a.smooth / (float)a.V, hit = 1.f - a.smooth;
#pragma unroll
    for (int j = 0; j < Core::FN; ++j) {
        const int t = n0 + wn + 32 * j + (lane & 31);
        if (t >= a.T) continue;
        const float m = a.stat[2 * (size_t)t], is = 1.f / a.stat[2 * (size_t)t + 1], co = a.coef[t];
        const long long rel = a.target[t] - (a.v0 + m0 + wm + 4 * half);
        E *g = (E *)a.g + (size_t)t * a.ldg + m0 + wm + 4 * half;
#pragma unroll
        for (int i = 0; i < Core::FM; ++i) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int off = 32 * i + 8 * q;
                float b[4], o[4];
                lce_bias4<DT>(a, a.v0 + m0 + wm + 4 * half + off, b);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float p = __expf(c.acc[i][j][4 * q + e] + b[e] - m) * is;
                    const float d = p - flat - (rel == off + e ? hit : 0.f);
                    o[e] = co == 0.f || m0 + wm + 4 * half + off + e >= a.vc ? 0.f : co * d;
                }
                if constexpr (DT == PNGPD_F32) *(f32x4 *)(g + off) = f32x4{o[0], o[1], o[2], o[3]};
                else *(uint2 *)(g + off) = make_uint2((unsigned)f_to_half(DT, o[0]) | ((unsigned)f_to_half(DT, o[1]) << 16),
                                                      (unsigned)f_to_half(DT, o[2]) | ((unsigned)f_to_half(DT, o[3]) << 16));
            }
        }
    }
}

// db of a piece: column sums of g (fp32, rounded g), 64 columns x 16 row lanes a workgroup
template <int DT>
__global__ __launch_bounds__(1024) void lce_db_kernel(const void *__restrict__ gp, int T, int vc, int ldg,
                                                      const float *__restrict__ scale, void *__restrict__ db, int f32) {
    __shared__ double sh[16][64];
    const int cx = threadIdx.x & 63, ry = threadIdx.x >> 6, v = blockIdx.x * 64 + cx;
    const typename elem<DT>::t *g = (const typename elem<DT>::t *)gp + v;
    double s = 0.0;
    for (int t = ry; t < T; t += 16) s += (double)ld_elem<DT>(g + (size_t)t * ldg);      // (columns are padded to 64)
    sh[ry][cx] = s;
    __syncthreads();
    if (ry || v >= vc) return;
    for (int k = 1; k < 16; ++k) s += sh[k][cx];
    const float o = (float)s * *scale;
    if (f32) ((float *)db)[v] = o;
    else st_elem<DT>((typename elem<DT>::t *)db + v, o);
}

struct LceOut {
    LceOperand a, b;
    int M, N, mt, nt;                      // M: m that exist in a's rows (padded); N likewise
    int mo, no;                            // outputs stored
    long long K, kper;                     // k of a split
    void *out;                             // typed: out[n * ldo + m] = scale * sum
    long long ldo;
    float *part;                           // or fp32 partial sums (splits, no, M), added to what is there
    int add;
    const float *scale;
    int vec;                               // out rows take 4 values at once
};

template <int DT, bool BMC, int BM, int BN, int WGM, int WGN>
__global__ __launch_bounds__(WGM * WGN * 64, 2) void lce_out_kernel(const LceOut a) {
    typedef LceCore<DT, true, BMC, BM, BN, WGM, WGN> Core;
    typedef typename elem<DT>::t E;
    extern __shared__ __align__(16) char smem[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int wm = (wave % WGM) * Core::WM, wn = (wave / WGM) * Core::WN;
    const int tiles = a.mt * a.nt, split = blockIdx.x / tiles;
    int tm, tn;
    lce_tile_of(blockIdx.x - split * tiles, tiles, a.mt, a.nt, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;
    const long long k0 = split * a.kper, k1 = k0 + a.kper < a.K ? k0 + a.kper : a.K;
    Core c;
    c.run(smem, a.a, a.b, m0, a.M, n0, a.N, k0, k1);
    const float sc = a.part ? 1.f : *a.scale;
#pragma unroll
    for (int j = 0; j < Core::FN; ++j) {
        const int n = n0 + wn + 32 * j + (lane & 31);
        if (n >= a.no) continue;
#pragma unroll
        for (int i = 0; i < Core::FM; ++i) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int m = m0 + wm + 32 * i + 8 * q + 4 * half;
                f32x4 v = {c.acc[i][j][4 * q], c.acc[i][j][4 * q + 1], c.acc[i][j][4 * q + 2], c.acc[i][j][4 * q + 3]};
                if (a.part) {
                    if (m < a.M) {
                        f32x4 *o = (f32x4 *)(a.part + ((size_t)split * a.no + n) * a.M + m);
                        *o = a.add ? *o + v : v;
                    }
                } else {
                    v *= sc;
                    E *o = (E *)a.out + n * a.ldo + m;
                    if (a.vec && m + 4 <= a.mo) {
                        if constexpr (DT == PNGPD_F32) *(f32x4 *)o = v;
                        else *(uint2 *)o = make_uint2((unsigned)f_to_half(DT, v[0]) | ((unsigned)f_to_half(DT, v[1]) << 16),
                                                      (unsigned)f_to_half(DT, v[2]) | ((unsigned)f_to_half(DT, v[3]) << 16));
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) if (m + e < a.mo) st_elem<DT>(o + e, v[e]);
                    }
                }
            }
        }
    }
}

// dx = scale * sum of the splits' partial sums (rows of Dp, a multiple of 4)
template <int DT>
__global__ __launch_bounds__(256) void lce_dx_kernel(const float *__restrict__ part, int splits, int T, int D, int Dp,
                                                     const float *__restrict__ scale, void *__restrict__ dx) {
    typedef typename elem<DT>::t E;
    const int per = Dp / 4;
    const long long q = (long long)blockIdx.x * 256 + threadIdx.x;
    if (q >= (long long)T * per) return;
    const long long t = q / per;
    const int d = (int)(q - t * per) * 4;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < splits; ++s) v += *(const f32x4 *)(part + ((size_t)s * T + t) * Dp + d);
    const float sc = *scale;
    E *o = (E *)dx + t * D + d;
#pragma unroll
    for (int e = 0; e < 4; ++e) if (d + e < D) st_elem<DT>(o + e, v[e] * sc);
}

// dst (R,Dp) = src (R,D) with zeros behind, and a row of zeros where the target is ignored (what such a row holds is
// nobody's: a NaN there must not meet g's zeros in a product).  One 16-byte chunk of dst a thread.
template <int DT>
__global__ __launch_bounds__(256) void lce_copy_kernel(const void *__restrict__ src, long long ld, int D, int Dp, long long R,
                                                       const long long *__restrict__ target, long long ignore,
                                                       void *__restrict__ dst) {
    typedef typename elem<DT>::t E;
    constexpr int EPC = 16 / (int)sizeof(E);
    const int per = Dp / EPC;
    const long long q = (long long)blockIdx.x * 256 + threadIdx.x;
    if (q >= R * per) return;
    const long long r = q / per;
    const int d = (int)(q - r * per) * EPC;
    const E *s = (const E *)src + r * ld + d;
    __align__(16) E v[EPC];
#pragma unroll
    for (int e = 0; e < EPC; ++e) v[e] = (E)0;
    if (!target || target[r] != ignore) {
        if (d + EPC <= D) __builtin_memcpy(v, s, 16);
        else {
#pragma unroll
            for (int e = 0; e < EPC; ++e) if (d + e < D) v[e] = s[e];
        }
    }
    *(uint4 *)((E *)dst + r * Dp + d) = *(const uint4 *)v;
}

// ---------------------------------------------------------------------------------------------------- host
typedef pngpd_lce_t Lce;
static inline size_t lce_up(size_t n) { return (n + 255) & ~(size_t)255; }
static inline int lce_esize(int dt) { return dt == PNGPD_F32 ? 4 : 2; }
static inline int lce_dp(const Lce *a) { const int c = 16 / lce_esize(a->dtype); return (a->D + c - 1) / c * c; }
// rows that the loads can take as they are: 16-byte aligned, D a whole number of chunks
static inline bool lce_plain(const Lce *a, const void *p, long long ld) {
    return lce_dp(a) == a->D && !((uintptr_t)p & 15) && (ld * lce_esize(a->dtype)) % 16 == 0;
}

// tile shapes: 0 = 256 x 128, 1 = 64 x 64, 2 = 64 x 32
static const int LCE_BM[3] = {256, 64, 64}, LCE_BN[3] = {128, 64, 32};
static inline int lce_cdiv(long long a, int b) { return (int)((a + b - 1) / b); }
// The large tile needs a workgroup for every CU; the narrow one is for rows that would leave half of 64 unused.
static int lce_shape(long long M, long long N) {
    if (N <= 32) return 2;
    return (long long)lce_cdiv(M, 256) * lce_cdiv(N, 128) >= 256 ? 0 : 1;
}

struct LcePlan {
    int Dp, fshape, fmt, padx, padw;
    int piece, ldg, gshape, xshape, splits, wshape;
    long long kper;
    size_t o_part, o_ps, o_zt, o_row, o_x, o_w, o_coef, o_scale, o_g, o_dx, bytes;
};

static LcePlan lce_plan(const Lce *a, bool bwd) {
    LcePlan p = {};
    const int es = lce_esize(a->dtype);
    p.Dp = lce_dp(a);
    p.padw = !lce_plain(a, a->w, a->ldw);
    size_t at = 0;
    auto take = [&](size_t n) { const size_t o = at; at += lce_up(n); return o; };
    if (p.padw) p.o_w = take((size_t)a->V * p.Dp * es);
    if (!bwd) {
        p.padx = !lce_plain(a, a->x, a->ldx);
        if (p.padx) p.o_x = take((size_t)a->T * p.Dp * es);
        p.fshape = lce_shape(a->V, a->T);
        p.fmt = lce_cdiv(a->V, LCE_BM[p.fshape]);
        p.o_part = take((size_t)p.fmt * a->T * 8);
        if (a->smoothing != 0.f) p.o_ps = take((size_t)p.fmt * a->T * 4);
        p.o_zt = take((size_t)a->T * 4);
        p.o_row = take((size_t)a->T * 4);
    } else {
        p.padx = 1;
        p.o_x = take((size_t)a->T * p.Dp * es);
        p.o_coef = take((size_t)a->T * 4);
        p.o_scale = take(4);
        // a piece: g of at most LCE_PIECE_BYTES, at least 256 classes, pieces of one size
        long long most = LCE_PIECE_BYTES / ((long long)a->T * es) / 256 * 256;
        if (most < 256) most = 256;
        const long long n = ((long long)a->V + most - 1) / most;
        p.piece = (int)((((long long)a->V + n - 1) / n + 255) / 256 * 256);
        p.ldg = p.piece;
        p.gshape = lce_shape(p.piece, a->T);
        p.o_g = take((size_t)a->T * p.ldg * es);
        p.wshape = lce_shape(p.Dp, p.piece) ? 1 : 0;
        // dx: few tiles and a long k: cut k until there are about 512 workgroups, of at least 256 classes
        p.xshape = a->T <= 32 ? 2 : a->T >= 128 && p.Dp >= 256 ? 0 : 1;
        const long long tiles = (long long)lce_cdiv(p.Dp, LCE_BM[p.xshape]) * lce_cdiv(a->T, LCE_BN[p.xshape]);
        long long s = 512 / tiles;
        if (s > p.piece / 256) s = p.piece / 256;
        if (s < 1) s = 1;
        p.kper = (((long long)p.piece + s - 1) / s + 63) / 64 * 64;
        p.splits = (int)(((long long)p.piece + p.kper - 1) / p.kper);
        p.o_dx = take((size_t)p.splits * a->T * p.Dp * 4);
    }
    p.bytes = at;
    return p;
}

static bool lce_bad(const Lce *a) {
    return !a || !a->x || !a->w || !a->target || a->T <= 0 || a->D <= 0 || a->V <= 0 || a->dtype < PNGPD_F32 || a->dtype > PNGPD_F16 ||
           a->ldx < (a->T > 1 ? a->D : 0) || a->ldw < (a->V > 1 ? a->D : 0) || (a->bias_dtype != PNGPD_F32 && a->bias_dtype != a->dtype) ||
           a->reduction < PNGPD_REDUCE_NONE || a->reduction > PNGPD_REDUCE_SUM || !(a->smoothing >= 0.f && a->smoothing <= 1.f) ||
           !a->stat || !a->kept;
}

template <int DT, int KIND, int BM, int BN, int WGM, int WGN>          // KIND 0: stats, 1: grad
static int lce_launch_z(const LceArgs &a, hipStream_t st) {
    constexpr int lds = LceCore<DT, false, false, BM, BN, WGM, WGN>::LDS;
    if constexpr (KIND == 0) {
        const int rc = pngpd_allow_lds((const void *)lce_stats_kernel<DT, BM, BN, WGM, WGN>, lds);
        if (rc) return rc;
        hipLaunchKernelGGL((lce_stats_kernel<DT, BM, BN, WGM, WGN>), dim3((unsigned)(a.mt * a.nt)), dim3(WGM * WGN * 64), lds, st, a);
    } else {
        const int rc = pngpd_allow_lds((const void *)lce_grad_kernel<DT, BM, BN, WGM, WGN>, lds);
        if (rc) return rc;
        hipLaunchKernelGGL((lce_grad_kernel<DT, BM, BN, WGM, WGN>), dim3((unsigned)(a.mt * a.nt)), dim3(WGM * WGN * 64), lds, st, a);
    }
    return pngpd_launch_status();
}
template <int DT, int KIND> static int lce_z(LceArgs &a, int shape, int M, hipStream_t st) {
    a.mt = lce_cdiv(M, LCE_BM[shape]); a.nt = lce_cdiv(a.T, LCE_BN[shape]);
    if ((long long)a.mt * a.nt > 0x7fffffffll) return PNGPD_ERR_UNSUPPORTED;
    if (shape == 0) return lce_launch_z<DT, KIND, 256, 128, 2, 2>(a, st);
    if (shape == 1) return lce_launch_z<DT, KIND, 64, 64, 2, 2>(a, st);
    return lce_launch_z<DT, KIND, 64, 32, 2, 1>(a, st);
}

template <int DT, bool BMC, int BM, int BN, int WGM, int WGN>
static int lce_launch_out(const LceOut &a, int splits, hipStream_t st) {
    constexpr int lds = LceCore<DT, true, BMC, BM, BN, WGM, WGN>::LDS;
    const int rc = pngpd_allow_lds((const void *)lce_out_kernel<DT, BMC, BM, BN, WGM, WGN>, lds);
    if (rc) return rc;
    hipLaunchKernelGGL((lce_out_kernel<DT, BMC, BM, BN, WGM, WGN>), dim3((unsigned)(a.mt * a.nt * splits)), dim3(WGM * WGN * 64), lds, st, a);
    return pngpd_launch_status();
}
template <int DT, bool BMC> static int lce_out(LceOut &a, int shape, int splits, hipStream_t st) {
    a.mt = lce_cdiv(a.M, LCE_BM[shape]); a.nt = lce_cdiv(a.no, LCE_BN[shape]);
    if ((long long)a.mt * a.nt * splits > 0x7fffffffll) return PNGPD_ERR_UNSUPPORTED;
    if (shape == 0) return lce_launch_out<DT, BMC, 256, 128, 2, 2>(a, splits, st);
    if (shape == 1) return lce_launch_out<DT, BMC, 64, 64, 2, 2>(a, splits, st);
    if constexpr (!BMC) return lce_launch_out<DT, BMC, 64, 32, 2, 1>(a, splits, st);
    return PNGPD_ERR_UNSUPPORTED;
}

template <int DT>
static void lce_copy(const Lce *a, const void *src, long long ld, long long R, const long long *target, void *dst, hipStream_t st) {
    const int Dp = lce_dp(a);
    const long long n = R * (Dp * lce_esize(DT) / 16);
    hipLaunchKernelGGL(lce_copy_kernel<DT>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, src, ld, a->D, Dp, R, target,
                       a->ignore_index, dst);
}

static LceArgs lce_args(const Lce *a) {
    LceArgs k = {};
    k.x = LceOperand{a->x, a->ldx}; k.w = LceOperand{a->w, a->ldw};
    k.bias = a->bias; k.bf32 = a->bias_dtype == PNGPD_F32; k.target = (const long long *)a->target; k.ignore = a->ignore_index;
    k.T = a->T; k.D = a->D; k.V = a->V; k.smooth = a->smoothing;
    return k;
}

template <int DT> static int lce_forward(const Lce *a, const LcePlan &p, hipStream_t st) {
    char *ws = (char *)a->workspace;
    LceArgs k = lce_args(a);
    if (p.padx) { lce_copy<DT>(a, a->x, a->ldx, a->T, nullptr, ws + p.o_x, st); k.x = LceOperand{ws + p.o_x, p.Dp}; }
    if (p.padw) { lce_copy<DT>(a, a->w, a->ldw, a->V, nullptr, ws + p.o_w, st); k.w = LceOperand{ws + p.o_w, p.Dp}; }
    k.D = p.Dp;
    k.pm = (float *)(ws + p.o_part); k.ps = (float *)(ws + p.o_ps); k.zt = (float *)(ws + p.o_zt);
    int rc = lce_z<DT, 0>(k, p.fshape, a->V, st);
    if (rc) return rc;
    float *row = a->reduction == PNGPD_REDUCE_NONE ? a->loss : (float *)(ws + p.o_row);
    hipLaunchKernelGGL(lce_join_kernel, dim3((unsigned)((a->T + 31) / 32)), dim3(256), 0, st, k, a->stat, row);
    if (a->reduction != PNGPD_REDUCE_NONE)
        hipLaunchKernelGGL(lce_loss_kernel, dim3(1), dim3(1024), 0, st, row, k.target, k.ignore, a->T, a->reduction, a->loss, a->kept);
    return pngpd_launch_status();
}

template <int DT> static int lce_backward(const Lce *a, const LcePlan &p, hipStream_t st) {
    typedef typename elem<DT>::t E;
    char *ws = (char *)a->workspace;
    LceArgs k = lce_args(a);
    lce_copy<DT>(a, a->x, a->ldx, a->T, k.target, ws + p.o_x, st);
    k.x = LceOperand{ws + p.o_x, p.Dp};
    if (p.padw) { lce_copy<DT>(a, a->w, a->ldw, a->V, nullptr, ws + p.o_w, st); k.w = LceOperand{ws + p.o_w, p.Dp}; }
    k.D = p.Dp;
    float *coef = (float *)(ws + p.o_coef), *scale = (float *)(ws + p.o_scale), *part = (float *)(ws + p.o_dx);
    hipLaunchKernelGGL(lce_coef_kernel, dim3(1), dim3(1024), 0, st, a->dloss, a->kept, k.target, k.ignore, a->T, a->V, a->reduction,
                       DT == PNGPD_F16 ? 32768.f : 1.f, coef, scale);
    k.stat = a->stat; k.coef = coef; k.g = ws + p.o_g; k.ldg = p.ldg;
    for (int v0 = 0; v0 < a->V; v0 += p.piece) {
        k.v0 = v0; k.vc = a->V - v0 < p.piece ? a->V - v0 : p.piece;
        const int cols = (k.vc + 63) / 64 * 64;                    // columns of g that are written (zeros past vc)
        int rc = lce_z<DT, 1>(k, p.gshape, k.vc, st);
        if (rc) return rc;
        const E *w = (const E *)k.w.p + (long long)v0 * k.w.ld;
        if (a->db) {
            void *db = a->bias_dtype == PNGPD_F32 ? (void *)((float *)a->db + v0) : (void *)((E *)a->db + v0);
            hipLaunchKernelGGL(lce_db_kernel<DT>, dim3((unsigned)(cols / 64)), dim3(1024), 0, st, k.g, a->T, k.vc, p.ldg, scale, db,
                               a->bias_dtype == PNGPD_F32);
        }
        if (a->dx) {
            LceOut o = {};
            o.a = LceOperand{w, k.w.ld}; o.b = LceOperand{k.g, p.ldg};
            o.M = p.Dp; o.N = a->T; o.mo = a->D; o.no = a->T; o.K = k.vc; o.kper = p.kper;
            o.part = part; o.add = v0 > 0; o.scale = scale;
            if ((rc = lce_out<DT, false>(o, p.xshape, p.splits, st))) return rc;
        }
        if (a->dw) {
            LceOut o = {};
            o.a = LceOperand{k.x.p, p.Dp}; o.b = LceOperand{k.g, p.ldg};
            o.M = p.Dp; o.N = cols; o.mo = a->D; o.no = k.vc; o.K = a->T; o.kper = a->T;
            o.out = (E *)a->dw + (long long)v0 * a->D; o.ldo = a->D; o.scale = scale;
            o.vec = a->D % 4 == 0 && !((uintptr_t)a->dw & 15);
            if ((rc = lce_out<DT, true>(o, p.wshape, 1, st))) return rc;
        }
    }
    if (a->dx) {
        const long long n = (long long)a->T * (p.Dp / 4);
        hipLaunchKernelGGL(lce_dx_kernel<DT>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, part, p.splits, a->T, a->D, p.Dp,
                           scale, a->dx);
    }
    return pngpd_launch_status();
}

extern "C" {

size_t pngpd_lce_workspace_bytes(const pngpd_lce_t *a, int backward) {
    return lce_bad(a) ? 0 : lce_plan(a, backward != 0).bytes;
}

int pngpd_lce_fwd(const pngpd_lce_t *a, void *stream) {
    if (lce_bad(a) || !a->loss) return PNGPD_ERR_INVALID_ARG;
    const LcePlan p = lce_plan(a, false);
    if (!a->workspace || ((uintptr_t)a->workspace & 255) || a->workspace_bytes < p.bytes) return PNGPD_ERR_WORKSPACE;
    hipStream_t st = (hipStream_t)stream;
    if (a->dtype == PNGPD_F32) return lce_forward<PNGPD_F32>(a, p, st);
    if (a->dtype == PNGPD_BF16) return lce_forward<PNGPD_BF16>(a, p, st);
    return lce_forward<PNGPD_F16>(a, p, st);
}

int pngpd_lce_bwd(const pngpd_lce_t *a, void *stream) {
    if (lce_bad(a) || !a->dloss || (a->db && !a->bias)) return PNGPD_ERR_INVALID_ARG;
    if (!a->dx && !a->dw && !a->db) return PNGPD_OK;
    const LcePlan p = lce_plan(a, true);
    if (!a->workspace || ((uintptr_t)a->workspace & 255) || a->workspace_bytes < p.bytes) return PNGPD_ERR_WORKSPACE;
    hipStream_t st = (hipStream_t)stream;
    if (a->dtype == PNGPD_F32) return lce_backward<PNGPD_F32>(a, p, st);
    if (a->dtype == PNGPD_BF16) return lce_backward<PNGPD_BF16>(a, p, st);
    return lce_backward<PNGPD_F16>(a, p, st);
}

}  // extern "C"
