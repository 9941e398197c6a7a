// Group norm with an activation over channels-last features, forward and backward.
//
//   x (B,N,C), group g of sample b = the channels [g Cg, (g+1) Cg) of all N rows, m = N Cg values:
//     mean = sum x / m      var = sum x^2 / m - mean^2      rstd = 1/sqrt(var + eps)      (sums in fp64)
//     xh = (x - mean) rstd      z = xh w_c + b_c      y = act(z)
//   dz = dy act'(z)      A_c = sum_n dz      B_c = sum_n dz xh      db_c = sum_b A_c      dw_c = sum_b B_c
//     S1 = sum_c w_c A_c / m      S2 = sum_c w_c B_c / m      dx = rstd (w_c dz - S1 - xh S2)
//
// Memory-bound: x is read and y written once forward, x and dy read and dx written once backward.  Two forms:
//   * slab: one workgroup owns the N rows of a few whole groups of one sample (32 bytes of a row to all of it; of short
//     samples, several) and holds them in REGISTERS between the sums and the output: each byte moves once, one launch;
//   * split: groups too large for that (a 50,000-point scene) are cut along N over workgroups: partial sums, a tiny
//     launch that joins them, a second walk over the data.
// A thread owns a fixed 16-byte column of channels, so w, b and the group's statistics sit in its registers, and the
// per-channel sums of the backward pass need no transposition.  Columns may start anywhere (Cg is any number): gfx950
// loads 16 bytes from any element's address; the ragged last column of a range goes element by element.
// The sums of x and x^2 are fp64: a cloud's coordinates-like features have means many times their spread, where a
// float32 E[x^2] - mean^2 loses the variance; memory hides the fp64 rate.  relu's slope is taken from a z in fp64 (its
// statistics are kept in fp64 for that): it jumps at 0, and a value next to it would otherwise take either side.
// Measured (a large copy reaches 4.9 TB/s on this card): bf16, 1024 samples of 1024 x 128 in 32 groups, gelu: forward 170 us
// (537 MB, 3.2 TB/s; the vector pipe is busy for 65 % of it, 29 instructions a value, the rest is loads and stores that little else
// of a workgroup overlaps), backward 286 us (805 MB, 2.8 TB/s; busy for 52 %, 39 a value; a workgroup's 32-byte pieces of a row
// reach memory with 26 % more writes); float32, 64 of 750 x 128: 16 and 18 + 4 us; fp16, one sample of 50,000 x 1024: forward
// 18 + 6 + 36 us, backward 46 + 6 + 60 (102 MB a walk; the second walk finds part of it in the last-level cache).
#include "pngpd_common.h"
#include "pngpd_types.h"

#define SLAB_THREADS 512                // of a slab's workgroup: two share a CU, one loads while the other computes

struct GnArgs {
    const void *x, *dy, *w, *b;
    void *y, *dx, *dw, *db;        // dw, db: where A, B of one row of ab are theirs, or NULL
    double *stats;                 // (B,G,2): mean, rstd
    float *ab;                     // (nab,C,2): A, B of a sample, or of the samples of one workgroup
    double *part;                  // split form: (B,S,units,2) sums;  backward: (B,S,C,2) as float
    float *gsum;                   // split form, backward: (B,G,2): S1, S2
    float *folded;                 // (fold,C,2): A, B of GN_FOLD neighbours of ab
    long long sB, sN;              // strides of x (elements)
    int B, N, C, G, Cg, act, wf32; // wf32: w, b are float32 (else of x's type)
    float eps;
    int lx;                        // log2 of the columns of a workgroup
    int gpr, ranges;               // slab: groups of a workgroup, workgroups of a sample
    int spw, cps;                  // slab: samples side by side in a workgroup, columns of one of them
    int per, nab;                  // slab, backward: times that a workgroup takes spw samples; rows of ab
    int cols, S, rows;             // split: column blocks, cuts of N, rows of one
};

// ---------------------------------------------------------------- columns of VEC elements, 16 bytes (or one element)
template <int DT, int VEC> struct Col {
    static constexpr int WORDS = VEC == 1 ? 1 : 4;
    unsigned q[WORDS];
    __device__ __forceinline__ float get(int e) const {
        if constexpr (DT == PNGPD_F32) return __uint_as_float(q[e]);
        else return half_to_f(DT, (u16)(q[e >> 1] >> (16 * (e & 1))));
    }
    // n of the VEC elements exist; the others read as 0
    __device__ __forceinline__ void load(const typename elem<DT>::t *p, int n) {
        if (VEC > 1 && n == VEC) { __builtin_memcpy(q, p, 16); return; }
        load_tail(p, n);
    }
    __device__ __forceinline__ void load_tail(const typename elem<DT>::t *p, int n) {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) q[i] = 0u;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            if (e < n) {
                if constexpr (DT == PNGPD_F32) q[e] = __float_as_uint(p[e]);
                else q[e >> 1] |= (unsigned)p[e] << (16 * (e & 1));
            }
        }
    }
    // adds the values (and their squares) of each SUB-th part to s, s2, all in fp64: float32 sums of 16-bit squares cost the
    // same time (bf16, 1024 samples of 1024 x 128, forward + backward: 433 and 432 us) and lose what var subtracts: eight
    // squares of float16 values near each other need 25 bits, and bfloat16 ones pass float32's range
    template <int SUB> __device__ __forceinline__ void sums(double (&s)[SUB], double (&s2)[SUB]) const {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const double v = (double)get(e);
            const int k = e * SUB / VEC;
            s[k] += v; s2[k] = fma(v, v, s2[k]);
        }
    }
    static __device__ __forceinline__ void store(typename elem<DT>::t *p, const float (&v)[VEC], int n) {
        if (VEC > 1 && n == VEC) {
            unsigned o[WORDS];
#pragma unroll
            for (int i = 0; i < WORDS; ++i) {
                if constexpr (DT == PNGPD_F32) o[i] = __float_as_uint(v[i]);
                else o[i] = pk_half<DT>(v[(2 * i) % VEC], v[(2 * i + 1) % VEC]);
            }
            __builtin_memcpy(p, o, 16);
            return;
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) if (e < n) st_elem<DT>(p + e, v[e]);
    }
};

// K rows row, row + step, ... of a column; a row at or past `end` reads row `row0` (which exists) in its place
template <int K, int DT, int VEC>
__device__ __forceinline__ void load_rows(Col<DT, VEC> (&q)[K], const typename elem<DT>::t *p, long long stride, int row,
                                          int step, int end, int n, int row0 = 0) {
    if (VEC > 1 && n == VEC) {
#pragma unroll
        for (int i = 0; i < K; ++i) {
            const int at = row + i * step;
            __builtin_memcpy(q[i].q, p + (long long)(at < end ? at : row0) * stride, 16);
        }
    } else {
#pragma unroll
        for (int i = 0; i < K; ++i) {
            const int at = row + i * step;
            q[i].load_tail(p + (long long)(at < end ? at : row0) * stride, n);
        }
    }
}

// ---------------------------------------------------------------- activations
// Phi(z), the normal distribution, and e = exp(-z^2/2): erf by Abramowitz & Stegun 7.1.26 (|error| < 1.5e-7), whose
// exponential is the density's too; 14 instructions where erff takes both its branches in a divergent wave.
__device__ __forceinline__ float phi_cdf(float z, float &e) {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f * 0.70710678118654752f, fabsf(z), 1.f));
    e = __builtin_amdgcn_exp2f(z * z * (-0.5f * 1.44269504088896340736f));
    const float p = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f), 0.5f * 1.421413741f),
                                     0.5f * -0.284496736f), 0.5f * 0.254829592f);
    const float tail = p * e;
    return z < 0.f ? tail : 1.f - tail;
}
__device__ __forceinline__ float sigmoid(float z) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.44269504088896340736f));
}
// ACT: PNGPD_ACT_*
template <int ACT> __device__ __forceinline__ float act_value(float z) {
    float e;
    if constexpr (ACT == PNGPD_ACT_RELU) return z < 0.f ? 0.f : z;                  // NaN passes
    else if constexpr (ACT == PNGPD_ACT_SILU) return z * sigmoid(z);
    else if constexpr (ACT == PNGPD_ACT_GELU) return z * phi_cdf(z, e);
    else return z;
}

// What a thread keeps of its column: w, b and, for each of the SUB groups it touches, the statistics.  SUB = 1: the column
// lies inside one group (Cg a multiple of VEC); 2: it is two whole groups; VEC: every element may belong to another one.
// With d = x - (the mean rounded to float32), xh = d r + c and z = d w' + b' (FOLD) are one FMA each; c and b' hold what the
// rounded mean leaves out, so the error is of |d|'s size and not of the mean's (two nearly equal values make a group too).
template <int VEC, int SUB> struct ColPar {
    float w[VEC], b[VEC];
    float m[SUB], r[SUB], c[SUB];          // mean, rstd, -(mean - m) rstd
    static __device__ __forceinline__ int sub(int e) { return e * SUB / VEC; }
};
template <int DT, int VEC, int SUB>
__device__ __forceinline__ void load_wb(const GnArgs &a, int c, int n, ColPar<VEC, SUB> &p) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        p.w[e] = 1.f; p.b[e] = 0.f;
        if (e < n) {
            if (a.w) p.w[e] = a.wf32 ? ((const float *)a.w)[c + e] : ld_elem<DT>((const typename elem<DT>::t *)a.w + c + e);
            if (a.b) p.b[e] = a.wf32 ? ((const float *)a.b)[c + e] : ld_elem<DT>((const typename elem<DT>::t *)a.b + c + e);
        }
    }
}
// statistics of the column's groups out of st (mean, rstd pairs), whose first entry is group g0; fold: w, b become w', b'
template <bool FOLD, int VEC, int SUB>
__device__ __forceinline__ void load_stats(const GnArgs &a, const double *st, int c, int n, int g0, ColPar<VEC, SUB> &p) {
#pragma unroll
    for (int k = 0; k < SUB; ++k) {
        const int at = k * (VEC / SUB);
        double mean = 0.0, rstd = 0.0;
        if (at < n) {
            const int g = (c + at) / a.Cg - g0;
            mean = st[2 * g]; rstd = st[2 * g + 1];
        }
        p.m[k] = (float)mean; p.r[k] = (float)rstd;
        const double c = -(mean - (double)p.m[k]) * rstd;
        p.c[k] = (float)c;
        if constexpr (FOLD) {
#pragma unroll
            for (int e = at; e < at + VEC / SUB; ++e) {
                p.b[e] = (float)((double)p.b[e] + c * (double)p.w[e]);
                p.w[e] = (float)(rstd * (double)p.w[e]);
            }
        }
    }
}
template <int ACT, int VEC, int SUB>
__device__ __forceinline__ void gn_apply(const ColPar<VEC, SUB> &p, const float (&x)[VEC], float (&y)[VEC]) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) y[e] = act_value<ACT>(fmaf(x[e] - p.m[p.sub(e)], p.w[e], p.b[e]));
}
// dz of one element; st: the fp64 statistics (mean, rstd) of its group, for relu's slope
template <int ACT>
__device__ __forceinline__ float gn_dz(float x, float xh, float dy, float w, float b, const double *st) {
    if constexpr (ACT == PNGPD_ACT_NONE) return dy;
    else if constexpr (ACT == PNGPD_ACT_RELU) return fma(((double)x - st[0]) * st[1], (double)w, (double)b) <= 0.0 ? 0.f : dy;
    else {
        const float z = fmaf(xh, w, b);
        if constexpr (ACT == PNGPD_ACT_SILU) { const float s = sigmoid(z); return dy * (s * fmaf(z, 1.f - s, 1.f)); }
        else { float e; const float s = phi_cdf(z, e); return dy * fmaf(z * 0.39894228040143268f, e, s); }
    }
}
// dx = rstd (w dz - S1 - xh S2) = r (w dz + d k1 + k0); r outside: r^2 leaves float32's range where spreads pass 1e19 or, with
// eps = 0, lie below 1e-19
template <int VEC, int SUB> struct DxPar {
    float w[VEC], r[SUB], k0[SUB], k1[SUB];
    // S: (S1, S2) of the column's groups in turn
    __device__ __forceinline__ void set(const ColPar<VEC, SUB> &p, int k, double S1, double S2) {
        r[k] = p.r[k];
        k1[k] = (float)(-(double)p.r[k] * S2);
        k0[k] = (float)(-(S1 + (double)p.c[k] * S2));
#pragma unroll
        for (int e = k * (VEC / SUB); e < (k + 1) * (VEC / SUB); ++e) w[e] = p.w[e];
    }
    __device__ __forceinline__ float dx(int e, float d, float dz) const {
        const int k = ColPar<VEC, SUB>::sub(e);
        return r[k] * fmaf(dz, w[e], fmaf(d, k1[k], k0[k]));
    }
};

// Sums of NV values of each column (tx) over the workgroup's rows: res[tx NV + v], in LDS (NV (threads + 64) values of
// scratch before res).  Every thread writes its values, conflict-free, and a group of lanes adds a column's up: NV reads and
// a few exchanges a thread, where sums over lanes alone exchange every value log2 times.  Fixed order.
template <class T, int NV> __device__ __forceinline__ T *cols_sum(T *sh, const T (&v)[NV], int lx) {
    const int tid = threadIdx.x, threads = blockDim.x, X = 1 << lx, TY = threads >> lx, pitch = TY + (64 >> lx);
    const int tx = tid & (X - 1), ty = tid >> lx;
#pragma unroll
    for (int i = 0; i < NV; ++i) sh[(i * X + tx) * pitch + ty] = v[i];
    __syncthreads();
    const int outs = NV * X;
    T *res = sh + NV * (threads + 64);
    int L = threads / outs;                               // lanes of an output (a power of two)
    if (L > 64) L = 64;
    if (L < 1) L = 1;
    for (int o = tid / L; o < outs; o += threads / L) {
        const T *c = sh + o * pitch;
        T u = 0;
        for (int k = tid & (L - 1); k < TY; k += L) u += c[k];
        for (int k = 1; k < L; k <<= 1) u += __shfl_xor(u, k);
        if ((tid & (L - 1)) == 0) res[(o & (X - 1)) * NV + (o >> lx)] = u;
    }
    __syncthreads();
    return res;
}

// sum over the lanes of a wave that hold the same column (lane ^ (1 << lx), ... )
template <class T> __device__ __forceinline__ T lanes_sum(T v, int lx) {
    for (int k = 1 << lx; k < 64; k <<= 1) v += __shfl_xor(v, k);
    return v;
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int k = 32; k >= 1; k >>= 1) v += __shfl_xor(v, k);
    return v;
}

// lanes that add up n values together: a power of two of at least n, at most a wave; as its logarithm
__device__ __forceinline__ int lanes_for(int n) { return n <= 1 ? 0 : min(6, 32 - __clz(n - 1)); }
__device__ __forceinline__ double part_sum(double v, int ll) {
    for (int k = 1; k < 1 << ll; k <<= 1) v += __shfl_xor(v, k);
    return v;
}

// ranges of one sample stay on one XCD (workgroup i runs on XCD i % 8): neighbouring ranges share cache lines
__device__ __forceinline__ int slab_item(int i, int ranges, int total) {
    const int whole = total / (8 * ranges) * (8 * ranges);
    if (i >= whole) return i;
    const int k = i >> 3;
    return (k / ranges) * 8 * ranges + (i & 7) * ranges + k % ranges;
}

// ---------------------------------------------------------------------------------------------- slab form
// MANY: a.spw samples side by side.  Otherwise the sample is the same in all lanes, and so are the addresses' bases (float32,
// 1024 samples of 1024 x 128: 253 us, and 313 with a base in every lane).
template <int DT, int VEC, int SUB, int RPT, int ACT, bool MANY>
__global__ __launch_bounds__(SLAB_THREADS) void gn_fwd_slab_kernel(const GnArgs a) {
    typedef typename elem<DT>::t T;
    extern __shared__ double sh[];
    const int tid = threadIdx.x, X = 1 << a.lx, tx = tid & (X - 1), ty = tid >> a.lx, TY = blockDim.x >> a.lx;
    const int item = slab_item(blockIdx.x, a.ranges, gridDim.x), ib = item / a.ranges, r = item - ib * a.ranges;
    const int g0 = r * a.gpr, gn = min(a.gpr, a.G - g0), c0 = g0 * a.Cg, c1 = c0 + gn * a.Cg;
    const int sb = MANY ? tx / a.cps : 0, c = c0 + (tx - sb * a.cps) * VEC;
    const int b0 = MANY ? ib * a.spw : ib, b = b0 + sb, have = MANY ? min(a.spw, a.B - b0) : 1;
    const int n = sb < have ? max(0, min(VEC, c1 - c)) : 0;
    const T *x = (const T *)a.x + (long long)b * a.sB + c;
    Col<DT, VEC> q[RPT];                                  // rows past the last one: row 0 again, never used
    load_rows<RPT>(q, x, a.sN, ty, TY, a.N, n);
    ColPar<VEC, SUB> p;
    load_wb<DT>(a, c, n, p);
    double s[SUB], s2[SUB], all[2 * SUB];
#pragma unroll
    for (int e = 0; e < SUB; ++e) { s[e] = 0.0; s2[e] = 0.0; }
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
        if (ty + i * TY < a.N) q[i].sums(s, s2);
    }
#pragma unroll
    for (int e = 0; e < SUB; ++e) { all[2 * e] = s[e]; all[2 * e + 1] = s2[e]; }
    const double *res = cols_sum(sh, all, a.lx);          // [column][part][sum, squares]
    double *st = sh + 2 * SUB * (blockDim.x + 64) + 2 * SUB * X;
    const int upg = a.Cg * SUB / VEC;                     // parts of a group
    const double m = (double)a.N * a.Cg;
    const int ll = lanes_for(upg), lane = tid & ((1 << ll) - 1);
    for (int i = tid >> ll; i < have * gn; i += blockDim.x >> ll) {
        const int is = MANY ? i / gn : 0, g = i - is * gn;
        double u = 0.0, v = 0.0;
        for (int k = lane; k < upg; k += 1 << ll) {
            const double *o = res + 2 * ((size_t)is * a.cps * SUB + g * upg + k);
            u += o[0]; v += o[1];
        }
        u = part_sum(u, ll); v = part_sum(v, ll);
        if (lane == 0) {
            const double mean = u / m;
            double var = v / m - mean * mean;
            var = var < 0.0 ? 0.0 : var;                  // NaN passes
            const double rstd = 1.0 / sqrt(var + (double)a.eps);
            st[2 * i] = mean; st[2 * i + 1] = rstd;
            double *o = a.stats + 2 * ((size_t)(b0 + is) * a.G + g0 + g);
            o[0] = mean; o[1] = rstd;
        }
    }
    __syncthreads();
    load_stats<true>(a, st + 2 * sb * gn, c, n, g0, p);
    T *y = (T *)a.y + (size_t)b * a.N * a.C + c;
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
        const int row = ty + i * TY;
        if (row < a.N && n > 0) {
            float v[VEC], o[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = q[i].get(e);
            gn_apply<ACT>(p, v, o);
            Col<DT, VEC>::store(y + (size_t)row * a.C, o, n);
        }
    }
}

// a channel's gradient, of w's and b's type; to NULL: none
template <int DT> __device__ __forceinline__ void gn_store(const GnArgs &a, void *to, size_t c, float v) {
    if (!to) return;
    if (a.wf32) ((float *)to)[c] = v; else st_elem<DT>((typename elem<DT>::t *)to + c, v);
}

// The samples b0 .. b0 + have - 1 (without MANY: one); dz stays in registers (float32) between the sums and dx where its
// slope is dear (silu, gelu); none and relu take dy again.  sum: A, B of the channels tid + i threads over the samples so far.
template <int DT, int VEC, int SUB, int RPT, int ACT, bool MANY>
__device__ __forceinline__ void gn_bwd_samples(const GnArgs &a, double *sh, int ib, int r, int b0, int have, bool first, bool last,
                                               double (&sum)[MANY ? VEC : 1][2]) {
    typedef typename elem<DT>::t T;
    constexpr bool KEEP = ACT == PNGPD_ACT_SILU || ACT == PNGPD_ACT_GELU;
    const int tid = threadIdx.x, X = 1 << a.lx, tx = tid & (X - 1), ty = tid >> a.lx, TY = blockDim.x >> a.lx;
    const int g0 = r * a.gpr, gn = min(a.gpr, a.G - g0), c0 = g0 * a.Cg, c1 = c0 + gn * a.Cg, nc = c1 - c0;
    const int sb = MANY ? tx / a.cps : 0, c = c0 + (tx - sb * a.cps) * VEC, b = b0 + sb;
    const int n = sb < have ? max(0, min(VEC, c1 - c)) : 0;
    double *st = sh + VEC * (blockDim.x + 64 + X);        // [samples][gn][2]: S1, S2   (behind 2 VEC (threads + 64 + X) floats)
    const T *x = (const T *)a.x + (long long)b * a.sB + c;
    const T *dy = (const T *)a.dy + (size_t)b * a.N * a.C + c;
    const double *stats = a.stats + 2 * ((size_t)b * a.G + g0);
    Col<DT, VEC> q[RPT], d[RPT];
    load_rows<RPT>(q, x, a.sN, ty, TY, a.N, n);
    load_rows<RPT>(d, dy, a.C, ty, TY, a.N, n);
    ColPar<VEC, SUB> p;
    load_wb<DT>(a, c, n, p);
    load_stats<false>(a, stats, c, n, g0, p);
    float A[VEC], Bs[VEC], keep[KEEP ? RPT : 1][VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) { A[e] = 0.f; Bs[e] = 0.f; }
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
        if (ty + i * TY < a.N && n > 0) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const int k = p.sub(e);
                const float xv = q[i].get(e), xh = fmaf(xv - p.m[k], p.r[k], p.c[k]);
                const double *st = stats + 2 * (ACT == PNGPD_ACT_RELU ? (c + min(e, n - 1)) / a.Cg - g0 : 0);
                const float dz = gn_dz<ACT>(xv, xh, d[i].get(e), p.w[e], p.b[e], st);
                if constexpr (KEEP) keep[i][e] = dz;
                A[e] += dz; Bs[e] = fmaf(dz, xh, Bs[e]);
            }
        }
    }
    float all[2 * VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) { all[2 * e] = A[e]; all[2 * e + 1] = Bs[e]; }
    const float *res = cols_sum((float *)sh, all, a.lx);  // [column][e][A, B]
#pragma unroll
    for (int i = 0; i < (MANY ? VEC : 1); ++i) {
        for (int k = tid + i * blockDim.x; k < nc; k += MANY ? nc : blockDim.x) {
            double u = MANY && !first ? sum[i][0] : 0.0, v = MANY && !first ? sum[i][1] : 0.0;
            for (int is = 0; is < have; ++is) {
                const float *o = res + 2 * (is * a.cps * VEC + k);
                u += (double)o[0]; v += (double)o[1];
            }
            if constexpr (MANY) { sum[i][0] = u; sum[i][1] = v; }
            if (a.ab && last) {
                const size_t ch = (size_t)ib * a.C + c0 + k;
                a.ab[2 * ch] = (float)u; a.ab[2 * ch + 1] = (float)v;
                gn_store<DT>(a, a.db, ch, (float)u); gn_store<DT>(a, a.dw, ch, (float)v);
            }
        }
    }
    const double m = (double)a.N * a.Cg;
    const int ll = lanes_for(a.Cg), lane = tid & ((1 << ll) - 1);
    for (int i = tid >> ll; i < have * gn; i += blockDim.x >> ll) {
        const int is = MANY ? i / gn : 0, g = i - is * gn;
        const float *o = res + 2 * (is * a.cps * VEC + g * a.Cg);
        double u = 0.0, v = 0.0;
        for (int k = lane; k < a.Cg; k += 1 << ll) {
            const int ch = c0 + g * a.Cg + k;
            const double w = !a.w ? 1.f : a.wf32 ? ((const float *)a.w)[ch] : ld_elem<DT>((const T *)a.w + ch);
            u += (double)o[2 * k] * w; v += (double)o[2 * k + 1] * w;
        }
        u = part_sum(u, ll); v = part_sum(v, ll);
        if (lane == 0) { st[2 * i] = u / m; st[2 * i + 1] = v / m; }
    }
    __syncthreads();
    if (n > 0 && a.dx) {
        DxPar<VEC, SUB> dp;
#pragma unroll
        for (int k = 0; k < SUB; ++k) {
            const int g = sb * gn + (c + min(k * (VEC / SUB), n - 1)) / a.Cg - g0;
            dp.set(p, k, st[2 * g], st[2 * g + 1]);
        }
        T *dx = (T *)a.dx + (size_t)b * a.N * a.C + c;
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            const int row = ty + i * TY;
            if (row < a.N) {
                float o[VEC];
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float xv = q[i].get(e);
                    const int k = p.sub(e);
                    float dz;
                    if constexpr (KEEP) dz = keep[i][e];
                    else dz = gn_dz<ACT>(xv, 0.f, d[i].get(e), p.w[e], p.b[e],
                                         stats + 2 * (ACT == PNGPD_ACT_RELU ? (c + min(e, n - 1)) / a.Cg - g0 : 0));
                    o[e] = dp.dx(e, xv - p.m[k], dz);
                }
                Col<DT, VEC>::store(dx + (size_t)row * a.C, o, n);
            }
        }
    }
}

// MANY: a workgroup takes spw samples a.per times and keeps its A, B over them (fp64): of many samples of a few rows each the
// sums would otherwise be larger than the data.
template <int DT, int VEC, int SUB, int RPT, int ACT, bool MANY>
__global__ __launch_bounds__(SLAB_THREADS) void gn_bwd_slab_kernel(const GnArgs a) {
    extern __shared__ double sh[];
    const int item = slab_item(blockIdx.x, a.ranges, gridDim.x), ib = item / a.ranges, r = item - ib * a.ranges;
    double sum[MANY ? VEC : 1][2];
    if constexpr (!MANY) gn_bwd_samples<DT, VEC, SUB, RPT, ACT, MANY>(a, sh, ib, r, ib, 1, true, true, sum);
    else {
        const long long span = (long long)a.per * a.spw, from = ib * span, to = min((long long)a.B, from + span);
#pragma unroll 1
        for (long long b0 = from; b0 < to; b0 += a.spw) {
            gn_bwd_samples<DT, VEC, SUB, RPT, ACT, MANY>(a, sh, ib, r, (int)b0, (int)min((long long)a.spw, to - b0), b0 == from,
                                                         b0 + a.spw >= to, sum);
            __syncthreads();                              // the next samples' sums go where these are read
        }
    }
}

// ---------------------------------------------------------------------------------------------- split form
// Workgroups of 256 threads: column block, cut and sample out of one index (a batch may pass a grid's 65535).
__device__ __forceinline__ void split_item(const GnArgs &a, int &col, int &sp, int &b) {
    const int i = blockIdx.x / a.cols;
    col = blockIdx.x - i * a.cols;
    b = i / a.S; sp = i - b * a.S;
}

template <int DT, int VEC, int SUB>
__global__ __launch_bounds__(256) void gn_fwd_part_kernel(const GnArgs a) {
    typedef typename elem<DT>::t T;
    extern __shared__ double sh[];
    const int tid = threadIdx.x, X = 1 << a.lx, tx = tid & (X - 1), ty = tid >> a.lx, TY = 256 >> a.lx;
    const int wave = tid >> 6, lane = tid & 63;
    int col, sp, b;
    split_item(a, col, sp, b);
    const int c = (col * X + tx) * VEC, n = max(0, min(VEC, a.C - c));
    const int r0 = sp * a.rows, r1 = min(a.N, r0 + a.rows);
    const T *x = (const T *)a.x + (long long)b * a.sB + c;
    double s[SUB], s2[SUB];
#pragma unroll
    for (int e = 0; e < SUB; ++e) { s[e] = 0.0; s2[e] = 0.0; }
    for (int row = r0 + ty; row < r1; row += 4 * TY) {
        Col<DT, VEC> q[4];
        load_rows<4>(q, x, a.sN, row, TY, r1, n, row);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (row + i * TY < r1) q[i].sums(s, s2);
        }
    }
    // X <= 64: the rows of a wave by shuffles, the four waves through LDS
    const int units = X * SUB;
#pragma unroll
    for (int e = 0; e < SUB; ++e) {
        const double u = lanes_sum(s[e], a.lx), v = lanes_sum(s2[e], a.lx);
        if (lane < X) {
            double *o = sh + 2 * (wave * units + tx * SUB + e);
            o[0] = u; o[1] = v;
        }
    }
    __syncthreads();
    const int per = VEC / SUB, total = a.C / per;                   // channels of a unit, units of a row
    double *out = a.part + 2 * ((size_t)b * a.S + sp) * total;
    for (int k = tid; k < units; k += 256) {
        const int u = col * units + k;
        if (u < total) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
                out[2 * (size_t)u + j] = (sh[2 * k + j] + sh[2 * (units + k) + j]) + (sh[2 * (2 * units + k) + j] + sh[2 * (3 * units + k) + j]);
        }
    }
}

// one workgroup a (sample, group): statistics from the partial sums; per: channels of a unit
__global__ __launch_bounds__(256) void gn_stats_kernel(const GnArgs a, int per) {
    __shared__ double sh[4][2];
    const int b = blockIdx.x / a.G, g = blockIdx.x - b * a.G, total = a.C / per, upg = a.Cg / per;
    const double *in = a.part + 2 * ((size_t)b * a.S * total + (size_t)g * upg);
    double u = 0.0, v = 0.0;
    for (long long k = threadIdx.x; k < (long long)a.S * upg; k += 256) {
        const long long s = k / upg, j = k - s * upg;
        const double *o = in + 2 * (s * total + j);
        u += o[0]; v += o[1];
    }
    u = wave_sum(u); v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) { sh[threadIdx.x >> 6][0] = u; sh[threadIdx.x >> 6][1] = v; }
    __syncthreads();
    if (threadIdx.x == 0) {
        const double m = (double)a.N * a.Cg;
        const double mean = ((sh[0][0] + sh[1][0]) + (sh[2][0] + sh[3][0])) / m;
        double var = ((sh[0][1] + sh[1][1]) + (sh[2][1] + sh[3][1])) / m - mean * mean;
        var = var < 0.0 ? 0.0 : var;
        a.stats[2 * (size_t)blockIdx.x] = mean;
        a.stats[2 * (size_t)blockIdx.x + 1] = 1.0 / sqrt(var + (double)a.eps);
    }
}

template <int DT, int VEC, int SUB, int ACT>
__global__ __launch_bounds__(256) void gn_fwd_apply_kernel(const GnArgs a) {
    typedef typename elem<DT>::t T;
    const int tid = threadIdx.x, X = 1 << a.lx, tx = tid & (X - 1), ty = tid >> a.lx, TY = 256 >> a.lx;
    int col, sp, b;
    split_item(a, col, sp, b);
    const int c = (col * X + tx) * VEC, n = max(0, min(VEC, a.C - c));
    if (n == 0) return;
    const int r0 = sp * a.rows, r1 = min(a.N, r0 + a.rows);
    ColPar<VEC, SUB> p;
    load_wb<DT>(a, c, n, p);
    const double *stats = a.stats + 2 * (size_t)b * a.G;
    load_stats<true>(a, stats, c, n, 0, p);
    const T *x = (const T *)a.x + (long long)b * a.sB + c;
    T *y = (T *)a.y + (size_t)b * a.N * a.C + c;
    for (int row = r0 + ty; row < r1; row += 4 * TY) {
        Col<DT, VEC> q[4];
        load_rows<4>(q, x, a.sN, row, TY, r1, n, row);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (row + i * TY < r1) {
                float v[VEC], o[VEC];
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[e] = q[i].get(e);
                gn_apply<ACT>(p, v, o);
                Col<DT, VEC>::store(y + (size_t)(row + i * TY) * a.C, o, n);
            }
        }
    }
}

template <int DT, int VEC, int SUB, int ACT>
__global__ __launch_bounds__(256) void gn_bwd_part_kernel(const GnArgs a) {
    typedef typename elem<DT>::t T;
    extern __shared__ double sh[];
    float *shf = (float *)sh;
    const int tid = threadIdx.x, X = 1 << a.lx, tx = tid & (X - 1), ty = tid >> a.lx, TY = 256 >> a.lx;
    const int wave = tid >> 6, lane = tid & 63;
    int col, sp, b;
    split_item(a, col, sp, b);
    const int c = (col * X + tx) * VEC, n = max(0, min(VEC, a.C - c));
    const int r0 = sp * a.rows, r1 = min(a.N, r0 + a.rows);
    ColPar<VEC, SUB> p;
    load_wb<DT>(a, c, n, p);
    const double *stats = a.stats + 2 * (size_t)b * a.G;
    load_stats<false>(a, stats, c, n, 0, p);
    const T *x = (const T *)a.x + (long long)b * a.sB + c;
    const T *dy = (const T *)a.dy + (size_t)b * a.N * a.C + c;
    float A[VEC], Bs[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) { A[e] = 0.f; Bs[e] = 0.f; }
    if (n > 0) {
        for (int row = r0 + ty; row < r1; row += 2 * TY) {
            Col<DT, VEC> q[2], d[2];
            load_rows<2>(q, x, a.sN, row, TY, r1, n, row);
            load_rows<2>(d, dy, a.C, row, TY, r1, n, row);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (row + i * TY < r1) {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const int k = p.sub(e);
                        const float xv = q[i].get(e), xh = fmaf(xv - p.m[k], p.r[k], p.c[k]);
                        const float dz = gn_dz<ACT>(xv, xh, d[i].get(e), p.w[e], p.b[e],
                                                    stats + 2 * (ACT == PNGPD_ACT_RELU ? (c + min(e, n - 1)) / a.Cg : 0));
                        A[e] += dz; Bs[e] = fmaf(dz, xh, Bs[e]);
                    }
                }
            }
        }
    }
    const int chans = X * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        const float u = lanes_sum(A[e], a.lx), v = lanes_sum(Bs[e], a.lx);
        if (lane < X) {
            float *o = shf + 2 * (wave * chans + tx * VEC + e);
            o[0] = u; o[1] = v;
        }
    }
    __syncthreads();
    float *out = (float *)a.part + 2 * ((size_t)b * a.S + sp) * a.C;
    for (int k = tid; k < chans; k += 256) {
        const int ch = col * chans + k;
        if (ch < a.C) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
                out[2 * (size_t)ch + j] = (shf[2 * k + j] + shf[2 * (chans + k) + j]) + (shf[2 * (2 * chans + k) + j] + shf[2 * (3 * chans + k) + j]);
        }
    }
}

// the channels' A, B over `per` neighbours (a sample's cuts, or samples): in (total,C,2), out (total / per, rounded up, C, 2);
// 32 channels x 32 lanes of neighbours a workgroup.  sums: S1, S2 of the groups too (Cg divides 32), in the place of
// gn_bwd_group_kernel; dw, db of an only sample, in the place of gn_dwdb_kernel (one sample of 50,000 x 1024: 5 us each).
template <int DT>
__global__ __launch_bounds__(1024) void gn_bwd_join_kernel(const GnArgs a, const float *in, float *out, int total, int per, int sums) {
    const int C = a.C;
    __shared__ double sh[32][32][2];
    const int cx = threadIdx.x & 31, sy = threadIdx.x >> 5, blocks = (C + 31) / 32;
    const int j = blockIdx.x / blocks, c = (blockIdx.x - j * blocks) * 32 + cx, s0 = j * per, n = min(per, total - s0);
    in += 2 * ((size_t)s0 * C + c);
    double u = 0.0, v = 0.0;
    if (c < C) {
#pragma unroll 4
        for (int s = sy; s < n; s += 32) {
            const f32x2 o = *(const f32x2 *)(in + 2 * (size_t)s * C);
            u += (double)o[0]; v += (double)o[1];
        }
    }
    sh[sy][cx][0] = u; sh[sy][cx][1] = v;
    __syncthreads();
    for (int k = 16; k >= 1; k >>= 1) {
        if (sy < k) { sh[sy][cx][0] += sh[sy + k][cx][0]; sh[sy][cx][1] += sh[sy + k][cx][1]; }
        __syncthreads();
    }
    if (sy) return;
    const float A = (float)sh[0][cx][0], B = (float)sh[0][cx][1];
    if (c < C) {
        float *o = out + 2 * ((size_t)j * C + c);
        o[0] = A; o[1] = B;
        if (a.nab == 1) { gn_store<DT>(a, a.db, c, A); gn_store<DT>(a, a.dw, c, B); }
    }
    if (!sums) return;
    const double w = c >= C || !a.w ? 1.f : a.wf32 ? ((const float *)a.w)[c] : ld_elem<DT>((const typename elem<DT>::t *)a.w + c);
    double S1 = (double)A * w, S2 = (double)B * w;        // (lanes past C: whole groups of them)
    for (int k = 1; k < a.Cg; k <<= 1) { S1 += __shfl_xor(S1, k); S2 += __shfl_xor(S2, k); }
    if (c < C && cx % a.Cg == 0) {
        const double m = (double)a.N * a.Cg;
        float *o = a.gsum + 2 * ((size_t)j * a.G + c / a.Cg);
        o[0] = (float)(S1 / m); o[1] = (float)(S2 / m);
    }
}

// one wave a (sample, group): S1, S2 from its channels' A, B
template <int DT>
__global__ __launch_bounds__(64) void gn_bwd_group_kernel(const GnArgs a) {
    const int b = blockIdx.x / a.G, g = blockIdx.x - b * a.G;
    double u = 0.0, v = 0.0;
    for (int k = threadIdx.x; k < a.Cg; k += 64) {
        const int c = g * a.Cg + k;
        const float *o = a.ab + 2 * ((size_t)b * a.C + c);
        const float w = !a.w ? 1.f : a.wf32 ? ((const float *)a.w)[c] : ld_elem<DT>((const typename elem<DT>::t *)a.w + c);
        u += (double)o[0] * w; v += (double)o[1] * w;
    }
    u = wave_sum(u); v = wave_sum(v);
    if (threadIdx.x == 0) {
        const double m = (double)a.N * a.Cg;
        a.gsum[2 * (size_t)blockIdx.x] = (float)(u / m);
        a.gsum[2 * (size_t)blockIdx.x + 1] = (float)(v / m);
    }
}

template <int DT, int VEC, int SUB, int ACT>
__global__ __launch_bounds__(256) void gn_bwd_apply_kernel(const GnArgs a) {
    typedef typename elem<DT>::t T;
    const int tid = threadIdx.x, X = 1 << a.lx, tx = tid & (X - 1), ty = tid >> a.lx, TY = 256 >> a.lx;
    int col, sp, b;
    split_item(a, col, sp, b);
    const int c = (col * X + tx) * VEC, n = max(0, min(VEC, a.C - c));
    if (n == 0) return;
    const int r0 = sp * a.rows, r1 = min(a.N, r0 + a.rows);
    ColPar<VEC, SUB> p;
    load_wb<DT>(a, c, n, p);
    const double *stats = a.stats + 2 * (size_t)b * a.G;
    load_stats<false>(a, stats, c, n, 0, p);
    DxPar<VEC, SUB> dp;
#pragma unroll
    for (int k = 0; k < SUB; ++k) {
        const float *o = a.gsum + 2 * ((size_t)b * a.G + (c + min(k * (VEC / SUB), n - 1)) / a.Cg);
        dp.set(p, k, (double)o[0], (double)o[1]);
    }
    const T *x = (const T *)a.x + (long long)b * a.sB + c;
    const T *dy = (const T *)a.dy + (size_t)b * a.N * a.C + c;
    T *dx = (T *)a.dx + (size_t)b * a.N * a.C + c;
    for (int row = r0 + ty; row < r1; row += 2 * TY) {
        Col<DT, VEC> q[2], d[2];
        load_rows<2>(q, x, a.sN, row, TY, r1, n, row);
        load_rows<2>(d, dy, a.C, row, TY, r1, n, row);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (row + i * TY < r1) {
                float o[VEC];
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const int k = p.sub(e);
                    const float xv = q[i].get(e), xh = fmaf(xv - p.m[k], p.r[k], p.c[k]);
                    const float dz = gn_dz<ACT>(xv, xh, d[i].get(e), p.w[e], p.b[e],
                                                stats + 2 * (ACT == PNGPD_ACT_RELU ? (c + min(e, n - 1)) / a.Cg : 0));
                    o[e] = dp.dx(e, xv - p.m[k], dz);
                }
                Col<DT, VEC>::store(dx + (size_t)(row + i * TY) * a.C, o, n);
            }
        }
    }
}

// db_c, dw_c = the A_c, B_c of ab (n,C,2) summed in fp64: 4 channels x 64 lanes a workgroup
template <int DT>
__global__ __launch_bounds__(256) void gn_dwdb_kernel(const GnArgs a, const float *ab, int n, void *dw, void *db) {
    __shared__ double sh[64][4][2];
    const int cx = threadIdx.x & 3, ry = threadIdx.x >> 2, c = blockIdx.x * 4 + cx;
    double u = 0.0, v = 0.0;
    if (c < a.C) {
#pragma unroll 4
        for (int b = ry; b < n; b += 64) {
            const f32x2 o = *(const f32x2 *)(ab + 2 * ((size_t)b * a.C + c));
            u += (double)o[0]; v += (double)o[1];
        }
    }
    sh[ry][cx][0] = u; sh[ry][cx][1] = v;
    __syncthreads();
    if (threadIdx.x >= 8) return;
    double s = 0.0;
    const int j = threadIdx.x >> 2;                       // 0: db of channel cx, 1: dw
    for (int k = 0; k < 64; ++k) s += sh[k][cx][j];
    void *to = j ? dw : db;
    if (c < a.C) gn_store<DT>(a, to, c, (float)s);
}

// ---------------------------------------------------------------------------------------------- plan
// rpt rows a thread can hold: forward 16 (64 registers of data), backward 8 of x and of dy.
#define GN_FOLD 256
struct GnPlan { int vec, sub, slab, lx, gpr, ranges, spw, cps, threads, rpt, per, nab, fold, cols, S, rows; };

static inline int log2_up(int n) { int k = 0; while ((1 << k) < n) ++k; return k; }

static GnPlan gn_plan(int B, int N, int C, int G, int dt, int act, int bwd) {
    GnPlan p;
    const int Cg = C / G, e = dt == PNGPD_F32 ? 4 : 2, wide = 16 / e;
    p.vec = C >= wide ? wide : 1;
    p.sub = Cg % p.vec == 0 ? 1 : 2 * Cg == p.vec ? 2 : p.vec;
    // slab: columns of a range = 128 bytes of a row (whole cache lines), or one group where that is more (up to 512
    // columns: 1000 samples of 60 x 1000 in one group, bf16, forward + backward: 233 us, cut by rows 318); halved, down to
    // 32 bytes, while the rows do not fit or there are fewer than 512 workgroups (two a CU: one loads while the other
    // computes).  Rows of a thread: 64 registers of x forward, x and dz (or dy) backward.
    p.slab = 0; p.gpr = p.ranges = p.threads = p.rpt = 0;
    p.per = p.spw = 1; p.nab = B; p.cps = 0;
    // 160 registers a thread where dz is kept for eight 16-bit channels: one workgroup of 512 a CU, three of 256 (bf16, 1024
    // samples of 1024 x 128: 322 and 292 us); otherwise 512 threads, on wider pieces of a row (float32, 64 x 750 x 128:
    // 19.7 and 23.7 us)
    const int most_threads = bwd && dt != PNGPD_F32 && act >= PNGPD_ACT_SILU ? SLAB_THREADS / 2 : SLAB_THREADS;
    for (int most = 8; most <= (bwd ? 8 : 16) && !p.slab; most *= 2) {
        for (int bytes = 128; bytes >= 32; bytes >>= 1) {
            int gpr = bytes / e / Cg;
            if (gpr < 1) gpr = 1;
            if (gpr > G) gpr = G;
            const int cols = (gpr * Cg + p.vec - 1) / p.vec;
            const int lx = log2_up(cols);
            if (lx > 9) break;
            const int ranges = (G + gpr - 1) / gpr;
            const long long need = ((long long)N + most - 1) / most << lx;
            if (need <= most_threads) {
                p.slab = 1; p.gpr = gpr; p.ranges = ranges; p.lx = lx;
                if ((long long)B * ranges >= 512) break;
            }
            if (gpr == 1) break;
        }
    }
    // more than 16 workgroups a CU, of a few rows each: wider ranges, then several samples side by side, up to 256 columns
    // (100,000 samples of 1 x 64, bf16, forward: 256 and 18 us; 20,000 of 1 x 1024 in 32 groups, forward + backward: 1311 and 300)
    while (p.slab && p.ranges > 1 && (long long)B * p.ranges > 4096 && (long long)N << p.lx <= 128) {
        p.gpr = p.gpr * 2 > G ? G : p.gpr * 2;
        p.ranges = (G + p.gpr - 1) / p.gpr;
        p.lx = log2_up((p.gpr * Cg + p.vec - 1) / p.vec);
    }
    if (p.slab) {
        p.cps = (p.gpr * Cg + p.vec - 1) / p.vec;
        while (p.ranges == 1 && B / p.spw > 4096 && (long long)N << p.lx <= 128) {
            p.spw *= 2;
            p.lx = log2_up(p.spw * p.cps);
        }
    }
    if (p.slab) {
        // as many threads as there are rows for, up to SLAB_THREADS; then the rows a thread holds
        long long t = (long long)N << p.lx;
        int th = 64;
        while (th < t && th < most_threads) th <<= 1;
        p.threads = th;
        int r = (int)(((long long)N + (th >> p.lx) - 1) / (th >> p.lx));
        p.rpt = r <= 2 ? 2 : r <= 4 ? 4 : r <= 8 ? 8 : 16;
        // backward of one row or two a thread: 4096 workgroups, each taking more samples in turn
        const long long sets = ((long long)B + p.spw - 1) / p.spw;
        if (bwd && p.rpt == 2 && sets * p.ranges > 4096) p.per = (int)((sets * p.ranges + 4095) / 4096);
        p.nab = (int)((sets + p.per - 1) / p.per);
        p.cols = p.S = p.rows = 0;
    }
    if (!p.slab) {
        const int cols = (C + p.vec - 1) / p.vec;
        p.lx = log2_up(cols);
        if (p.lx > 6) p.lx = 6;
        p.cols = (cols + (1 << p.lx) - 1) >> p.lx;
        // cuts: 1024 workgroups (4 a CU), of at least 4 rows a thread
        const int TY = 256 >> p.lx;
        long long S = 1024 / ((long long)B * p.cols);
        const long long top = ((long long)N + 4 * TY - 1) / (4 * TY);
        if (S > top) S = top;
        if (S < 1) S = 1;
        p.rows = (int)(((long long)N + S - 1) / S);
        p.S = (N + p.rows - 1) / p.rows;
    }
    // dw, db of thousands of sums: GN_FOLD of them at a time first (a second launch, but whole cache lines)
    p.fold = p.nab >= 2048 ? (p.nab + GN_FOLD - 1) / GN_FOLD : 0;
    return p;
}

static size_t gn_part_bytes(const GnPlan &p, int B, int C, int bwd) {
    if (p.slab || (bwd && p.S == 1)) return 0;            // one cut: its sums are the sample's
    return (size_t)B * p.S * (bwd ? (size_t)C * 8 : (size_t)(C / (p.vec / p.sub)) * 16);
}

static size_t gn_ab_bytes(const GnPlan &p, int C) { return ((size_t)p.nab * C * 8 + 255) & ~(size_t)255; }
static size_t gn_gsum_bytes(const GnPlan &p, int B, int G) { return p.slab ? 0 : ((size_t)B * G * 8 + 255) & ~(size_t)255; }

// workgroups of one launch past the grid's (and the kernels' int) range
static bool gn_too_many(const GnPlan &p, int B, int C, int G) {
    const long long most = 0x7fffffffll;
    return p.slab ? (long long)B * p.ranges > most
                  : (long long)p.cols * p.S * B > most || (long long)B * G > most || (long long)B * ((C + 31) / 32) > most;
}

static bool gn_bad(const void *x, int dt, int B, int N, int C, int G, int act, const void *w, int wdt, float eps) {
    return !x || dt < PNGPD_F32 || dt > PNGPD_F16 || B <= 0 || N <= 0 || N > (1 << 30) || C <= 0 || C > (1 << 30) || G <= 0 || C % G ||
           act < PNGPD_ACT_NONE || act > PNGPD_ACT_GELU || !(eps >= 0.f) || (wdt != PNGPD_F32 && wdt != dt);
}

template <class K> static int gn_slab_launch(K kernel, const GnArgs &a, const GnPlan &p, size_t lds, hipStream_t st) {
    const int rc = pngpd_allow_lds((const void *)kernel, lds);
    if (rc) return rc;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(p.nab * p.ranges)), dim3(p.threads), lds, st, a);
    return PNGPD_OK;
}

template <int DT, int VEC, int SUB, int ACT>
static int gn_fwd_launch(GnArgs &a, const GnPlan &p, hipStream_t st) {
    if (p.slab) {
        const size_t lds = (size_t)2 * SUB * (p.threads + 64 + (1 << p.lx)) * 8 + (size_t)p.spw * p.gpr * 16;
        const int rc = p.spw > 1  ? gn_slab_launch(gn_fwd_slab_kernel<DT, VEC, SUB, 2, ACT, true>, a, p, lds, st)
                     : p.rpt == 2 ? gn_slab_launch(gn_fwd_slab_kernel<DT, VEC, SUB, 2, ACT, false>, a, p, lds, st)
                     : p.rpt == 4 ? gn_slab_launch(gn_fwd_slab_kernel<DT, VEC, SUB, 4, ACT, false>, a, p, lds, st)
                     : p.rpt == 8 ? gn_slab_launch(gn_fwd_slab_kernel<DT, VEC, SUB, 8, ACT, false>, a, p, lds, st)
                                  : gn_slab_launch(gn_fwd_slab_kernel<DT, VEC, SUB, 16, ACT, false>, a, p, lds, st);
        return rc ? rc : pngpd_launch_status();
    }
    const dim3 grid((unsigned)(p.cols * p.S * a.B));
    hipLaunchKernelGGL((gn_fwd_part_kernel<DT, VEC, SUB>), grid, dim3(256), (size_t)4 * (1 << p.lx) * SUB * 16, st, a);
    hipLaunchKernelGGL(gn_stats_kernel, dim3((unsigned)(a.B * a.G)), dim3(256), 0, st, a, VEC / SUB);
    hipLaunchKernelGGL((gn_fwd_apply_kernel<DT, VEC, SUB, ACT>), grid, dim3(256), 0, st, a);
    return pngpd_launch_status();
}

template <int DT, int VEC, int SUB, int ACT>
static int gn_bwd_launch(GnArgs &a, const GnPlan &p, void *dw, void *db, hipStream_t st) {
    const int blocks = (a.C + 31) / 32;                   // of a join, for one output row
    if (p.nab == 1) { a.dw = dw; a.db = db; }
    bool done = p.slab && p.nab == 1;                     // dw, db are written
    if (p.slab) {
        const bool many = p.per > 1 || p.spw > 1;
        const size_t lds = (size_t)2 * VEC * (p.threads + 64 + (1 << p.lx)) * 4 + (size_t)p.spw * p.gpr * 16;
        const int rc = many       ? gn_slab_launch(gn_bwd_slab_kernel<DT, VEC, SUB, 2, ACT, true>, a, p, lds, st)
                     : p.rpt == 2 ? gn_slab_launch(gn_bwd_slab_kernel<DT, VEC, SUB, 2, ACT, false>, a, p, lds, st)
                     : p.rpt == 4 ? gn_slab_launch(gn_bwd_slab_kernel<DT, VEC, SUB, 4, ACT, false>, a, p, lds, st)
                                  : gn_slab_launch(gn_bwd_slab_kernel<DT, VEC, SUB, 8, ACT, false>, a, p, lds, st);
        if (rc) return rc;
    } else {
        const dim3 grid((unsigned)(p.cols * p.S * a.B));
        hipLaunchKernelGGL((gn_bwd_part_kernel<DT, VEC, SUB, ACT>), grid, dim3(256), (size_t)4 * (1 << p.lx) * VEC * 8, st, a);
        const bool joined = p.S > 1, sums = joined && a.dx && 32 % a.Cg == 0;
        done = joined && p.nab == 1;
        if (joined) hipLaunchKernelGGL(gn_bwd_join_kernel<DT>, dim3((unsigned)(a.B * blocks)), dim3(1024), 0, st, a, (const float *)a.part,
                                       a.ab, a.B * p.S, p.S, (int)sums);
        if (a.dx) {
            if (!sums) hipLaunchKernelGGL(gn_bwd_group_kernel<DT>, dim3((unsigned)(a.B * a.G)), dim3(64), 0, st, a);
            hipLaunchKernelGGL((gn_bwd_apply_kernel<DT, VEC, SUB, ACT>), grid, dim3(256), 0, st, a);
        }
    }
    if (!done && (dw || db)) {
        const float *ab = a.ab;
        if (p.fold) {
            hipLaunchKernelGGL(gn_bwd_join_kernel<DT>, dim3((unsigned)(p.fold * blocks)), dim3(1024), 0, st, a, ab, a.folded, p.nab, GN_FOLD, 0);
            ab = a.folded;
        }
        hipLaunchKernelGGL(gn_dwdb_kernel<DT>, dim3((unsigned)((a.C + 3) / 4)), dim3(256), 0, st, a, ab, p.fold ? p.fold : p.nab,
                           dw, db);
    }
    return pngpd_launch_status();
}

template <int DT, int VEC, int SUB>
static int gn_launch(GnArgs &a, const GnPlan &p, bool bwd, void *dw, void *db, hipStream_t st) {
#define GN_ACT(A) case A: return bwd ? gn_bwd_launch<DT, VEC, SUB, A>(a, p, dw, db, st) : gn_fwd_launch<DT, VEC, SUB, A>(a, p, st)
    switch (a.act) {
        GN_ACT(PNGPD_ACT_NONE);
        GN_ACT(PNGPD_ACT_RELU);
        GN_ACT(PNGPD_ACT_SILU);
        GN_ACT(PNGPD_ACT_GELU);
    }
#undef GN_ACT
    return PNGPD_ERR_INVALID_ARG;
}
template <int DT, int VEC>
static int gn_launch_vec(GnArgs &a, const GnPlan &p, bool bwd, void *dw, void *db, hipStream_t st) {
    if (p.vec == 1) return gn_launch<DT, 1, 1>(a, p, bwd, dw, db, st);
    return p.sub == 1 ? gn_launch<DT, VEC, 1>(a, p, bwd, dw, db, st) : p.sub == 2 ? gn_launch<DT, VEC, 2>(a, p, bwd, dw, db, st)
                                                                              : gn_launch<DT, VEC, VEC>(a, p, bwd, dw, db, st);
}
static int gn_launch_type(GnArgs &a, int dtype, const GnPlan &p, bool bwd, void *dw, void *db, hipStream_t st) {
    return dtype == PNGPD_F32 ? gn_launch_vec<PNGPD_F32, 4>(a, p, bwd, dw, db, st)
         : dtype == PNGPD_BF16 ? gn_launch_vec<PNGPD_BF16, 8>(a, p, bwd, dw, db, st)
                               : gn_launch_vec<PNGPD_F16, 8>(a, p, bwd, dw, db, st);
}

extern "C" {

size_t pngpd_group_norm_workspace_bytes(int B, int N, int C, int G, int dtype, int act, int backward) {
    if (B <= 0 || N <= 0 || C <= 0 || G <= 0 || C % G || dtype < PNGPD_F32 || dtype > PNGPD_F16) return 0;
    const GnPlan p = gn_plan(B, N, C, G, dtype, act, backward != 0);
    size_t n = (gn_part_bytes(p, B, C, backward != 0) + 255) & ~(size_t)255;
    if (backward) n += gn_ab_bytes(p, C) + gn_gsum_bytes(p, B, G) + (size_t)p.fold * C * 8;
    return n;
}

int pngpd_group_norm_fwd(const void *x, int dtype, int B, int N, int C, long long stride_b, long long stride_n, int G,
                         const void *w, const void *b, int wdtype, float eps, int act, void *y, double *stats,
                         void *workspace, size_t workspace_bytes, void *stream) {
    if (gn_bad(x, dtype, B, N, C, G, act, w, wdtype, eps) || !y || !stats) return PNGPD_ERR_INVALID_ARG;
    const GnPlan p = gn_plan(B, N, C, G, dtype, act, 0);
    if (gn_too_many(p, B, C, G)) return PNGPD_ERR_UNSUPPORTED;
    if (workspace_bytes < pngpd_group_norm_workspace_bytes(B, N, C, G, dtype, act, 0) || (!p.slab && !workspace)) return PNGPD_ERR_WORKSPACE;
    GnArgs a = {};
    a.spw = p.spw; a.cps = p.cps;
    a.x = x; a.w = w; a.b = b; a.y = y; a.stats = stats; a.part = (double *)workspace;
    a.sB = stride_b; a.sN = stride_n; a.B = B; a.N = N; a.C = C; a.G = G; a.Cg = C / G; a.act = act;
    a.wf32 = wdtype == PNGPD_F32; a.eps = eps; a.lx = p.lx; a.gpr = p.gpr; a.ranges = p.ranges; a.cols = p.cols; a.S = p.S; a.rows = p.rows;
    return gn_launch_type(a, dtype, p, false, nullptr, nullptr, (hipStream_t)stream);
}

int pngpd_group_norm_bwd(const void *x, int dtype, int B, int N, int C, long long stride_b, long long stride_n, int G,
                         const void *w, const void *b, int wdtype, float eps, int act, const double *stats,
                         const void *dy, void *dx, void *dw, void *db, void *workspace, size_t workspace_bytes,
                         void *stream) {
    if (gn_bad(x, dtype, B, N, C, G, act, w, wdtype, eps) || !stats || !dy) return PNGPD_ERR_INVALID_ARG;
    if (!dx && !dw && !db) return PNGPD_OK;
    const GnPlan p = gn_plan(B, N, C, G, dtype, act, 1);
    if (gn_too_many(p, B, C, G)) return PNGPD_ERR_UNSUPPORTED;
    if (workspace_bytes < pngpd_group_norm_workspace_bytes(B, N, C, G, dtype, act, 1) || !workspace) return PNGPD_ERR_WORKSPACE;
    GnArgs a = {};
    char *ws = (char *)workspace;
    const size_t part = (gn_part_bytes(p, B, C, 1) + 255) & ~(size_t)255;
    a.x = x; a.dy = dy; a.w = w; a.b = b; a.dx = dx; a.stats = (double *)stats; a.part = (double *)ws;
    a.ab = dw || db || !p.slab ? (float *)(ws + part) : nullptr;
    a.gsum = (float *)(ws + part + gn_ab_bytes(p, C));
    a.folded = (float *)(ws + part + gn_ab_bytes(p, C) + gn_gsum_bytes(p, B, G));
    a.per = p.per; a.nab = p.nab; a.spw = p.spw; a.cps = p.cps;
    if (!p.slab && p.S == 1) a.part = (double *)a.ab;
    a.sB = stride_b; a.sN = stride_n; a.B = B; a.N = N; a.C = C; a.G = G; a.Cg = C / G; a.act = act;
    a.wf32 = wdtype == PNGPD_F32; a.eps = eps; a.lx = p.lx; a.gpr = p.gpr; a.ranges = p.ranges; a.cols = p.cols; a.S = p.S; a.rows = p.rows;
    return gn_launch_type(a, dtype, p, true, dw, db, (hipStream_t)stream);
}

}  // extern "C"
