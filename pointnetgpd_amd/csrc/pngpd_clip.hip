// Global gradient norm over many tensors, clipping in place, and the same inside the flat Adam update.
//
//   norm = (sum |g|^2)^(1/2)  |  sum |g|  |  max |g|      over every element of every tensor
//   c    = min(1, max_norm / (norm + 1e-6)),   g <- c g
//
// Memory-bound: the norm reads every gradient once, the clipping reads and writes it once more (nothing when c = 1:
// multiplying by one changes no bit, so those workgroups leave).  Two launches whatever the number of tensors up to
// CLIP_TABLE: the tensors travel as a table in the kernel arguments (no device-side table, no copy, capturable), a
// workgroup takes 8192-element chunks of the concatenation and finds its tensor by bisection of the chunk prefix.
// A workgroup writes ONE fp64 partial; there are at most CLIP_PARTS + tables of them, and every workgroup of the second
// launch sums them again in the same order (8 KB out of L2) instead of a third launch or an atomic whose order varies.
// fp64 partial sums: the squares of float32 / bfloat16 gradients leave float32's range at 1.8e19 and below 1e-23; the
// conversion and the fp64 FMA (half the fp32 rate) stay under the time of the loads.
// Measured (a large copy reaches 4.9 TB/s here): 220 M bf16 gradients, norm 100 us (4.4 TB/s), scaling 135 us (880 MB moved, half
// of what is read out of the last-level cache); 110 M parameters, norm 113 us (3.9 TB/s), Adam update 605 us (3.1 GB, 5.1 TB/s);
// the 44 gradients of a grasp classifier, 1.6 M float32: 6 + 8 us.
#include <algorithm>
#include <vector>

#include "pngpd_common.h"
#include "pngpd_types.h"

#define CLIP_TABLE 128                 // tensors of one launch: 2.7 KB of kernel arguments
#define CLIP_CHUNK 8192                // elements of one chunk: 32 (fp32) elements a thread
#define CLIP_PARTS 1024                // workgroups of the norm over all launches: 4 per CU, 16 waves x 8 KB in flight

enum { KIND_INF = 0, KIND_L1 = 1, KIND_L2 = 2 };

struct ClipTable {
    void *ptr[CLIP_TABLE];
    long long n[CLIP_TABLE];
    int first[CLIP_TABLE + 1];         // first chunk of every tensor; first[count] = chunks
    unsigned char dt[CLIP_TABLE];
    int count;
};

__device__ __forceinline__ double norm_join(int kind, double a, double b) {
    return kind == KIND_INF ? ((b > a || b != b) ? b : a) : a + b;      // a NaN maximum stays (every comparison fails)
}
__device__ __forceinline__ void norm_add(int kind, double &a, float x) {
    const double d = (double)x;
    if (kind == KIND_L2) a = fma(d, d, a);
    else a = norm_join(kind, a, fabs(d));
}

// sum / max over the 256 threads of the workgroup, in every thread
__device__ __forceinline__ double norm_block(int kind, double a) {
    __shared__ double sh[4];
#pragma unroll
    for (int k = 32; k >= 1; k >>= 1) a = norm_join(kind, a, __shfl_xor(a, k));
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = a;
    __syncthreads();
    return norm_join(kind, norm_join(kind, sh[0], sh[1]), norm_join(kind, sh[2], sh[3]));
}

// the tensor of a chunk: largest i with first[i] <= c (tables hold no empty tensor)
__device__ __forceinline__ int clip_find(const ClipTable &t, int c) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= c) lo = mid; else hi = mid - 1;
    }
    return lo;
}

template <int KIND>
__global__ __launch_bounds__(256) void grad_norm_kernel(const ClipTable t, double *__restrict__ part) {
    double a0 = 0.0, a1 = 0.0;
    for (int c = blockIdx.x; c < t.first[t.count]; c += gridDim.x) {
        const int i = clip_find(t, c);
        const long long at = (long long)(c - t.first[i]) * CLIP_CHUNK;
        const long long left = t.n[i] - at;
        const int n = left < CLIP_CHUNK ? (int)left : CLIP_CHUNK;
        const int dt = t.dt[i];
        if (dt == PNGPD_F32) {
            const float *g = (const float *)t.ptr[i] + at;
            if (n == CLIP_CHUNK && !((uintptr_t)g & 15)) {
                f32x4 v[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = ((const f32x4 *)g)[k * 256 + threadIdx.x];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    norm_add(KIND, a0, v[k][0]); norm_add(KIND, a1, v[k][1]);
                    norm_add(KIND, a0, v[k][2]); norm_add(KIND, a1, v[k][3]);
                }
            } else {
                for (int k = threadIdx.x; k < n; k += 256) norm_add(KIND, a0, g[k]);
            }
        } else {
            const u16 *g = (const u16 *)t.ptr[i] + at;
            if (n == CLIP_CHUNK && !((uintptr_t)g & 15)) {
                uint4 v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = ((const uint4 *)g)[k * 256 + threadIdx.x];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const unsigned w[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        norm_add(KIND, a0, half_to_f(dt, (u16)w[e])); norm_add(KIND, a1, half_to_f(dt, (u16)(w[e] >> 16)));
                    }
                }
            } else {
                for (int k = threadIdx.x; k < n; k += 256) norm_add(KIND, a0, half_to_f(dt, g[k]));
            }
        }
    }
    const double a = norm_block(KIND, norm_join(KIND, a0, a1));
    if (threadIdx.x == 0) part[blockIdx.x] = a;
}

// norm and clip factor from the partials, the same in every workgroup; the first one of the launch may store the norm.
// scale: the factor the gradients carry already (1, or the data-parallel mean's)
__device__ __forceinline__ float clip_factor(int kind, const double *__restrict__ part, int nparts, double scale,
                                             float max_norm, float *__restrict__ total) {
    double a = 0.0;
    for (int i = threadIdx.x; i < nparts; i += 256) a = norm_join(kind, a, part[i]);
    a = norm_block(kind, a);
    if (kind == KIND_L2) a = sqrt(a);
    const float norm = (float)(a * fabs(scale));
    if (total && blockIdx.x == 0 && threadIdx.x == 0) *total = norm;
    if (max_norm == INFINITY) return 1.f;           // the norm alone, an infinite one too
    const float c = (float)((double)max_norm / ((double)norm + 1e-6));
    return c > 1.f ? 1.f : c;                       // NaN stays NaN: the gradients of a diverged step must show it
}

__global__ __launch_bounds__(256) void grad_scale_kernel(const ClipTable t, int kind, const double *__restrict__ part,
                                                         int nparts, float max_norm, float *__restrict__ total) {
    const float c = clip_factor(kind, part, nparts, 1.0, max_norm, total);
    if (c == 1.f) return;
    // from the end: the norm's launch read that last, and up to 256 MB of it are still in the last-level cache
    for (int ch = t.first[t.count] - 1 - (int)blockIdx.x; ch >= 0; ch -= gridDim.x) {
        const int i = clip_find(t, ch);
        const long long at = (long long)(ch - t.first[i]) * CLIP_CHUNK;
        const long long left = t.n[i] - at;
        const int n = left < CLIP_CHUNK ? (int)left : CLIP_CHUNK;
        const int dt = t.dt[i];
        if (dt == PNGPD_F32) {
            float *g = (float *)t.ptr[i] + at;
            if (n == CLIP_CHUNK && !((uintptr_t)g & 15)) {
                f32x4 v[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = ((const f32x4 *)g)[k * 256 + threadIdx.x];
#pragma unroll
                for (int k = 0; k < 8; ++k) ((f32x4 *)g)[k * 256 + threadIdx.x] = v[k] * c;
            } else {
                for (int k = threadIdx.x; k < n; k += 256) g[k] *= c;
            }
        } else {
            u16 *g = (u16 *)t.ptr[i] + at;
            if (n == CLIP_CHUNK && !((uintptr_t)g & 15)) {
                uint4 v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = ((const uint4 *)g)[k * 256 + threadIdx.x];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    unsigned w[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        w[e] = (unsigned)f_to_half(dt, half_to_f(dt, (u16)w[e]) * c) |
                               ((unsigned)f_to_half(dt, half_to_f(dt, (u16)(w[e] >> 16)) * c) << 16);
                    ((uint4 *)g)[k * 256 + threadIdx.x] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            } else {
                for (int k = threadIdx.x; k < n; k += 256) g[k] = f_to_half(dt, half_to_f(dt, g[k]) * c);
            }
        }
    }
}

// a product that is rounded before anything else is done with it (never half of an FMA)
__device__ __forceinline__ float mul_rn(float a, float b) {
#pragma clang fp contract(off)
    return a * b;
}

// adam_flat_kernel's update with the clip factor on the gradient: the buffer is read, never rewritten, and the scaled
// gradient is rounded as it would be in the buffer.  1 - beta and the bias corrections come from fp64 (float32's
// 1 - 0.999f is 1.3e-5 off, and so is its 1 - 0.999^t).  Workgroups walk the run (at most 2048 of them: each sums the
// partials once) where adam_flat_kernel has one quad a thread.
struct AdamArgs {
    float *p, *m, *v;
    const float *g, *lr_dev, *step_dev, *gdiv_dev;
    const double *part;
    float *total;
    long long n;
    double b1, b2;
    float b2f, om1, om2;              // beta2, 1 - beta1, 1 - beta2
    float lr, bc1, bc2s;              // bc1 = 1 - beta1^t, bc2s = sqrt(1 - beta2^t) where t is known on the host
    float eps, gscale, max_norm;
    int nparts;
};
__global__ __launch_bounds__(256) void adam_flat_clip_kernel(const AdamArgs a) {
    __shared__ float bc[2];
    if (a.step_dev && threadIdx.x == 0) {
        const double t = (double)*a.step_dev;
        bc[0] = (float)(1.0 - pow(a.b1, t)); bc[1] = (float)sqrt(1.0 - pow(a.b2, t));
    }
    float gscale = a.gscale;
    if (a.gdiv_dev) gscale /= fmaxf(*a.gdiv_dev, 1.f);
    const float c = clip_factor(KIND_L2, a.part, a.nparts, gscale, a.max_norm, a.total);      // (holds a barrier)
    const float step_size = (a.lr_dev ? *a.lr_dev : a.lr) / (a.step_dev ? bc[0] : a.bc1);
    const float bc2s = a.step_dev ? bc[1] : a.bc2s;
    const long long quads = a.n >> 2;
    // from the end, as grad_scale_kernel
    for (long long q = quads - 1 - ((long long)blockIdx.x * 256 + threadIdx.x); q >= 0; q -= (long long)gridDim.x * 256) {
        f32x4 pv = ((const f32x4 *)a.p)[q], mv = ((const f32x4 *)a.m)[q], vv = ((const f32x4 *)a.v)[q];
        const f32x4 gv = ((const f32x4 *)a.g)[q];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float gg = mul_rn(mul_rn(gv[e], gscale), c);
            mv[e] = mv[e] + (gg - mv[e]) * a.om1;
            vv[e] = vv[e] * a.b2f + a.om2 * gg * gg;
            pv[e] = pv[e] - step_size * (mv[e] / (sqrtf(vv[e]) / bc2s + a.eps));
        }
        ((f32x4 *)a.p)[q] = pv; ((f32x4 *)a.m)[q] = mv; ((f32x4 *)a.v)[q] = vv;
    }
    const long long i = (quads << 2) + threadIdx.x;
    if (blockIdx.x == 0 && i < a.n) {
        const float gg = mul_rn(mul_rn(a.g[i], gscale), c);
        const float mm = a.m[i] + (gg - a.m[i]) * a.om1;
        const float vq = a.v[i] * a.b2f + a.om2 * gg * gg;
        a.m[i] = mm; a.v[i] = vq;
        a.p[i] = a.p[i] - step_size * (mm / (sqrtf(vq) / bc2s + a.eps));
    }
}

static inline long long clip_chunks(long long n) { return (n + CLIP_CHUNK - 1) / CLIP_CHUNK; }

// Calls fn(table, chunks) for the tensors in order, CLIP_TABLE non-empty ones at a time.
template <class F>
static int clip_tables(void *const *g, const long long *numel, const int *dtype, int n, F fn) {
    ClipTable t;
    t.count = 0; t.first[0] = 0;
    for (int i = 0; i <= n; ++i) {
        if (t.count == CLIP_TABLE || (i == n && t.count)) {
            const int rc = fn(t);
            if (rc != PNGPD_OK) return rc;
            t.count = 0;
        }
        if (i == n || !numel[i]) continue;
        const int k = t.count++;
        t.ptr[k] = g[i]; t.n[k] = numel[i]; t.dt[k] = (unsigned char)(dtype ? dtype[i] : PNGPD_F32);
        t.first[k + 1] = t.first[k] + (int)clip_chunks(numel[i]);
    }
    return PNGPD_OK;
}

// launches the norm; *nparts = partials written
static int clip_norm(void *const *g, const long long *numel, const int *dtype, int n, long long chunks, int kind,
                     double *part, int *nparts, hipStream_t st) {
    int at = 0;
    const int rc = clip_tables(g, numel, dtype, n, [&](const ClipTable &t) {
        const int ch = t.first[t.count];
        long long wg = (long long)ch * CLIP_PARTS / (chunks > CLIP_PARTS ? chunks : CLIP_PARTS);   // <= ch; sums to <= CLIP_PARTS
        if (wg < 1) wg = 1;
        if (kind == KIND_L2) hipLaunchKernelGGL(grad_norm_kernel<KIND_L2>, dim3((unsigned)wg), dim3(256), 0, st, t, part + at);
        else if (kind == KIND_L1) hipLaunchKernelGGL(grad_norm_kernel<KIND_L1>, dim3((unsigned)wg), dim3(256), 0, st, t, part + at);
        else hipLaunchKernelGGL(grad_norm_kernel<KIND_INF>, dim3((unsigned)wg), dim3(256), 0, st, t, part + at);
        at += (int)wg;
        return pngpd_launch_status();
    });
    *nparts = at;
    return rc;
}

// total chunks; -1 when an argument is wrong (more than 2^31 chunks included), -2 when two tensors share memory
static long long clip_check(void *const *g, const long long *numel, const int *dtype, int n) {
    if (n < 0 || (n > 0 && (!g || !numel))) return -1;
    long long chunks = 0;
    std::vector<std::pair<uintptr_t, uintptr_t>> spans;
    try { spans.reserve(n); } catch (...) { return -1; }
    for (int i = 0; i < n; ++i) {
        const int dt = dtype ? dtype[i] : PNGPD_F32;
        if (numel[i] < 0 || (numel[i] && !g[i]) || dt < PNGPD_F32 || dt > PNGPD_F16) return -1;
        if ((uintptr_t)g[i] & (dt == PNGPD_F32 ? 3 : 1)) return -1;
        chunks += clip_chunks(numel[i]);
        if (numel[i]) spans.emplace_back((uintptr_t)g[i], (uintptr_t)g[i] + (uintptr_t)numel[i] * (dt == PNGPD_F32 ? 4 : 2));
    }
    std::sort(spans.begin(), spans.end());
    for (size_t i = 1; i < spans.size(); ++i)
        if (spans[i - 1].second > spans[i].first) return -2;
    return chunks < (1ll << 31) ? chunks : -1;
}

extern "C" {

size_t pngpd_grad_clip_workspace_bytes(int n) {
    return n < 0 ? 0 : (size_t)(CLIP_PARTS + n / CLIP_TABLE + 1) * sizeof(double);
}

int pngpd_grad_clip(void *const *g, const long long *numel, const int *dtype, int n, int norm_kind, float max_norm,
                    float *total_norm, void *workspace, size_t workspace_bytes, void *stream) {
    const long long chunks = clip_check(g, numel, dtype, n);
    if (chunks == -2) return PNGPD_ERR_UNSUPPORTED;
    if (chunks < 0 || !total_norm || norm_kind < KIND_INF || norm_kind > KIND_L2 || !(max_norm >= 0.f))
        return PNGPD_ERR_INVALID_ARG;
    if (!workspace || ((uintptr_t)workspace & 7) || workspace_bytes < pngpd_grad_clip_workspace_bytes(n)) return PNGPD_ERR_WORKSPACE;
    hipStream_t st = (hipStream_t)stream;
    double *part = (double *)workspace;
    int nparts = 0;
    int rc = clip_norm(g, numel, dtype, n, chunks, norm_kind, part, &nparts, st);
    if (rc != PNGPD_OK) return rc;
    if (!chunks) {                                   // nothing to clip: the norm of no element is 0
        ClipTable t;
        t.count = 0; t.first[0] = 0;
        hipLaunchKernelGGL(grad_scale_kernel, dim3(1), dim3(256), 0, st, t, norm_kind, part, 0, max_norm, total_norm);
        return pngpd_launch_status();
    }
    return clip_tables(g, numel, dtype, n, [&](const ClipTable &t) {
        const int wg = t.first[t.count] < 2 * CLIP_PARTS ? t.first[t.count] : 2 * CLIP_PARTS;
        hipLaunchKernelGGL(grad_scale_kernel, dim3((unsigned)wg), dim3(256), 0, st, t, norm_kind, part, nparts, max_norm, total_norm);
        return pngpd_launch_status();
    });
}

int pngpd_adam_flat_clip(float *p, const float *g, float *m, float *v, const long long *offset, const long long *length,
                         int runs, float lr, const float *lr_dev, double beta1, double beta2, float eps, float step,
                         const float *step_dev, float gscale, const float *gdiv_dev, float max_norm, float *total_norm,
                         void *workspace, size_t workspace_bytes, void *stream) {
    if (!p || !g || !m || !v || runs <= 0 || !offset || !length || !total_norm || !(max_norm >= 0.f) ||
        (((uintptr_t)p | (uintptr_t)g | (uintptr_t)m | (uintptr_t)v) & 15))
        return PNGPD_ERR_INVALID_ARG;
    if (!step_dev && step < 1.f) return PNGPD_ERR_INVALID_ARG;
    if (!workspace || ((uintptr_t)workspace & 7) || workspace_bytes < pngpd_grad_clip_workspace_bytes(runs)) return PNGPD_ERR_WORKSPACE;
    hipStream_t st = (hipStream_t)stream;
    long long chunks = 0;
    for (int i = 0; i < runs; ++i) {
        if (offset[i] < 0 || length[i] <= 0 || (offset[i] & 3)) return PNGPD_ERR_INVALID_ARG;
        chunks += clip_chunks(length[i]);
    }
    if (chunks >= (1ll << 31)) return PNGPD_ERR_UNSUPPORTED;
    double *part = (double *)workspace;
    int nparts = 0;
    // the runs, CLIP_TABLE at a time (one, unless a fused piece sat the step out)
    for (int i = 0; i < runs; i += CLIP_TABLE) {
        void *ptr[CLIP_TABLE];
        const int k = runs - i < CLIP_TABLE ? runs - i : CLIP_TABLE;
        for (int j = 0; j < k; ++j) ptr[j] = (void *)(g + offset[i + j]);
        int got = 0;
        const int rc = clip_norm(ptr, length + i, nullptr, k, chunks, KIND_L2, part + nparts, &got, st);
        if (rc != PNGPD_OK) return rc;
        nparts += got;
    }
    AdamArgs a = {};
    a.lr_dev = lr_dev; a.step_dev = step_dev; a.gdiv_dev = gdiv_dev; a.part = part; a.total = total_norm;
    a.b1 = beta1; a.b2 = beta2; a.b2f = (float)beta2; a.om1 = (float)(1.0 - beta1); a.om2 = (float)(1.0 - beta2);
    a.lr = lr; a.eps = eps; a.gscale = gscale; a.max_norm = max_norm; a.nparts = nparts;
    if (!step_dev) {
        a.bc1 = (float)(1.0 - pow(beta1, (double)step));
        a.bc2s = (float)sqrt(1.0 - pow(beta2, (double)step));
    }
    for (int i = 0; i < runs; ++i) {
        const long long o = offset[i], wg = ((length[i] + 3) / 4 + 255) / 256;
        a.p = p + o; a.g = g + o; a.m = m + o; a.v = v + o; a.n = length[i];
        hipLaunchKernelGGL(adam_flat_clip_kernel, dim3((unsigned)(wg < 2048 ? wg : 2048)), dim3(256), 0, st, a);
        const int rc = pngpd_launch_status();
        if (rc != PNGPD_OK) return rc;
    }
    return PNGPD_OK;
}

}  // extern "C"
