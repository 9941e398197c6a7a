// The matrix-product core of the linear cross entropy: out[n][m] = sum_k A(m,k) B(n,k) on the matrix cores, tile by tile,
// with an epilogue that sees the accumulators (softmax statistics, the gradient of the logits, a plain store).
//
// An operand is "KC" (its k run is contiguous: row m, k along the row) or "MC" (its m run is contiguous: row k, m along the
// row), so the three products of the loss take their inputs as they lie in memory:
//     logits^T  M = V, N = T, K = D:  A = W (KC),  B = x (KC)
//     dx^T      M = D, N = T, K = V:  A = W (MC),  B = g (KC)
//     dW^T      M = D, N = V, K = T:  A = x (MC),  B = g (MC)
// The transposed products put the output's contiguous dimension on the accumulator's registers: a lane of
// v_mfma_f32_32x32x* holds one column n and 16 rows m in runs of four — softmax statistics of a row of logits reduce
// inside a lane, and stores are 8 or 16 bytes.
//
// A K tile (128 bytes of k: 64 of 16 bits, 32 of 32, four steps of the matrix instructions) of both operands goes from
// global memory straight into LDS (global_load_lds_dwordx4, no registers, the address a scalar base that walks along k
// plus a 32-bit lane offset that stays), up to PIPE - 1 tiles ahead of the matrix instructions.  A wave reads the
// fragments of a step while the products of the step before run; the one barrier of a tile stands before its last
// step, which has its fragments.  The LDS destination of that load is lane after lane, so the XOR swizzle
// against bank conflicts is put on the SOURCE: slot p of LDS row r holds chunk p ^ f(r).
//   KC: fragments are ds_read_b128 (8 or 4 consecutive k of a row);
//   MC, 16 bits: ds_read_b64_tr_b16, which transposes a [4 k][16 m] block over 16 lanes; 32 bits: ds_read_b32 per k.
// (Measured: no bank conflict in any of the three products.)
// float32 runs on v_mfma_f32_32x32x2_f32 (exact products, fp32 accumulation); chunk j of the two lane halves are k and
// k + 4 of the same 8, for A and B alike.
#pragma once
#include "pngpd_common.h"
#include "pngpd_types.h"

typedef _Float16 lce_f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 lce_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 lce_bf16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) lce_bf16x4 lds_lce_bf16x4;
typedef __attribute__((address_space(3))) char lds_char;

#define LCE_KB 128                         // bytes of k in a tile: a cache line of every row of a KC operand
#define LCE_BAND 4                         // n tiles of a band (lce_tile_of)

struct LceOperand {
    const void *p;
    long long ld;                          // elements from row to row
};

// 16 bytes per lane from each lane's own address to LDS, lane after lane, at `lds` (wave-uniform byte address).
// lce_wait_barrier() is what waits for it.
__device__ __forceinline__ void lce_load16(const void *g, unsigned lds) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)g,
                                     (__attribute__((address_space(3))) void *)(uintptr_t)lds, 16, 0, 0);
}
// all but the youngest N loads of this wave have landed, and every wave of the workgroup says so
template <int N> __device__ __forceinline__ void lce_wait_barrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(N) : "memory");
}

// all but the youngest tiles' loads have landed: of MOST tiles that may be on their way behind the one waited for, `n` are
template <int LOADS, int MOST> __device__ __forceinline__ void lce_wait_tile(int n) {
    if (MOST >= 3 && n >= 3) lce_wait_barrier<3 * LOADS>();
    else if (MOST >= 2 && n == 2) lce_wait_barrier<2 * LOADS>();
    else if (MOST >= 1 && n == 1) lce_wait_barrier<LOADS>();
    else if (n <= 0) lce_wait_barrier<0>();
    else lce_wait_barrier<MOST * LOADS>();
}
// LDS is settled between the waves; loads on their way stay so
__device__ __forceinline__ void lce_lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");
}

__device__ __align__(16) unsigned lce_zero[4];       // what a chunk past the end of k reads

// One operand's tile: ROWS values of m (or n) by LCE_KB bytes of k.
template <int DT, bool MC, int ROWS, int THREADS> struct LceTile {
    static constexpr int E = DT == PNGPD_F32 ? 4 : 2, EPC = 16 / E, BK = LCE_KB / E;
    static constexpr int BYTES = ROWS * LCE_KB, LOADS = BYTES / (THREADS * 16);
    static constexpr int RB = MC ? ROWS * E : LCE_KB, CPR = RB / 16;      // bytes, chunks of an LDS row
    static_assert(BYTES % (THREADS * 16) == 0, "a tile is whole loads of the workgroup");
    const char *base;                      // uniform: the tile's start
    unsigned off[LOADS];                   // bytes from there to the lane's chunks (below 4 GiB: the host sees to it)

    static __device__ __forceinline__ int swz(int row) {
        if constexpr (!MC) return (row >> 1) & 7;
        else if constexpr (DT == PNGPD_F32) return RB >= 256 ? ((row >> 2) & 1) << 3 : 0;
        else return RB >= 256 ? (row & 3) << 2 : RB == 128 ? ((row >> 1) & 1) << 2 : 0;
    }
    static __device__ __forceinline__ int row_of(int i) { return (i * THREADS + (int)threadIdx.x) / CPR; }
    static __device__ __forceinline__ int chunk_of(int i) { return ((i * THREADS + (int)threadIdx.x) % CPR) ^ swz(row_of(i)); }
    // m0: first m of the tile, M: how many exist; k0: first k; rows (KC): where row m of the operand lies, NULL: at m
    __device__ __forceinline__ void init(const LceOperand &o, const int *rows, int m0, int M, long long k0) {
        if constexpr (MC) base = (const char *)o.p + (k0 * o.ld + m0) * E;
        else base = (const char *)o.p + ((rows ? 0 : m0 * o.ld) + k0) * E;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int row = row_of(i), c = chunk_of(i) * EPC;
            if constexpr (MC) {
                // (a column past M: the last one there is; outputs past M are not stored)
                off[i] = (unsigned)(row * o.ld + (m0 + c < M ? c : M - EPC - m0)) * E;
            } else {
                const int m = m0 + row < M ? m0 + row : M - 1;
                off[i] = (unsigned)((rows ? rows[m] : m - m0) * o.ld + c) * E;
            }
        }
    }
    // left: k that exist from the tile's start (a whole tile where left >= BK)
    __device__ __forceinline__ void load(unsigned lds, int left, long long ld) {
        const unsigned to = __builtin_amdgcn_readfirstlane(lds + (threadIdx.x & ~63u) * 16);
        if (left >= BK) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) lce_load16(base + (unsigned long long)off[i], to + i * THREADS * 16);
        } else {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const char *g = (MC ? row_of(i) : chunk_of(i) * EPC) < left ? base + (unsigned long long)off[i] : (const char *)lce_zero;
                lce_load16(g, to + i * THREADS * 16);
            }
        }
        base += MC ? ld * BK * E : (long long)LCE_KB;
    }
    // the fragment of rows [row0, row0 + 32) at step s (16 or 8 values of k)
    static __device__ __forceinline__ f32x4 frag(const char *lds, int row0, int s, int lane) {
        if constexpr (!MC) {
            const int row = row0 + (lane & 31);
            return *(const f32x4 *)(lds + row * RB + (((2 * s + (lane >> 5)) ^ swz(row)) << 4));
        } else if constexpr (DT == PNGPD_F32) {
            f32x4 v;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int kk = 8 * s + 4 * (lane >> 5) + j, col = row0 + (lane & 31);
                v[j] = *(const float *)(lds + kk * RB + (((col >> 2) ^ swz(kk)) << 4) + (col & 3) * 4);
            }
            return v;
        } else {
            uint2 h[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int kk = 16 * s + 8 * (lane >> 5) + 4 * j + ((lane & 15) >> 2);
                const int col = row0 + (lane & 16) + 4 * (lane & 3);
                const char *at = lds + kk * RB + (((col >> 3) ^ swz(kk)) << 4) + (col & 7) * 2;
                h[j] = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_lce_bf16x4 *)at));
            }
            return f32x4{__uint_as_float(h[0].x), __uint_as_float(h[0].y), __uint_as_float(h[1].x), __uint_as_float(h[1].y)};
        }
    }
};

template <int DT> __device__ __forceinline__ f32x16 lce_mma(const f32x4 &a, const f32x4 &b, f32x16 c) {
    if constexpr (DT == PNGPD_F32) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c = mfma32(a[j], b[j], c);
        return c;
    } else if constexpr (DT == PNGPD_BF16) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(lce_bf16x8, a), __builtin_bit_cast(lce_bf16x8, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(lce_f16x8, a), __builtin_bit_cast(lce_f16x8, b), c, 0, 0, 0);
    }
}

// One workgroup's tile: BM x BN, WGM x WGN waves, PIPE tiles of k in LDS.  start() sends the first loads on their way (the
// LDS is free from the end of finish() on, so the next tile's may run under this one's epilogue), finish() does the rest.
template <int DT, bool AMC, bool BMC, int BM, int BN, int WGM, int WGN, int PIPE> struct LceCore {
    static constexpr int THREADS = WGM * WGN * 64, WM = BM / WGM, WN = BN / WGN, FM = WM / 32, FN = WN / 32;
    typedef LceTile<DT, AMC, BM, THREADS> TA;
    typedef LceTile<DT, BMC, BN, THREADS> TB;
    static constexpr int STAGE = TA::BYTES + TB::BYTES, LDS = PIPE * STAGE, BK = TA::BK, LOADS = TA::LOADS + TB::LOADS;
    static_assert(PIPE >= 2 && PIPE <= 5, "lce_wait_tile counts up to three tiles");
    static constexpr int STEPS = LCE_KB / 32;
    f32x16 acc[FM][FN];
    TA ta;
    TB tb;
    long long left;                        // k that the next tile to load has
    int tiles, stage;                      // tiles of k; where the next one goes
    unsigned lds0;

    __device__ __forceinline__ void load(long long lda, long long ldb) {
        const int l = left < BK ? (int)left : BK;
        ta.load(lds0 + stage * STAGE, l, lda);
        tb.load(lds0 + stage * STAGE + TA::BYTES, l, ldb);
        left -= BK;
        stage = stage == PIPE - 1 ? 0 : stage + 1;
    }
    // k in [k0, k1)
    __device__ __forceinline__ void start(char *smem, const LceOperand &a, const LceOperand &b, const int *rows, int m0, int M,
                                          int n0, int N, long long k0, long long k1) {
        lds0 = (unsigned)(uintptr_t)(lds_char *)smem;
        ta.init(a, nullptr, m0, M, k0);
        tb.init(b, rows, n0, N, k0);
        left = k1 - k0;
        tiles = left > 0 ? (int)((left + BK - 1) / BK) : 0;
        stage = 0;
#pragma unroll
        for (int t = 0; t < PIPE - 1; ++t) if (t < tiles) load(a.ld, b.ld);
    }
    __device__ __forceinline__ void frags(f32x4 (&fa)[FM], f32x4 (&fb)[FN], const char *sa, int wm, int wn, int s, int lane) {
        const char *sb = sa + TA::BYTES;
#pragma unroll
        for (int j = 0; j < FN; ++j) fb[j] = TB::frag(sb, wn + 32 * j, s, lane);
#pragma unroll
        for (int i = 0; i < FM; ++i) fa[i] = TA::frag(sa, wm + 32 * i, s, lane);
    }
    __device__ __forceinline__ void products(const f32x4 (&fa)[FM], const f32x4 (&fb)[FN]) {
#pragma unroll
        for (int i = 0; i < FM; ++i) {
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = lce_mma<DT>(fa[i], fb[j], acc[i][j]);
        }
    }
    __device__ __forceinline__ void finish(const char *smem, long long lda, long long ldb) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        const int wm = (wave % WGM) * WM, wn = (wave / WGM) * WN;
#pragma unroll
        for (int i = 0; i < FM; ++i) {
#pragma unroll
            for (int j = 0; j < FN; ++j) {
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
            }
        }
        if (tiles == 0) { lce_wait_barrier<0>(); return; }
        f32x4 fa[2][FM], fb[2][FN];
        lce_wait_tile<LOADS, PIPE - 2>(tiles - 1);
        frags(fa[0], fb[0], smem, wm, wn, 0, lane);
        int cur = 0;
        for (int t = 0; t < tiles; ++t) {
            const char *sa = smem + cur * STAGE;
            cur = cur == PIPE - 1 ? 0 : cur + 1;
            if (t + PIPE - 1 < tiles) load(lda, ldb);              // over tile t - 1, which every wave has read
#pragma unroll
            for (int s = 0; s + 1 < STEPS; ++s) {
                frags(fa[(s + 1) & 1], fb[(s + 1) & 1], sa, wm, wn, s + 1, lane);
                products(fa[s & 1], fb[s & 1]);
                __builtin_amdgcn_sched_barrier(0);
            }
            lce_wait_tile<LOADS, PIPE - 2>(tiles - 2 - t);         // tile t + 1 is there, tile t is read
            if (t + 1 < tiles) frags(fa[0], fb[0], smem + cur * STAGE, wm, wn, 0, lane);
            products(fa[1], fb[1]);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
};

// Workgroup -> tile.  Workgroup i runs on XCD i % 8: each XCD takes a contiguous stretch of a walk over the tiles that
// goes down bands of LCE_BAND n tiles, so the operands of its running workgroups overlap in its own L2.  (i < mt * nt)
__device__ __forceinline__ void lce_tile_of(int i, int mt, int nt, int &m, int &n) {
    const int per = (mt * nt) >> 3;
    int w = i;
    if (i < per * 8) w = (i & 7) * per + (i >> 3);
    const int band = w / (LCE_BAND * mt), r = w - band * LCE_BAND * mt;
    const int wide = nt - band * LCE_BAND < LCE_BAND ? nt - band * LCE_BAND : LCE_BAND;
    m = r / wide; n = band * LCE_BAND + r % wide;
}
