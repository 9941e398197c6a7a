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
// A K tile (64 bytes of k: 32 of 16 bits, 16 of 32) of both operands goes from global memory straight into LDS
// (global_load_lds_dwordx4, no registers), one tile ahead of the matrix instructions, one barrier a tile; two workgroups
// share a CU, so one's barrier and epilogue hide behind the other's products.  The LDS destination of that load is lane
// after lane, so the XOR swizzle against bank conflicts is put on the SOURCE: slot p of LDS row r holds chunk p ^ f(r).
//   KC: fragments are ds_read_b128 (8 or 4 consecutive k of a row);
//   MC, 16 bits: ds_read_b64_tr_b16, which transposes a [4 k][16 m] block over 16 lanes; 32 bits: ds_read_b32 per k.
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

#define LCE_KB 64                          // bytes of k in a tile
#define LCE_PIPE 2                         // tiles in LDS

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

__device__ __align__(16) unsigned lce_zero[4];       // what a chunk past the end of k reads

// One operand's tile: ROWS values of m (or n) by LCE_KB bytes of k.
template <int DT, bool MC, int ROWS, int THREADS> struct LceTile {
    static constexpr int E = DT == PNGPD_F32 ? 4 : 2, EPC = 16 / E, BK = LCE_KB / E;
    static constexpr int BYTES = ROWS * LCE_KB, LOADS = BYTES / (THREADS * 16);
    static constexpr int RB = MC ? ROWS * E : LCE_KB, CPR = RB / 16;      // bytes, chunks of an LDS row
    static_assert(BYTES % (THREADS * 16) == 0, "a tile is whole loads of the workgroup");
    const char *p[LOADS];
    int k[LOADS];                          // k of the chunk (KC) or of the row (MC), from the tile's start

    static __device__ __forceinline__ int swz(int row) {
        if constexpr (!MC) return (row >> 2) & 3;
        else if constexpr (DT == PNGPD_F32) return RB >= 256 ? ((row >> 2) & 1) << 3 : 0;
        else return RB >= 256 ? (row & 3) << 2 : RB == 128 ? ((row >> 1) & 1) << 2 : 0;
    }
    // m0: first m of the tile, M: how many exist; k0: first k
    __device__ __forceinline__ void init(const LceOperand &o, int m0, int M, long long k0) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int q = i * THREADS + (int)threadIdx.x, row = q / CPR, c = (q % CPR) ^ swz(row);
            if constexpr (MC) {
                int m = m0 + c * EPC;
                if (m >= M) m = M - EPC;                       // outputs past M are not stored
                k[i] = row;
                p[i] = (const char *)o.p + ((k0 + row) * o.ld + m) * E;
            } else {
                const int m = m0 + row < M ? m0 + row : M - 1;
                k[i] = c * EPC;
                p[i] = (const char *)o.p + ((long long)m * o.ld + k0 + k[i]) * E;
            }
        }
    }
    // left: k that exist from the tile's start (a whole tile where left >= BK)
    __device__ __forceinline__ void load(unsigned lds, int left, long long ld) {
        const unsigned base = lds + (threadIdx.x & ~63u) * 16;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const char *g = p[i];
            if (left < BK) g = k[i] < left ? g : (const char *)lce_zero;
            lce_load16(g, __builtin_amdgcn_readfirstlane(base + i * THREADS * 16));
            p[i] += MC ? ld * BK * E : (long long)LCE_KB;
        }
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

// The accumulators of one workgroup's tile: BM x BN, WGM x WGN waves.  k in [k0, k1).
template <int DT, bool AMC, bool BMC, int BM, int BN, int WGM, int WGN> struct LceCore {
    static constexpr int THREADS = WGM * WGN * 64, WM = BM / WGM, WN = BN / WGN, FM = WM / 32, FN = WN / 32;
    typedef LceTile<DT, AMC, BM, THREADS> TA;
    typedef LceTile<DT, BMC, BN, THREADS> TB;
    static constexpr int STAGE = TA::BYTES + TB::BYTES, LDS = LCE_PIPE * STAGE, BK = TA::BK;
    f32x16 acc[FM][FN];

    __device__ __forceinline__ void run(char *smem, const LceOperand &a, const LceOperand &b, int m0, int M, int n0, int N,
                                        long long k0, long long k1) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        const int wm = (wave % WGM) * WM, wn = (wave / WGM) * WN;
        const unsigned lds0 = (unsigned)(uintptr_t)(lds_char *)smem;
#pragma unroll
        for (int i = 0; i < FM; ++i) {
#pragma unroll
            for (int j = 0; j < FN; ++j) {
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
            }
        }
        TA ta;
        TB tb;
        ta.init(a, m0, M, k0);
        tb.init(b, n0, N, k0);
        const long long K = k1 - k0;
        const int tiles = (int)((K + BK - 1) / BK);
        ta.load(lds0, K < BK ? (int)K : BK, a.ld);
        tb.load(lds0 + TA::BYTES, K < BK ? (int)K : BK, b.ld);
        for (int t = 0; t < tiles; ++t) {
            lce_wait_barrier<0>();
            const int cur = t % LCE_PIPE, nxt = (t + 1) % LCE_PIPE;
            if (t + 1 < tiles) {
                const long long left = K - (long long)(t + 1) * BK;
                const int l = left < BK ? (int)left : BK;
                ta.load(lds0 + nxt * STAGE, l, a.ld);
                tb.load(lds0 + nxt * STAGE + TA::BYTES, l, b.ld);
            }
            const char *sa = smem + cur * STAGE, *sb = sa + TA::BYTES;
#pragma unroll
            for (int s = 0; s < LCE_KB / 32; ++s) {
                f32x4 fa[FM], fb[FN];
#pragma unroll
                for (int j = 0; j < FN; ++j) fb[j] = TB::frag(sb, wn + 32 * j, s, lane);
#pragma unroll
                for (int i = 0; i < FM; ++i) fa[i] = TA::frag(sa, wm + 32 * i, s, lane);
#pragma unroll
                for (int i = 0; i < FM; ++i) {
#pragma unroll
                    for (int j = 0; j < FN; ++j) acc[i][j] = lce_mma<DT>(fa[i], fb[j], acc[i][j]);
                }
            }
        }
        lce_wait_barrier<0>();                                     // the epilogue may use the LDS
    }
};

// Workgroup -> tile.  Workgroup i runs on XCD i % 8: each XCD takes a contiguous stretch of a walk over the tiles that
// goes down bands of 8 n tiles, so the operands of its running workgroups overlap in its own L2.
__device__ __forceinline__ void lce_tile_of(int i, int total, int mt, int nt, int &m, int &n) {
    const int per = total >> 3;
    int w = i;
    if (i < per * 8) w = (i & 7) * per + (i >> 3);
    const int band = w / (8 * mt), r = w - band * 8 * mt;
    const int wide = nt - band * 8 < 8 ? nt - band * 8 : 8;
    m = r / wide; n = band * 8 + r % wide;
}
