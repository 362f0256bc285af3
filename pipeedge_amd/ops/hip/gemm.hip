// bf16 MFMA GEMM with fused epilogue (bias + activation + residual add).
//
// Computes C[M,N] = act(A[M,K] @ B^T + bias) [+ residual] with B stored
// [N,K] - the framework's native weight layout. [N,K] makes BOTH operands
// k-contiguous per row, so A- and B-tiles stage identically.
//
// Two paths (cdna_hip_programming.md section 5):
// - glds path (K % 64 == 0, the transformer shapes): 64x64x64 tiles staged
//   with 16-B `global_load_lds` directly into double-buffered LDS
//   (no VGPR round trip - Common-mistake #1), XOR-swizzled via the SOURCE
//   address (rule 21) so ds_read_b128 fragment reads are low-conflict (T2),
//   2-phase pipeline: next tile's glds issued before the current tile's
//   MFMAs (T3 minimum recipe);
// - generic path (any K): plain vectorized staging into padded LDS.
//
// Replaces what the reference ran through HF Linear modules on CPU
// (reference vit.py:45-53).
#include <torch/extension.h>

#include <cstdlib>

#include "common.h"

namespace {

constexpr int BM = 64;
constexpr int BN = 64;
constexpr int BK = 64;
constexpr int PAD = 8;

__device__ __forceinline__ void glds_b128(const void* gsrc, void* lds_dst) {
    __builtin_amdgcn_global_load_lds(
        (const __attribute__((address_space(1))) unsigned int*)gsrc,
        (__attribute__((address_space(3))) unsigned int*)lds_dst, 16, 0, 0);
}

// read a bf16x8 fragment from a lane-linear [rows][KB] tile with a byte
// XOR swizzle matching the staging source permutation. The XOR spans the
// row's 16-B columns: 8 columns at KB=64 (<=2-way residual conflict), 16 at
// KB=128 (conflict-free - rows of a fragment group are distinct mod 16).
template <int KB>
constexpr int swz_mask() { return (KB / 8 < 16 ? KB / 8 : 16) - 1; }

template <int KB>  // K extent of the tile in elements
__device__ __forceinline__ bf16x8 lds_read_swz(const __bf16* tile, int row,
                                               int kelem) {
    const int byte = (row * (KB * 2) + kelem * 2) ^
                     ((row & swz_mask<KB>()) << 4);
    return *reinterpret_cast<const bf16x8*>(
        reinterpret_cast<const char*>(tile) + byte);
}

// bijective XCD-aware block remap (guide T1): contiguous grid chunks per XCD
__device__ __forceinline__ int xcd_swizzle(int bid, int nblocks) {
    const int nxcd = 8;
    const int q = nblocks / nxcd, r = nblocks % nxcd;
    const int xcd = bid % nxcd, i = bid / nxcd;
    return (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + i;
}

struct EpilogueArgs {
    const __bf16* bias;
    const __bf16* residual;
    __bf16* C;
    int M, N, act;
    // folded-LN input adjustment (see ops/__init__.py ln_linear): the GEMM
    // ran on RAW x against W' = W*ln_w; the epilogue applies
    //   out = r*acc - r*mu*ln_s[col] + ln_c[col]
    // with per-row mu/r from the SUMMED partial stats
    // ln_stats[p][row][2] (p < ln_parts), each partial written without
    // atomics by one (column-block, column-wave) of the producing GEMM.
    const float* ln_stats;   // [M][ln_parts][2] or nullptr
    int ln_parts;
    const float* ln_s;       // [N] row-sums of W'
    const float* ln_c;       // [N] ln_b @ W^T
    float ln_eps;
    int ln_k;                // LN normalization length (= GEMM K)
    float ln_rk;             // 1.0f / ln_k (full f32 div is ~10 instrs)
    // output-stats emission: this block's (col-block by, col-wave) slice of
    // stats_out[parts][M][2]; plain stores, no zeroing needed
    float* stats_out;        // or nullptr
    int stats_parts;
};

// cooperative per-block LN-coefficient pass: thread t < TBM sums row
// (bm + t)'s partials and writes (mu, rstd) into the (reused) LDS tile -
// one thread per row, loads pipeline in parallel, no cross-lane shuffles,
// no divisions in the per-element epilogue loops.
template <int TBM>
__device__ __forceinline__ void ln_coeffs_to_lds(
        const EpilogueArgs& ep, int bm, int tid, float* lnbuf) {
    __syncthreads();  // k-loop reads of the LDS tile are done
    if (tid < TBM) {
        const int row = bm + tid;
        float mu = 0.0f, rstd = 1.0f;
        if (row < ep.M) {
            const float* rp = ep.ln_stats + (long)row * ep.ln_parts * 2;
            float s1 = 0.0f, s2 = 0.0f;
            for (int p = 0; p < ep.ln_parts; ++p) {
                s1 += rp[p * 2];
                s2 += rp[p * 2 + 1];
            }
            mu = s1 * ep.ln_rk;
            rstd = rsqrtf(s2 * ep.ln_rk - mu * mu + ep.ln_eps);
        }
        lnbuf[tid * 2] = mu;
        lnbuf[tid * 2 + 1] = rstd;
    }
    __syncthreads();
}

template <int MI, int NI, int EPM>  // EPM: 0 plain, 1 ln-in, 2 stats-out
__device__ __forceinline__ void gemm_epilogue(
        const f32x4 (&acc)[MI][NI], const EpilogueArgs& ep, int bm, int bn,
        int wm, int wn, int lane, int part_idx, const float* lnbuf) {
    // per-row LN coefficients from the block's LDS buffer (broadcast reads)
    float mu[MI][4], rstd[MI][4];
    if constexpr (EPM == 1) {
        #pragma unroll
        for (int mi = 0; mi < MI; ++mi) {
            #pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int lrow = wm + mi * 16 + (lane >> 4) * 4 + r;
                mu[mi][r] = lnbuf[lrow * 2];
                rstd[mi][r] = lnbuf[lrow * 2 + 1];
            }
        }
    }
    float row_sum[EPM == 2 ? MI : 1][4] = {};
    float row_sumsq[EPM == 2 ? MI : 1][4] = {};
    #pragma unroll
    for (int mi = 0; mi < MI; ++mi) {
        #pragma unroll
        for (int ni = 0; ni < NI; ++ni) {
            const int col = bn + wn + ni * 16 + (lane & 15);
            if (col >= ep.N) continue;
            const float bv = ep.bias != nullptr ? bf2f(ep.bias[col]) : 0.0f;
            const float sv = EPM == 1 ? ep.ln_s[col] : 0.0f;
            const float cv = EPM == 1 ? ep.ln_c[col] : 0.0f;
            #pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = bm + wm + mi * 16 + (lane >> 4) * 4 + r;
                if (row >= ep.M) continue;
                float v = acc[mi][ni][r];
                if constexpr (EPM == 1)
                    v = rstd[mi][r] * v - rstd[mi][r] * mu[mi][r] * sv + cv;
                v += bv;
                if (ep.act == ACT_GELU) v = gelu_f(v);
                else if (ep.act == ACT_TANH) v = tanhf(v);
                if (ep.residual != nullptr)
                    v += bf2f(ep.residual[(long)row * ep.N + col]);
                ep.C[(long)row * ep.N + col] = f2bf(v);
                if constexpr (EPM == 2) {
                    row_sum[mi][r] += v;
                    row_sumsq[mi][r] += v * v;
                }
            }
        }
    }
    if constexpr (EPM == 2) {
        // reduce across the 16 lanes sharing each C-fragment row; ONE plain
        // store per (row, this block's column-wave slice); layout [M][P][2]
        #pragma unroll
        for (int mi = 0; mi < MI; ++mi) {
            #pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float s1 = group16_reduce(row_sum[mi][r], SumOp());
                const float s2 = group16_reduce(row_sumsq[mi][r], SumOp());
                const int row = bm + wm + mi * 16 + (lane >> 4) * 4 + r;
                if ((lane & 15) == 0 && row < ep.M) {
                    float* slot = ep.stats_out +
                        ((long)row * ep.stats_parts + part_idx) * 2;
                    slot[0] = s1;
                    slot[1] = s2;
                }
            }
        }
    }
}

// ---------------------------------------------------------------------------
// glds path: K % 64 == 0. Tile = (32*MI) x (32*NI) with 4 waves in 2x2,
// each wave an MIxNI grid of 16x16 fragments. <2,2> = 64x64 (small-N
// shapes need the block count), <4,4> = 128x128 (fc1/qkv class).
// ---------------------------------------------------------------------------
template <int MI, int NI, int KT = 1, bool XCD = false, int EPM = 0>
__global__ __launch_bounds__(256) void gemm_bf16_glds_kernel(
        const __bf16* __restrict__ A, const __bf16* __restrict__ B,
        __bf16* __restrict__ C, int M, int N, int K, EpilogueArgs ep) {
    constexpr int TBM = 32 * MI;
    constexpr int TBN = 32 * NI;
    constexpr int KB = BK * KT;          // K extent per staged tile
    // ONE shared object (guide section 5 trap 4a): [buf][TBM+TBN rows][KB]
    __shared__ __bf16 smem[2][TBM + TBN][KB];

    int bx = blockIdx.x, by = blockIdx.y;
    if (XCD) {
        const int nb = gridDim.x * gridDim.y;
        const int id = xcd_swizzle(by * gridDim.x + bx, nb);
        bx = id % gridDim.x;
        by = id / gridDim.x;
    }
    const int bm = bx * TBM;
    const int bn = by * TBN;
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wid = tid >> 6;
    const int wm = (wid >> 1) * (16 * MI);
    const int wn = (wid & 1) * (16 * NI);

    // staging: 1-KiB glds pieces of R=8/KT rows x (8*KT) 16-B columns each;
    // source column XOR-swizzled to match the read-side (row&7)<<4 swizzle
    constexpr int RPP = 8 / KT;              // rows per piece
    const int srow = lane / (8 * KT);        // row within piece
    const int cdst = lane % (8 * KT);

    // the XOR swizzle keys off the GLOBAL tile row mod 8, which spans
    // multiple pieces when RPP < 8. Running per-piece pointers (stage k0
    // is monotone +KB) keep address math out of the k-loop.
    const __bf16* a_pc[TBM / (32 / KT)];
    const __bf16* b_pc[TBN / (32 / KT)];
    #pragma unroll
    for (int i = 0; i < TBM / (32 / KT); ++i) {
        const int p = wid * (TBM / (32 / KT)) + i;
        const int trow = p * RPP + srow;
        const int csrc = cdst ^ (trow & swz_mask<KB>());
        a_pc[i] = A + (long)min(bm + trow, M - 1) * K + csrc * 8;
    }
    #pragma unroll
    for (int i = 0; i < TBN / (32 / KT); ++i) {
        const int p = wid * (TBN / (32 / KT)) + i;
        const int trow = p * RPP + srow;
        const int csrc = cdst ^ (trow & swz_mask<KB>());
        b_pc[i] = B + (long)min(bn + trow, N - 1) * K + csrc * 8;
    }
    auto stage = [&](int buf) {
        #pragma unroll
        for (int i = 0; i < TBM / (32 / KT); ++i) {
            const int p = wid * (TBM / (32 / KT)) + i;
            glds_b128(a_pc[i], &smem[buf][p * RPP][0]);
            a_pc[i] += KB;
        }
        #pragma unroll
        for (int i = 0; i < TBN / (32 / KT); ++i) {
            const int p = wid * (TBN / (32 / KT)) + i;
            glds_b128(b_pc[i], &smem[buf][TBM + p * RPP][0]);
            b_pc[i] += KB;
        }
    };

    f32x4 acc[MI][NI] = {};
    stage(0);
    __syncthreads();  // barrier waits vmcnt(0) while glds in flight

    const int n_tiles = K / KB;
    for (int t = 0; t < n_tiles; ++t) {
        const int buf = t & 1;
        if (t + 1 < n_tiles) stage(buf ^ 1);
        #pragma unroll
        for (int kk = 0; kk < KB; kk += 32) {
            const int kgrp = kk + (lane >> 4) * 8;
            bf16x8 af[MI], bfr[NI];
            #pragma unroll
            for (int mi = 0; mi < MI; ++mi)
                af[mi] = lds_read_swz<KB>(&smem[buf][0][0],
                                          wm + mi * 16 + (lane & 15), kgrp);
            #pragma unroll
            for (int ni = 0; ni < NI; ++ni)
                bfr[ni] = lds_read_swz<KB>(&smem[buf][TBM][0],
                                           wn + ni * 16 + (lane & 15), kgrp);
            #pragma unroll
            for (int mi = 0; mi < MI; ++mi)
                #pragma unroll
                for (int ni = 0; ni < NI; ++ni)
                    acc[mi][ni] = mfma_16x16x32_bf16(af[mi], bfr[ni],
                                                     acc[mi][ni]);
        }
        __syncthreads();
    }

    float* lnbuf = reinterpret_cast<float*>(&smem[0][0][0]);
    if constexpr (EPM == 1)
        ln_coeffs_to_lds<TBM>(ep, bm, tid, lnbuf);
    gemm_epilogue<MI, NI, EPM>(acc, ep, bm, bn, wm, wn, lane,
                               (bn / TBN) * 2 + (wid & 1), lnbuf);
}

// ---------------------------------------------------------------------------
// NBUF-buffer glds pipeline (K % 64 == 0): NBUF-2 K-tiles of loads stay in
// flight ACROSS barriers (guide "Pipelining across barriers"): raw
// s_barrier + counted `s_waitcnt vmcnt(N)` instead of __syncthreads(),
// whose fence would drain the in-flight LDS-DMA to vmcnt(0) every tile.
// NBUF=3: 48 KiB LDS -> 3 blocks/CU (the default t7). NBUF=4 (t10): one
// more tile in flight at 64 KiB -> 2 blocks/CU - a depth-vs-occupancy
// trade for the latency-bound regime the final PMC shows
// (profiles/hot_pmc_final.csv: MemUnitStalled ~0.1, zero LDS conflicts).
// ---------------------------------------------------------------------------
template <int MI, int NI, bool XCD = false, int EPM = 0, int NBUF = 3>
__global__ __launch_bounds__(256) void gemm_bf16_glds3_kernel(
        const __bf16* __restrict__ A, const __bf16* __restrict__ B,
        __bf16* __restrict__ C, int M, int N, int K, EpilogueArgs ep) {
    constexpr int TBM = 32 * MI;
    constexpr int TBN = 32 * NI;
    constexpr int KB = BK;
    __shared__ __bf16 smem[NBUF][TBM + TBN][KB];

    int bx = blockIdx.x, by = blockIdx.y;
    if (XCD) {
        const int nb = gridDim.x * gridDim.y;
        const int id = xcd_swizzle(by * gridDim.x + bx, nb);
        bx = id % gridDim.x;
        by = id / gridDim.x;
    }
    const int bm = bx * TBM;
    const int bn = by * TBN;
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wid = tid >> 6;
    const int wm = (wid >> 1) * (16 * MI);
    const int wn = (wid & 1) * (16 * NI);

    const int srow = lane >> 3;
    const int cdst = lane & 7;

    // glds per wave per tile: TBM/32 + TBN/32. Per-piece RUNNING global
    // pointers advanced by KB per stage call (stage k0 is monotone +KB):
    // the round-1 per-call arow*K + k0 recompute left only 8 of 60 k-loop
    // instructions as MFMA (22 SALU + 16 VALU of address math).
    constexpr int GLDS_PER_TILE = TBM / 32 + TBN / 32;
    const __bf16* a_pc[TBM / 32];
    const __bf16* b_pc[TBN / 32];
    #pragma unroll
    for (int i = 0; i < TBM / 32; ++i) {
        const int p = wid * (TBM / 32) + i;
        const int trow = p * 8 + srow;
        const int csrc = cdst ^ (trow & 7);
        a_pc[i] = A + (long)min(bm + trow, M - 1) * K + csrc * 8;
    }
    #pragma unroll
    for (int i = 0; i < TBN / 32; ++i) {
        const int p = wid * (TBN / 32) + i;
        const int trow = p * 8 + srow;
        const int csrc = cdst ^ (trow & 7);
        b_pc[i] = B + (long)min(bn + trow, N - 1) * K + csrc * 8;
    }
    auto stage = [&](int buf) {
        #pragma unroll
        for (int i = 0; i < TBM / 32; ++i) {
            const int p = wid * (TBM / 32) + i;
            glds_b128(a_pc[i], &smem[buf][p * 8][0]);
            a_pc[i] += KB;
        }
        #pragma unroll
        for (int i = 0; i < TBN / 32; ++i) {
            const int p = wid * (TBN / 32) + i;
            glds_b128(b_pc[i], &smem[buf][TBM + p * 8][0]);
            b_pc[i] += KB;
        }
    };

    f32x4 acc[MI][NI] = {};
    const int n_tiles = K / KB;
    #pragma unroll
    for (int p = 0; p < NBUF - 1; ++p)
        if (p < n_tiles) stage(p);

    // single loop (a main/tail split measured WORSE: the compiler cloned
    // the k-body and shuffled the accumulators through 12-32 accvgpr
    // copies per iteration); rotating buffer indices avoid the %NBUF
    for (int t = 0, cbuf = 0, sbuf = NBUF - 1; t < n_tiles; ++t) {
        // tile t's LDS-DMA retired for THIS wave; up to NBUF-2 more tiles
        // stay in flight across the barrier
        const int inflight = min(NBUF - 2, n_tiles - 1 - t);
        switch (inflight) {
        case 0:
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            break;
        case 1:
            asm volatile("s_waitcnt vmcnt(%0)" ::"i"(GLDS_PER_TILE)
                         : "memory");
            break;
        default:
            asm volatile("s_waitcnt vmcnt(%0)" ::"i"(2 * GLDS_PER_TILE)
                         : "memory");
            break;
        }
        __builtin_amdgcn_s_barrier();
        if (t + NBUF - 1 < n_tiles) {
            stage(sbuf);
            sbuf = sbuf + 1 == NBUF ? 0 : sbuf + 1;
        }
        const int buf = cbuf;
        cbuf = cbuf + 1 == NBUF ? 0 : cbuf + 1;
        #pragma unroll
        for (int kk = 0; kk < KB; kk += 32) {
            const int kgrp = kk + (lane >> 4) * 8;
            bf16x8 af[MI], bfr[NI];
            #pragma unroll
            for (int mi = 0; mi < MI; ++mi)
                af[mi] = lds_read_swz<KB>(&smem[buf][0][0],
                                          wm + mi * 16 + (lane & 15), kgrp);
            #pragma unroll
            for (int ni = 0; ni < NI; ++ni)
                bfr[ni] = lds_read_swz<KB>(&smem[buf][TBM][0],
                                           wn + ni * 16 + (lane & 15), kgrp);
            #pragma unroll
            for (int mi = 0; mi < MI; ++mi)
                #pragma unroll
                for (int ni = 0; ni < NI; ++ni)
                    acc[mi][ni] = mfma_16x16x32_bf16(af[mi], bfr[ni],
                                                     acc[mi][ni]);
        }
        // no trailing barrier: the next iteration's entry barrier orders
        // every wave's reads of buf before anyone overwrites it
    }
    __builtin_amdgcn_s_barrier();

    float* lnbuf = reinterpret_cast<float*>(&smem[0][0][0]);
    if constexpr (EPM == 1)
        ln_coeffs_to_lds<TBM>(ep, bm, tid, lnbuf);
    gemm_epilogue<MI, NI, EPM>(acc, ep, bm, bn, wm, wn, lane,
                               (bn / TBN) * 2 + (wid & 1), lnbuf);
}

// ---------------------------------------------------------------------------
// Split-K 3-buffer glds kernel with IN-LAUNCH combine (guide section 5
// "sampling-regime projection GEMM" recipe): the fc2/out-proj-class grids
// (M~1576, N<=1024) make only ~300 64x64 blocks - barely 1 per CU, so waves
// sit parked with no partner to hide stalls (profiles/sqwait_r02.txt:
// parked 44-65%). gridDim.z = SPLITK slices per output tile; each slice
// writes an f32 slab in REGISTER layout ([tid][16] - coalesced dwordx4 both
// ways), publishes with the plain-store + agent-release + ticket recipe,
// and the LAST arriver combines all slices + runs the epilogue. No
// spinning: non-last slices exit after the ticket, so any dispatch order /
// occupancy is deadlock-free.
// ---------------------------------------------------------------------------
template <int MI, int NI, int NBUF = 3>
__global__ __launch_bounds__(256) void gemm_bf16_splitk_kernel(
        const __bf16* __restrict__ A, const __bf16* __restrict__ B,
        __bf16* __restrict__ C, int M, int N, int K,
        float* __restrict__ slabs, unsigned int* __restrict__ tickets,
        EpilogueArgs ep) {
    constexpr int TBM = 32 * MI;
    constexpr int TBN = 32 * NI;
    constexpr int KB = BK;
    __shared__ __bf16 smem[NBUF][TBM + TBN][KB];

    const int SK = gridDim.z;
    const int slice = blockIdx.z;
    int bx = blockIdx.x, by = blockIdx.y;
    {
        const int nb = gridDim.x * gridDim.y;
        const int id = xcd_swizzle(by * gridDim.x + bx, nb);
        bx = id % gridDim.x;
        by = id / gridDim.x;
    }
    const int tile_id = by * gridDim.x + bx;
    const int bm = bx * TBM;
    const int bn = by * TBN;
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wid = tid >> 6;
    const int wm = (wid >> 1) * (16 * MI);
    const int wn = (wid & 1) * (16 * NI);

    // this slice's K range: contiguous KB-multiples
    const int tiles_total = K / KB;
    const int per = (tiles_total + SK - 1) / SK;
    const int t0 = slice * per;
    const int t1 = min(tiles_total, t0 + per);
    const int n_tiles = t1 - t0;

    const int srow = lane >> 3;
    const int cdst = lane & 7;
    constexpr int GLDS_PER_TILE = TBM / 32 + TBN / 32;
    const __bf16* a_pc[TBM / 32];
    const __bf16* b_pc[TBN / 32];
    #pragma unroll
    for (int i = 0; i < TBM / 32; ++i) {
        const int p = wid * (TBM / 32) + i;
        const int trow = p * 8 + srow;
        const int csrc = cdst ^ (trow & 7);
        a_pc[i] = A + (long)min(bm + trow, M - 1) * K + t0 * KB + csrc * 8;
    }
    #pragma unroll
    for (int i = 0; i < TBN / 32; ++i) {
        const int p = wid * (TBN / 32) + i;
        const int trow = p * 8 + srow;
        const int csrc = cdst ^ (trow & 7);
        b_pc[i] = B + (long)min(bn + trow, N - 1) * K + t0 * KB + csrc * 8;
    }
    auto stage = [&](int buf) {
        #pragma unroll
        for (int i = 0; i < TBM / 32; ++i) {
            glds_b128(a_pc[i], &smem[buf][(wid * (TBM / 32) + i) * 8][0]);
            a_pc[i] += KB;
        }
        #pragma unroll
        for (int i = 0; i < TBN / 32; ++i) {
            glds_b128(b_pc[i],
                      &smem[buf][TBM + (wid * (TBN / 32) + i) * 8][0]);
            b_pc[i] += KB;
        }
    };

    f32x4 acc[MI][NI] = {};
    #pragma unroll
    for (int p = 0; p < NBUF - 1; ++p)
        if (p < n_tiles) stage(p);
    for (int t = 0; t < n_tiles; ++t) {
        const int inflight = min(NBUF - 2, n_tiles - 1 - t);
        switch (inflight) {
        case 0:
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            break;
        case 1:
            asm volatile("s_waitcnt vmcnt(%0)" ::"i"(GLDS_PER_TILE)
                         : "memory");
            break;
        default:
            asm volatile("s_waitcnt vmcnt(%0)" ::"i"(2 * GLDS_PER_TILE)
                         : "memory");
            break;
        }
        __builtin_amdgcn_s_barrier();
        if (t + NBUF - 1 < n_tiles)
            stage((t + NBUF - 1) % NBUF);
        const int buf = t % NBUF;
        #pragma unroll
        for (int kk = 0; kk < KB; kk += 32) {
            const int kgrp = kk + (lane >> 4) * 8;
            bf16x8 af[MI], bfr[NI];
            #pragma unroll
            for (int mi = 0; mi < MI; ++mi)
                af[mi] = lds_read_swz<KB>(&smem[buf][0][0],
                                          wm + mi * 16 + (lane & 15), kgrp);
            #pragma unroll
            for (int ni = 0; ni < NI; ++ni)
                bfr[ni] = lds_read_swz<KB>(&smem[buf][TBM][0],
                                           wn + ni * 16 + (lane & 15), kgrp);
            #pragma unroll
            for (int mi = 0; mi < MI; ++mi)
                #pragma unroll
                for (int ni = 0; ni < NI; ++ni)
                    acc[mi][ni] = mfma_16x16x32_bf16(af[mi], bfr[ni],
                                                     acc[mi][ni]);
        }
    }
    __builtin_amdgcn_s_barrier();

    // ---- publish this slice's partial (register layout: [tid][16]) ----
    constexpr int ELEMS = MI * NI * 4;       // f32 per thread
    float* slab = slabs + ((long)tile_id * SK + slice) * (256 * ELEMS)
                + tid * ELEMS;
    #pragma unroll
    for (int mi = 0; mi < MI; ++mi)
        #pragma unroll
        for (int ni = 0; ni < NI; ++ni)
            *reinterpret_cast<f32x4*>(slab + (mi * NI + ni) * 4) =
                acc[mi][ni];
    // plain stores -> every wave drains its own -> block sync -> lane-0
    // agent release + restated vmcnt wait (ROCm 7.2 drops the post-wbl2
    // wait when the scoreboard is provably empty - guide G16 pitfall 12)
    // -> ticket. Order is fence THEN fetch_add, never the reverse.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    // "I am last" broadcast through the ONE shared array (guide trap 4a: a
    // second __shared__ object de-pipelines the glds k-loop)
    int* last_flag = reinterpret_cast<int*>(&smem[0][0][0]);
    if (tid == 0) {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "agent");
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        const unsigned prev = __hip_atomic_fetch_add(
            &tickets[tile_id], 1u, __ATOMIC_RELAXED,
            __HIP_MEMORY_SCOPE_AGENT);
        *last_flag = (prev == (unsigned)(SK - 1));
    }
    __syncthreads();
    if (!*last_flag) return;

    // ---- last arriver: combine all slices + epilogue ----
    if (tid == 0)
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    __syncthreads();
    const float* base = slabs + (long)tile_id * SK * (256 * ELEMS)
                      + tid * ELEMS;
    #pragma unroll
    for (int mi = 0; mi < MI; ++mi)
        #pragma unroll
        for (int ni = 0; ni < NI; ++ni)
            acc[mi][ni] = f32x4{};
    for (int s = 0; s < SK; ++s) {
        const float* sp = base + (long)s * (256 * ELEMS);
        #pragma unroll
        for (int mi = 0; mi < MI; ++mi)
            #pragma unroll
            for (int ni = 0; ni < NI; ++ni)
                acc[mi][ni] += *reinterpret_cast<const f32x4*>(
                    sp + (mi * NI + ni) * 4);
    }
    gemm_epilogue<MI, NI, 0>(acc, ep, bm, bn, wm, wn, lane, 0, nullptr);
}

// ---------------------------------------------------------------------------
// 8-wave big-tile pipeline (512 threads, wave grid 2(M) x 4(N)): the
// large-shape kernel (ViT-H fc1 / 4k^3 class) where the 256-thread 64x64
// tiles are ~3x off the library (profiles/blaslt_probe.txt). Structure per
// the guide's measured tiers (cdna_hip_programming.md section 5): BK=64
// glds staging, raw s_barrier + counted vmcnt (NBUF=3: one tile of LDS-DMA
// in flight across each barrier), XOR source swizzle; 512 threads put TWO
// waves on every SIMD so MFMA issue and LDS/DMA segments of partner waves
// overlap (MI355X_MICROARCH "Two waves per SIMD").
//   <4,4,3>: 128x256 tile, 144 KiB LDS, 1 block/CU
//   <8,4,2>: 256x256 tile, 128 KiB LDS, 1 block/CU (classic 2-buffer)
// ---------------------------------------------------------------------------
template <int MI, int NI, int NBUF, bool XCD = true>
__global__ __launch_bounds__(512) void gemm_bf16_glds8_kernel(
        const __bf16* __restrict__ A, const __bf16* __restrict__ B,
        __bf16* __restrict__ C, int M, int N, int K, EpilogueArgs ep) {
    constexpr int TBM = 2 * 16 * MI;     // 2 wave-rows
    constexpr int TBN = 4 * 16 * NI;     // 4 wave-cols
    constexpr int KB = BK;
    __shared__ __bf16 smem[NBUF][TBM + TBN][KB];

    int bx = blockIdx.x, by = blockIdx.y;
    if (XCD) {
        const int nb = gridDim.x * gridDim.y;
        const int id = xcd_swizzle(by * gridDim.x + bx, nb);
        bx = id % gridDim.x;
        by = id / gridDim.x;
    }
    const int bm = bx * TBM;
    const int bn = by * TBN;
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wid = tid >> 6;            // 0..7
    const int wm = (wid >> 2) * (16 * MI);
    const int wn = (wid & 3) * (16 * NI);

    const int srow = lane >> 3;          // row within an 8-row piece
    const int cdst = lane & 7;           // 16-B column chunk

    // pieces of 8 rows x 64 elems; (TBM+TBN)/8 pieces split across 8
    // waves; running per-piece pointers keep address math out of the loop
    constexpr int PIECES_A = TBM / 8 / 8;   // per wave
    constexpr int PIECES_B = TBN / 8 / 8;
    constexpr int GLDS_PER_TILE = PIECES_A + PIECES_B;
    const __bf16* a_pc[PIECES_A];
    const __bf16* b_pc[PIECES_B];
    #pragma unroll
    for (int i = 0; i < PIECES_A; ++i) {
        const int p = wid * PIECES_A + i;
        const int trow = p * 8 + srow;
        const int csrc = cdst ^ (trow & 7);
        a_pc[i] = A + (long)min(bm + trow, M - 1) * K + csrc * 8;
    }
    #pragma unroll
    for (int i = 0; i < PIECES_B; ++i) {
        const int p = wid * PIECES_B + i;
        const int trow = p * 8 + srow;
        const int csrc = cdst ^ (trow & 7);
        b_pc[i] = B + (long)min(bn + trow, N - 1) * K + csrc * 8;
    }
    auto stage = [&](int buf) {
        #pragma unroll
        for (int i = 0; i < PIECES_A; ++i) {
            const int p = wid * PIECES_A + i;
            glds_b128(a_pc[i], &smem[buf][p * 8][0]);
            a_pc[i] += KB;
        }
        #pragma unroll
        for (int i = 0; i < PIECES_B; ++i) {
            const int p = wid * PIECES_B + i;
            glds_b128(b_pc[i], &smem[buf][TBM + p * 8][0]);
            b_pc[i] += KB;
        }
    };

    f32x4 acc[MI][NI] = {};
    const int n_tiles = K / KB;
    #pragma unroll
    for (int p = 0; p < NBUF - 1; ++p)
        if (p < n_tiles) stage(p);

    // Same raw-barrier counted-vmcnt loop as the 256-thread glds3 kernel
    // (a stage-before-wait restructure with an extra barrier measured
    // SLOWER - sq4k 132->143us - because the post-barrier stage already
    // flies under compute); rotating buffer indices + constant vmcnt
    // immediates keep the modulo/switch SALU out of the hot loop.
    for (int t = 0, cbuf = 0, sbuf = NBUF - 1; t < n_tiles; ++t) {
        const int inflight = min(NBUF - 2, n_tiles - 1 - t);
        switch (inflight) {
        case 0:
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            break;
        case 1:
            asm volatile("s_waitcnt vmcnt(%0)" ::"i"(GLDS_PER_TILE)
                         : "memory");
            break;
        default:
            asm volatile("s_waitcnt vmcnt(%0)" ::"i"(2 * GLDS_PER_TILE)
                         : "memory");
            break;
        }
        __builtin_amdgcn_s_barrier();
        if (t + NBUF - 1 < n_tiles) {
            stage(sbuf);
            sbuf = sbuf + 1 == NBUF ? 0 : sbuf + 1;
        }
        const int buf = cbuf;
        cbuf = cbuf + 1 == NBUF ? 0 : cbuf + 1;
        #pragma unroll
        for (int kk = 0; kk < KB; kk += 32) {
            const int kgrp = kk + (lane >> 4) * 8;
            bf16x8 af[MI], bfr[NI];
            #pragma unroll
            for (int mi = 0; mi < MI; ++mi)
                af[mi] = lds_read_swz<KB>(&smem[buf][0][0],
                                          wm + mi * 16 + (lane & 15), kgrp);
            #pragma unroll
            for (int ni = 0; ni < NI; ++ni)
                bfr[ni] = lds_read_swz<KB>(&smem[buf][TBM][0],
                                           wn + ni * 16 + (lane & 15), kgrp);
            #pragma unroll
            for (int mi = 0; mi < MI; ++mi)
                #pragma unroll
                for (int ni = 0; ni < NI; ++ni)
                    acc[mi][ni] = mfma_16x16x32_bf16(af[mi], bfr[ni],
                                                     acc[mi][ni]);
        }
    }
    __builtin_amdgcn_s_barrier();
    gemm_epilogue<MI, NI, 0>(acc, ep, bm, bn, wm, wn, lane, 0, nullptr);
}

// ---------------------------------------------------------------------------
// Phase-segregated 256x256 kernel (t16): the guide's 8-phase discipline
// (cdna_hip_programming.md section 5 "256^2 8-phase template", measured
// 1320-1340 TF random-data vs ~1100 for the 2-barrier structure). Each
// K-tile is computed as 4 quadrant-phases; within a phase every wave
// posts its quadrant's 12 ds_read_b128 + 2 glds, hits a raw barrier +
// lgkmcnt(0), then issues 16 MFMAs under setprio(1) - reads and MFMAs are
// SEGREGATED so the matrix pipe runs the MFMA segment back-to-back for
// both co-resident waves instead of stalling on interleaved dependencies.
// Tile t+1 stages into the buffer not being read (2 glds/wave/phase); the
// tile boundary pays one vmcnt(0) for the phase-3-issued glds (a
// conservative deviation from the template's vmcnt(6), which needs a
// 2-tile staging lead the 2-buffer LDS cannot hold).
// ---------------------------------------------------------------------------
// PHV 0: 2 glds/phase, 2 barriers/phase, boundary vmcnt(0).
// PHV 1: glds front-loaded into phases 0-1 (boundary waits 2-phase-old
//        loads instead of just-issued ones).
// PHV 2: PHV1 + phase-end barrier dropped (reads of the next quadrant
//        overlap the partner wave's MFMA tail).
template <int PHV = 0>
__global__ __launch_bounds__(512) void gemm_bf16_phase8_kernel(
        const __bf16* __restrict__ A, const __bf16* __restrict__ B,
        __bf16* __restrict__ C, int M, int N, int K, EpilogueArgs ep) {
    constexpr int MI = 8, NI = 4;
    constexpr int TBM = 256, TBN = 256, KB = 64;
    __shared__ __bf16 smem[2][TBM + TBN][KB];

    int bx = blockIdx.x, by = blockIdx.y;
    {
        const int nb = gridDim.x * gridDim.y;
        const int id = xcd_swizzle(by * gridDim.x + bx, nb);
        bx = id % gridDim.x;
        by = id / gridDim.x;
    }
    const int bm = bx * TBM;
    const int bn = by * TBN;
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wid = tid >> 6;
    const int wm = (wid >> 2) * (16 * MI);
    const int wn = (wid & 3) * (16 * NI);

    // staging: 8 glds per wave per tile, 2 per phase
    const int srow = lane >> 3;
    const int cdst = lane & 7;
    const __bf16* a_pc[4];
    const __bf16* b_pc[4];
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int p = wid * 4 + i;
        const int trow = p * 8 + srow;
        const int csrc = cdst ^ (trow & 7);
        a_pc[i] = A + (long)min(bm + trow, M - 1) * K + csrc * 8;
        b_pc[i] = B + (long)min(bn + trow, N - 1) * K + csrc * 8;
    }
    // glds pair g (0..3) of buffer `buf`: A piece g for g<... interleave
    // A/B so each phase stages one A and one B piece
    auto stage2 = [&](int buf, int g) {
        const int p = wid * 4 + g;
        glds_b128(a_pc[g], &smem[buf][p * 8][0]);
        a_pc[g] += KB;
        glds_b128(b_pc[g], &smem[buf][TBM + p * 8][0]);
        b_pc[g] += KB;
    };

    f32x4 acc[MI][NI] = {};
    const int n_tiles = K / KB;
    // prologue: stage tile 0 fully, drain
    #pragma unroll
    for (int g = 0; g < 4; ++g) stage2(0, g);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();

    for (int t = 0; t < n_tiles; ++t) {
        const int buf = t & 1;
        const bool more = t + 1 < n_tiles;
        #pragma unroll
        for (int q = 0; q < 4; ++q) {
            // quadrant q = (mh, nh): M-frags mh*4.., N-frags nh*2..
            const int mh = q >> 1, nh = q & 1;
            bf16x8 af[4][2], bfr[2][2];
            #pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                const int kgrp = kk * 32 + (lane >> 4) * 8;
                #pragma unroll
                for (int mi = 0; mi < 4; ++mi)
                    af[mi][kk] = lds_read_swz<KB>(
                        &smem[buf][0][0],
                        wm + (mh * 4 + mi) * 16 + (lane & 15), kgrp);
                #pragma unroll
                for (int ni = 0; ni < 2; ++ni)
                    bfr[ni][kk] = lds_read_swz<KB>(
                        &smem[buf][TBM][0],
                        wn + (nh * 2 + ni) * 16 + (lane & 15), kgrp);
            }
            if (more) {
                if (PHV == 0) {
                    stage2(buf ^ 1, q);
                } else if (q < 2) {
                    stage2(buf ^ 1, 2 * q);
                    stage2(buf ^ 1, 2 * q + 1);
                }
            }
            __builtin_amdgcn_s_barrier();
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_setprio(1);
            #pragma unroll
            for (int kk = 0; kk < 2; ++kk)
                #pragma unroll
                for (int mi = 0; mi < 4; ++mi)
                    #pragma unroll
                    for (int ni = 0; ni < 2; ++ni)
                        acc[mh * 4 + mi][nh * 2 + ni] = mfma_16x16x32_bf16(
                            af[mi][kk], bfr[ni][kk],
                            acc[mh * 4 + mi][nh * 2 + ni]);
            __builtin_amdgcn_s_setprio(0);
            if (PHV < 2)
                __builtin_amdgcn_s_barrier();
        }
        // tile boundary: next phase reads buf^1; its glds were issued
        // during this tile's phases (latest in phase 3)
        if (more)
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
    }
    gemm_epilogue<MI, NI, 0>(acc, ep, bm, bn, wm, wn, lane, 0, nullptr);
}

// ---------------------------------------------------------------------------
// generic path: any K (padded LDS, plain vectorized staging)
// ---------------------------------------------------------------------------
template <int EPM = 0>
__global__ __launch_bounds__(256) void gemm_bf16_generic_kernel(
        const __bf16* __restrict__ A, const __bf16* __restrict__ B,
        __bf16* __restrict__ C, int M, int N, int K, EpilogueArgs ep) {
    __shared__ __bf16 As[BM][BK + PAD];
    __shared__ __bf16 Bs[BN][BK + PAD];

    const int bm = blockIdx.x * BM;
    const int bn = blockIdx.y * BN;
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wid = tid >> 6;
    const int wm = (wid >> 1) * 32;
    const int wn = (wid & 1) * 32;

    f32x4 acc[2][2] = {};

    for (int k0 = 0; k0 < K; k0 += BK) {
        #pragma unroll
        for (int it = 0; it < 2; ++it) {
            const int r = (tid >> 3) + it * 32;
            const int c = (tid & 7) * 8;
            const int gc = k0 + c;
            bf16x8 va = {}, vb = {};
            if (bm + r < M && gc + 7 < K) {
                va = *reinterpret_cast<const bf16x8*>(
                    A + (long)(bm + r) * K + gc);
            } else if (bm + r < M) {
                for (int j = 0; j < 8; ++j)
                    if (gc + j < K) va[j] = A[(long)(bm + r) * K + gc + j];
            }
            if (bn + r < N && gc + 7 < K) {
                vb = *reinterpret_cast<const bf16x8*>(
                    B + (long)(bn + r) * K + gc);
            } else if (bn + r < N) {
                for (int j = 0; j < 8; ++j)
                    if (gc + j < K) vb[j] = B[(long)(bn + r) * K + gc + j];
            }
            *reinterpret_cast<bf16x8*>(&As[r][c]) = va;
            *reinterpret_cast<bf16x8*>(&Bs[r][c]) = vb;
        }
        __syncthreads();

        #pragma unroll
        for (int kk = 0; kk < BK; kk += 32) {
            const int kgrp = kk + (lane >> 4) * 8;
            bf16x8 af[2], bfr[2];
            #pragma unroll
            for (int mi = 0; mi < 2; ++mi)
                af[mi] = *reinterpret_cast<const bf16x8*>(
                    &As[wm + mi * 16 + (lane & 15)][kgrp]);
            #pragma unroll
            for (int ni = 0; ni < 2; ++ni)
                bfr[ni] = *reinterpret_cast<const bf16x8*>(
                    &Bs[wn + ni * 16 + (lane & 15)][kgrp]);
            #pragma unroll
            for (int mi = 0; mi < 2; ++mi)
                #pragma unroll
                for (int ni = 0; ni < 2; ++ni)
                    acc[mi][ni] = mfma_16x16x32_bf16(af[mi], bfr[ni],
                                                     acc[mi][ni]);
        }
        __syncthreads();
    }

    float* lnbuf = reinterpret_cast<float*>(&As[0][0]);
    if constexpr (EPM == 1)
        ln_coeffs_to_lds<BM>(ep, bm, tid, lnbuf);
    gemm_epilogue<2, 2, EPM>(acc, ep, bm, bn, wm, wn, lane,
                             (bn / BN) * 2 + (wid & 1), lnbuf);
}

}  // namespace

std::tuple<torch::Tensor, torch::Tensor> gemm_bf16(
        torch::Tensor a2d, torch::Tensor b,
        c10::optional<torch::Tensor> bias, int64_t act,
        c10::optional<torch::Tensor> residual2d, int64_t tile,
        c10::optional<torch::Tensor> ln_stats,
        c10::optional<torch::Tensor> ln_s,
        c10::optional<torch::Tensor> ln_c, double ln_eps, bool want_stats) {
    TORCH_CHECK(a2d.is_cuda() && a2d.dtype() == torch::kBFloat16,
                "gemm: A must be bf16 on GPU");
    TORCH_CHECK(b.dtype() == torch::kBFloat16, "gemm: B must be bf16");
    TORCH_CHECK(a2d.dim() == 2 && b.dim() == 2);
    const int M = a2d.size(0), K = a2d.size(1), N = b.size(0);
    TORCH_CHECK(b.size(1) == K, "gemm: inner dims mismatch (B is [N,K])");
    auto a_c = a2d.contiguous();
    auto b_c = b.contiguous();
    auto out = torch::empty({M, N}, a2d.options());
    const __bf16* bias_p = nullptr;
    torch::Tensor bias_c;
    if (bias.has_value()) {
        bias_c = bias->contiguous();
        TORCH_CHECK(bias_c.numel() == N, "gemm: bias size mismatch");
        bias_p = reinterpret_cast<const __bf16*>(bias_c.data_ptr());
    }
    const __bf16* res_p = nullptr;
    torch::Tensor res_c;
    if (residual2d.has_value()) {
        res_c = residual2d->contiguous();
        TORCH_CHECK(res_c.size(0) == M && res_c.size(1) == N,
                    "gemm: residual shape mismatch");
        res_p = reinterpret_cast<const __bf16*>(res_c.data_ptr());
    }
    const auto* ap = reinterpret_cast<const __bf16*>(a_c.data_ptr());
    const auto* bp = reinterpret_cast<const __bf16*>(b_c.data_ptr());
    auto* cp = reinterpret_cast<__bf16*>(out.data_ptr());

    EpilogueArgs ep{bias_p, res_p, cp, M, N, (int)act,
                    nullptr, 0, nullptr, nullptr, (float)ln_eps, K,
                    1.0f / K, nullptr, 0};
    if (ln_stats.has_value()) {
        TORCH_CHECK(ln_s.has_value() && ln_c.has_value(),
                    "gemm: ln_stats requires ln_s and ln_c");
        TORCH_CHECK(ln_stats->dtype() == torch::kFloat32 &&
                    ln_stats->dim() == 3 && ln_stats->size(0) == M &&
                    ln_stats->size(2) == 2, "ln_stats must be [M, P, 2]");
        TORCH_CHECK(ln_s->numel() == N && ln_c->numel() == N);
        ep.ln_stats = ln_stats->data_ptr<float>();
        ep.ln_parts = ln_stats->size(1);
        ep.ln_s = ln_s->data_ptr<float>();
        ep.ln_c = ln_c->data_ptr<float>();
    }
    int t = 0;
    if (K % BK == 0) {
        // tile choice: empirically swept (tests/gpu sweep); override via
        // the `tile` arg (0 = auto heuristic)
        t = (int)tile;
        if (t == 0) {
            // experiment hook: PIPEEDGE_GEMM_T=<n> forces the auto choice
            // (bench A/Bs without a rebuild); callers passing tile!=0 win.
            static const int env_t = [] {
                const char* s = std::getenv("PIPEEDGE_GEMM_T");
                return s ? std::atoi(s) : 0;
            }();
            t = env_t;
        }
        if (t == 0) {
            // From the on-HW sweeps (round 2: tools/bigtile_sweep.py medians,
            // profiles/bigtile_sweep_r02.txt): the 512-thread 8-wave 256x256
            // 2-buffer kernel (t13) for the big near-square and ViT-H fc1
            // regimes (sq4k 127us vs r1-auto 162; vitH-fc1 55 vs 62; the r1
            // choice t2 also showed multi-hundred-us pathologies there);
            // 256x128 3-buffer (t14) for the ViT-L fc1 class; 3-buffer
            // 64x64 (t7) for mid-size long-K; XCD-swizzled 64x64 (t5)
            // otherwise.
            // PIPEEDGE_GEMM_MIDT overrides the mid-size (flagship-class)
            // default for e2e A/Bs: the SQ-wait PMC (profiles/
            // sqwait_r02.txt) shows the 2-buffer t5 parked 65% of wave
            // cycles vs 44% for the 3-buffer t7
            static const int midt = [] {
                const char* s = std::getenv("PIPEEDGE_GEMM_MIDT");
                return s ? std::atoi(s) : 0;
            }();
            if (M >= 3072 && N >= 3072 && K >= 2048) t = 13;
            // t15 (256x192) for the wide-N M>=2048 class: solo probes say
            // t7 is faster at shallow K (s384-fc1 44.8 vs 53.6us,
            // profiles/m3072_probe.txt) but the s384 e2e bench REGRESSED
            // 6.1k -> 5.7k items/s with t7 there - t15's single-block/CU
            // footprint co-schedules better with the second microbatch
            // stream. e2e wins over solo: keep t15.
            else if (M >= 2048) t = (N >= 3072) ? 15 : 5;
            // the wide-N branches below were tuned at M=1576 (ViT); at
            // M=1024 (BERT u8 s128) t5 wins them (bertL-fc1: 28.9us vs
            // t14 37.9 / t7 31.7 - profiles/bertL_probe.txt)
            else if (M >= 1280 && N >= 4096 && K < 2048) t = 14;
            else if (K >= 2048 || (N >= 3072 && M >= 1280)) t = 7;
            else if (midt != 0 && M >= 256) t = midt;
            else t = 5;
        }
        if (t == 4 && K % (2 * BK) != 0) t = 1;
        if (t == 6 && K % (2 * BK) != 0) t = 5;

    }
    torch::Tensor stats;
    if (want_stats) {
        const int bn_tile = (t == 3 || t == 9) ? 128 : 64;
        const int parts = ((N + bn_tile - 1) / bn_tile) * 2;
        stats = torch::empty({M, parts, 2},
                             a2d.options().dtype(torch::kFloat32));
        ep.stats_out = stats.data_ptr<float>();
        ep.stats_parts = parts;
    } else {
        stats = torch::empty({0}, a2d.options().dtype(torch::kFloat32));
    }
    const int epm = ep.ln_stats != nullptr ? 1
                    : (ep.stats_out != nullptr ? 2 : 0);
#define PE_LAUNCH_GLDS(MI_, NI_, KT_, XCD_, GRID_)                           \
    do {                                                                     \
        if (epm == 1)                                                        \
            hipLaunchKernelGGL(                                              \
                (gemm_bf16_glds_kernel<MI_, NI_, KT_, XCD_, 1>), GRID_,      \
                dim3(256), 0, pe_current_stream(), ap, bp, cp, M, N, K, ep); \
        else if (epm == 2)                                                   \
            hipLaunchKernelGGL(                                              \
                (gemm_bf16_glds_kernel<MI_, NI_, KT_, XCD_, 2>), GRID_,      \
                dim3(256), 0, pe_current_stream(), ap, bp, cp, M, N, K, ep); \
        else                                                                 \
            hipLaunchKernelGGL(                                              \
                (gemm_bf16_glds_kernel<MI_, NI_, KT_, XCD_, 0>), GRID_,      \
                dim3(256), 0, pe_current_stream(), ap, bp, cp, M, N, K, ep); \
    } while (0)
    if (K % BK == 0) {
#define PE_LAUNCH_GLDS3(MI_, NI_, NBUF_, GRID_)                              \
    do {                                                                     \
        if (epm == 1)                                                        \
            hipLaunchKernelGGL(                                              \
                (gemm_bf16_glds3_kernel<MI_, NI_, true, 1, NBUF_>), GRID_,   \
                dim3(256), 0, pe_current_stream(), ap, bp, cp, M, N, K, ep); \
        else if (epm == 2)                                                   \
            hipLaunchKernelGGL(                                              \
                (gemm_bf16_glds3_kernel<MI_, NI_, true, 2, NBUF_>), GRID_,   \
                dim3(256), 0, pe_current_stream(), ap, bp, cp, M, N, K, ep); \
        else                                                                 \
            hipLaunchKernelGGL(                                              \
                (gemm_bf16_glds3_kernel<MI_, NI_, true, 0, NBUF_>), GRID_,   \
                dim3(256), 0, pe_current_stream(), ap, bp, cp, M, N, K, ep); \
    } while (0)
        if (t == 20 && epm == 0) {
            // split-K in-launch-combine for CU-underfilled grids; slice
            // count from PIPEEDGE_GEMM_SK (default 2)
            const char* sk_s = std::getenv("PIPEEDGE_GEMM_SK");
            const int sk_env = sk_s ? std::atoi(sk_s) : 2;
            int sk = sk_env < 2 ? 2 : sk_env;
            if (sk > K / BK) sk = K / BK;
            dim3 grid((M + BM - 1) / BM, (N + BN - 1) / BN, sk);
            const long ntiles = (long)grid.x * grid.y;
            auto slabs = torch::empty({ntiles * sk * 256 * 16},
                                      a2d.options().dtype(torch::kFloat32));
            auto tickets = torch::zeros({ntiles},
                                        a2d.options().dtype(torch::kInt32));
            hipLaunchKernelGGL((gemm_bf16_splitk_kernel<2, 2, 3>), grid,
                               dim3(256), 0, pe_current_stream(), ap, bp, cp,
                               M, N, K, slabs.data_ptr<float>(),
                               reinterpret_cast<unsigned int*>(
                                   tickets.data_ptr<int>()),
                               ep);
        } else if ((t == 12 || t == 13 || t == 14) && epm == 0) {
            // 8-wave big-tile kernels (epilogue modes 1/2 unsupported here;
            // the auto heuristic only picks these for plain big shapes)
            if (t == 12) {
                dim3 grid((M + 127) / 128, (N + 255) / 256);
                hipLaunchKernelGGL((gemm_bf16_glds8_kernel<4, 4, 3>), grid,
                                   dim3(512), 0, pe_current_stream(), ap, bp,
                                   cp, M, N, K, ep);
            } else if (t == 13) {
                dim3 grid((M + 255) / 256, (N + 255) / 256);
                hipLaunchKernelGGL((gemm_bf16_glds8_kernel<8, 4, 2>), grid,
                                   dim3(512), 0, pe_current_stream(), ap, bp,
                                   cp, M, N, K, ep);
            } else {
                dim3 grid((M + 255) / 256, (N + 127) / 128);
                hipLaunchKernelGGL((gemm_bf16_glds8_kernel<8, 2, 3>), grid,
                                   dim3(512), 0, pe_current_stream(), ap, bp,
                                   cp, M, N, K, ep);
            }
        } else if (t == 16 && epm == 0) {
            dim3 grid((M + 255) / 256, (N + 255) / 256);
            const char* pv = std::getenv("PIPEEDGE_P8V");
            const int phv = pv ? std::atoi(pv) : 1;
            if (phv == 2)
                hipLaunchKernelGGL((gemm_bf16_phase8_kernel<2>), grid,
                                   dim3(512), 0, pe_current_stream(), ap, bp,
                                   cp, M, N, K, ep);
            else if (phv == 0)
                hipLaunchKernelGGL((gemm_bf16_phase8_kernel<0>), grid,
                                   dim3(512), 0, pe_current_stream(), ap, bp,
                                   cp, M, N, K, ep);
            else
                hipLaunchKernelGGL((gemm_bf16_phase8_kernel<1>), grid,
                                   dim3(512), 0, pe_current_stream(), ap, bp,
                                   cp, M, N, K, ep);
        } else if (t == 15 && epm == 0) {
            // 256x192 2-buffer (112 KiB LDS): ViT-H fc1 grid = 9x27 = 243
            // blocks ~ one full chip wave (256x256 gives only 180)
            dim3 grid((M + 255) / 256, (N + 191) / 192);
            hipLaunchKernelGGL((gemm_bf16_glds8_kernel<8, 3, 2>), grid,
                               dim3(512), 0, pe_current_stream(), ap, bp,
                               cp, M, N, K, ep);
        } else if (t == 7 || t == 12 || t == 13 || t == 14 || t == 15 ||
                   t == 16 || t == 20) {
            dim3 grid((M + BM - 1) / BM, (N + BN - 1) / BN);
            PE_LAUNCH_GLDS3(2, 2, 3, grid);
        } else if (t == 10) {
            // 4-buffer pipeline: one more tile in flight, 2 blocks/CU
            dim3 grid((M + BM - 1) / BM, (N + BN - 1) / BN);
            PE_LAUNCH_GLDS3(2, 2, 4, grid);
        } else if (t == 8) {
            // 128x64 3-buffer: double arithmetic intensity vs t7 (the 64x64
            // tiles are HBM/L2-bound at ~32 FLOP/B); 72 KiB LDS -> 2/CU
            dim3 grid((M + 127) / 128, (N + BN - 1) / BN);
            PE_LAUNCH_GLDS3(4, 2, 3, grid);
        } else if (t == 9) {
            // 128x128 3-buffer: 96 KiB LDS -> 1/CU
            dim3 grid((M + 127) / 128, (N + 127) / 128);
            PE_LAUNCH_GLDS3(4, 4, 3, grid);
        } else if (t == 4 || t == 5 || t == 6) {
            dim3 grid((M + BM - 1) / BM, (N + BN - 1) / BN);
            if (t == 4) PE_LAUNCH_GLDS(2, 2, 2, false, grid);
            else if (t == 5) PE_LAUNCH_GLDS(2, 2, 1, true, grid);
            else PE_LAUNCH_GLDS(2, 2, 2, true, grid);
        } else if (t == 3) {
            dim3 grid((M + 127) / 128, (N + 127) / 128);
            PE_LAUNCH_GLDS(4, 4, 1, false, grid);
        } else if (t == 2) {
            dim3 grid((M + 127) / 128, (N + 63) / 64);
            PE_LAUNCH_GLDS(4, 2, 1, false, grid);
        } else {
            dim3 grid((M + BM - 1) / BM, (N + BN - 1) / BN);
            PE_LAUNCH_GLDS(2, 2, 1, false, grid);
        }
    } else {
        dim3 grid((M + BM - 1) / BM, (N + BN - 1) / BN);
        if (epm == 1)
            hipLaunchKernelGGL((gemm_bf16_generic_kernel<1>), grid, dim3(256),
                               0, pe_current_stream(), ap, bp, cp, M, N, K,
                               ep);
        else if (epm == 2)
            hipLaunchKernelGGL((gemm_bf16_generic_kernel<2>), grid, dim3(256),
                               0, pe_current_stream(), ap, bp, cp, M, N, K,
                               ep);
        else
            hipLaunchKernelGGL((gemm_bf16_generic_kernel<0>), grid, dim3(256),
                               0, pe_current_stream(), ap, bp, cp, M, N, K,
                               ep);
    }
#undef PE_LAUNCH_GLDS
#undef PE_LAUNCH_GLDS3
    HIP_CHECK_LAST();
    return {out, stats};
}

// debug helper: one 16x16x32 MFMA tile with the documented fragment layout -
// used by the GPU tests to pin the lane->element mapping on real hardware
torch::Tensor debug_mfma_tile(torch::Tensor a, torch::Tensor b);

namespace {
__global__ void debug_mfma_kernel(const __bf16* __restrict__ A,
                                  const __bf16* __restrict__ B,
                                  float* __restrict__ D) {
    const int lane = threadIdx.x & 63;
    bf16x8 a, b;
    #pragma unroll
    for (int j = 0; j < 8; ++j) {
        a[j] = A[(lane & 15) * 32 + (lane >> 4) * 8 + j];   // A[row][k]
        b[j] = B[((lane >> 4) * 8 + j) * 16 + (lane & 15)]; // B[k][col]
    }
    f32x4 c = {};
    c = mfma_16x16x32_bf16(a, b, c);
    #pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int row = (lane >> 4) * 4 + r;
        const int col = lane & 15;
        D[row * 16 + col] = c[r];
    }
}
}  // namespace

torch::Tensor debug_mfma_tile(torch::Tensor a, torch::Tensor b) {
    TORCH_CHECK(a.sizes() == torch::IntArrayRef({16, 32}));
    TORCH_CHECK(b.sizes() == torch::IntArrayRef({32, 16}));
    auto a_c = a.to(torch::kBFloat16).contiguous();
    auto b_c = b.to(torch::kBFloat16).contiguous();
    auto out = torch::empty({16, 16}, a.options().dtype(torch::kFloat32));
    hipLaunchKernelGGL(debug_mfma_kernel, dim3(1), dim3(64), 0,
                       pe_current_stream(),
                       reinterpret_cast<const __bf16*>(a_c.data_ptr()),
                       reinterpret_cast<const __bf16*>(b_c.data_ptr()),
                       out.data_ptr<float>());
    HIP_CHECK_LAST();
    return out;
}
