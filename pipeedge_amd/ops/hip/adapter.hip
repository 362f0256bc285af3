// Projection with low-rank adapters of many requests,
//   y = act(x W^T + b + s_i (x A_i^T) B_i^T) + residual,   i = id of the row,
// in two launches: the inner values s_i x A_i^T of all rows, and the shared
// product, which adds theirs with B_i to its accumulators before bias and
// activation, so y is written once and W is read as without adapters. The
// inner values are rounded to bf16 once, as the operand of the second product;
// the sums before and after stay in fp32. Few rows are bound by the latency of
// two launches and of reading W (8 rows, 1024 to 4096 columns, rank 16: 10 us),
// many by the product and by its epilogue, which nothing hides with one block a
// CU (12608 rows, 1280 to 5120 columns, rank 64, gelu: 12 us and 233, 710
// TFLOP/s). Each further adapter among a tile's rows is a turn of its own in
// both launches (4096 rows, 1280 to 1280, rank 64, ids mixed row by row: 28 us
// without adapters, 36 with one, 88 with 8, 462 with 64).
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>

#include <algorithm>

#include "common.h"
#include "mfma_tiles.h"

namespace {

// Which rows belong to which adapter, and what the second product reads.
struct AdapterRows {
    const __bf16* inner;        // [M][rank_pad], zero behind rank
    const __bf16* up;           // [n_adapters][N][rank]
    const int* row_ids;         // one for rows_per_id rows each
    int rows_per_id, n_adapters, rank, rank_pad;
};

struct ProductArgs {
    const __bf16 *x, *w, *bias, *residual;
    __bf16* out;
    int M, N, K, act;
    bool vec;                   // K a multiple of 8
    int m_blocks, n_blocks;
    AdapterRows ad;
};

struct InnerArgs {
    const __bf16* x;            // [M][K]
    const __bf16* down;         // [n][rank][K]
    const int* row_ids;
    const float* scales;        // [n] or nullptr
    __bf16* inner;              // [M][rank_pad]
    int M, K, rows_per_id, n_adapters, rank, rank_pad;
    int item_rows, item_blocks; // rows that blocks do not cross
    bool vec;                   // rows lie at multiples of 16 bytes
    // up with its rows padded to whole chunks, or nullptr
    const __bf16* up;           // [up_rows][rank]
    __bf16* up_padded;          // [up_rows][chunks][8]
    long up_rows;
    int row_blocks;             // blocks behind these pad
};

__device__ __forceinline__ bf16x8 inner_load(const __bf16* p, int k, int K,
                                             bool vec) {
    bf16x8 v = {};
    if (vec) {
        if (k < K) v = *reinterpret_cast<const bf16x8*>(p + k);
    } else {
        #pragma unroll
        for (int j = 0; j < 8; ++j)
            if (k + j < K) v[j] = p[k + j];
    }
    return v;
}

// The blocks behind a.row_blocks: rows of up as whole chunks of 8.
__device__ __forceinline__ void pad_rows(const InnerArgs& a) {
    if (blockIdx.y > 0) return;
    const int chunks = (a.rank + 7) / 8;
    const long count = a.up_rows * chunks;
    const long step = (long)(gridDim.x - a.row_blocks) * blockDim.x;
    for (long i = (long)(blockIdx.x - a.row_blocks) * blockDim.x
                  + threadIdx.x; i < count; i += step) {
        const long row = i / chunks;
        reinterpret_cast<bf16x8*>(a.up_padded)[i] = inner_load(
            a.up + row * a.rank, (int)(i - row * chunks) * 8, a.rank, false);
    }
}

// x Phi(x) with Phi(-z) = exp(-z^2 / 2) r(z), z >= 0. r, the half of the
// scaled complementary error function, falls slowly, and a polynomial of
// degree 8 in 1 / (1 + 0.29 z) follows it to 4e-7 of its value on [0, 16]
// (own least squares fit, reweighted towards the largest error), where the
// exponential ends. With one block a CU nothing else hides the epilogue (12608
// rows, 1280 to 5120 columns, rank 64: 239 us without an activation, 251 with
// this one, 299 with the library's erfc).
__device__ __forceinline__ float gelu_tail(float x) {
    const float z = fabsf(x);
    const float t = __builtin_amdgcn_rcpf(fmaf(0.29f, z, 1.0f));
    float r = 0.03704957291483879f;
    r = fmaf(r, t, -0.18275977671146393f);
    r = fmaf(r, t, 0.2875499427318573f);
    r = fmaf(r, t, -0.13273395597934723f);
    r = fmaf(r, t, 0.17503269016742706f);
    r = fmaf(r, t, 0.08038167655467987f);
    r = fmaf(r, t, 0.12021259218454361f);
    r = fmaf(r, t, 0.11524859070777893f);
    r = fmaf(r, t, 1.8610380720929243e-05f);
    // exp(-z^2 / 2) in powers of two
    r *= __builtin_amdgcn_exp2f(z * z * -0.72134752044448170f);
    return x * (x < 0.0f ? r : 1.0f - r);
}

// Many rows: a block takes 16 rows by 16 * NC inner columns, its 4 waves a
// quarter of K each, for each adapter among the rows; the waves' sums meet in
// LDS and rows keep those of their own adapter.
template <int NC, bool VEC>
__global__ __launch_bounds__(256) void adapter_inner_kernel(InnerArgs a) {
    constexpr int DEPTH = 4;    // steps of 32 whose loads are on their way
    __shared__ float parts[4][NC][64][4];
    if (blockIdx.x >= a.row_blocks) { pad_rows(a); return; }
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
    const int l15 = lane & 15, quad = lane >> 4;
    const int row0 = blockIdx.x * 16, col0 = blockIdx.y * 16 * NC;
    const int row = row0 + l15;
    int id = row < a.M ? a.row_ids[row / a.rows_per_id] : -1;
    if (id >= a.n_adapters) id = -1;

    const int steps = (a.K + 31) / 32;
    const int first = wid * steps / 4, last = (wid + 1) * steps / 4;
    const int whole = min(last, a.K / 32);      // steps inside K
    const __bf16* x = a.x + (long)min(row, a.M - 1) * a.K + quad * 8;
    f32x4 mine[NC] = {};
    unsigned long long left = __ballot(id >= 0);
    while (left) {
        const int cur = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
        left &= ~__ballot(id == cur);
        const unsigned rows = (unsigned)__ballot(id == cur) >> (quad * 4);
        const __bf16* down = a.down + (long)cur * a.rank * a.K + quad * 8;
        const __bf16* d[NC];
        #pragma unroll
        for (int n = 0; n < NC; ++n)
            d[n] = down + (long)min(col0 + n * 16 + l15, a.rank - 1) * a.K;
        f32x4 acc[NC] = {};
        int s = first;
        if constexpr (VEC)
            for (; s + DEPTH <= whole; s += DEPTH) {
                bf16x8 xv[DEPTH], dv[DEPTH][NC];
                #pragma unroll
                for (int i = 0; i < DEPTH; ++i) {
                    const int k = (s + i) * 32;
                    xv[i] = *reinterpret_cast<const bf16x8*>(x + k);
                    #pragma unroll
                    for (int n = 0; n < NC; ++n)
                        dv[i][n] = *reinterpret_cast<const bf16x8*>(d[n] + k);
                }
                // all loads before the first wait
                __builtin_amdgcn_sched_barrier(0);
                #pragma unroll
                for (int i = 0; i < DEPTH; ++i)
                    #pragma unroll
                    for (int n = 0; n < NC; ++n)
                        acc[n] = mfma_16x16x32_bf16(xv[i], dv[i][n], acc[n]);
            }
        for (; s < last; ++s) {
            const int k = s * 32, end = a.K - quad * 8;
            const bf16x8 xv = inner_load(x, k, end, VEC);
            #pragma unroll
            for (int n = 0; n < NC; ++n)
                acc[n] = mfma_16x16x32_bf16(xv, inner_load(d[n], k, end, VEC),
                                            acc[n]);
        }
        #pragma unroll
        for (int n = 0; n < NC; ++n)
            #pragma unroll
            for (int r = 0; r < 4; ++r)
                if ((rows >> r) & 1) mine[n][r] = acc[n][r];
    }
    #pragma unroll
    for (int n = 0; n < NC; ++n)
        *reinterpret_cast<f32x4*>(parts[wid][n][lane]) = mine[n];
    __syncthreads();
    // 16 columns a wave; the padding behind the last is written by the last
    // block of columns
    const int pad = blockIdx.y + 1 == gridDim.y ? a.rank_pad
                                                : col0 + 16 * NC;
    for (int n = wid; col0 + n * 16 < pad; n += 4) {
        const int col = col0 + n * 16 + l15;
        #pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int out_row = row0 + quad * 4 + r;
            const int out_id = __shfl(id, quad * 4 + r);
            if (out_row >= a.M) continue;
            float v = 0.0f;
            if (n < NC && col < a.rank && out_id >= 0) {
                v = parts[0][n][lane][r] + parts[1][n][lane][r]
                    + parts[2][n][lane][r] + parts[3][n][lane][r];
                if (a.scales != nullptr) v *= a.scales[out_id];
            }
            a.inner[(long)out_row * a.rank_pad + col] = f2bf(v);
        }
    }
}

// The same through LDS, for so many rows that the operands' way into the
// registers is the bound: fragments loaded straight from memory come in
// pieces of 64 B, at a quarter of the rate of whole lines, and each wave
// loads the adapters for itself. A block takes 32 WM rows by 32 WN inner
// columns; WK groups of waves take a part of K each, in slices of 64 that are
// loaded BUFS - 1 turns ahead of their use.
template <int WN, int WM, int WK, int BUFS>
__global__ __launch_bounds__(64 * WN * WM * WK)
void adapter_inner_tile_kernel(InnerArgs a) {
    constexpr int BN = 32 * WN, BM = 32 * WM, BK = 64, CH = BK / 8;
    constexpr int SLICE = (BN + BM) * BK;
    constexpr int PIECES = (BN + BM) / 8 / (WN * WM);
    typedef TileVec<__bf16>::v8 v8;
    __shared__ __attribute__((aligned(256))) __bf16 lds[WK * BUFS * SLICE];
    if (blockIdx.x >= a.row_blocks) { pad_rows(a); return; }

    const int tid = threadIdx.x, lane = tid & 63;
    const int l31 = lane & 31, hi = lane >> 5;
    const int all = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wid = all % (WN * WM), wk = all / (WN * WM);
    const int wn = wid % WN, wm = wid / WN;
    const int item = blockIdx.x / a.item_blocks;
    const int m0 = item * a.item_rows
                   + (blockIdx.x - item * a.item_blocks) * BM;
    const int end = min(m0 + BM, (item + 1) * a.item_rows);
    const int n0 = blockIdx.y * BN;
    __bf16* const smem = lds + wk * BUFS * SLICE;

    // adapters of the block's rows, row l and l + 64 in lane l
    int left[(BM + 63) / 64];
    #pragma unroll
    for (int i = 0; i < (BM + 63) / 64; ++i) {
        const int r = i * 64 + lane;
        const int v = r < BM && m0 + r < end
            ? a.row_ids[(m0 + r) / a.rows_per_id] : -1;
        left[i] = v < a.n_adapters ? v : -1;
    }
    const int row = m0 + wm * 32 + l31;
    const int id = row < end ? a.row_ids[row / a.rows_per_id] : -1;
    // slices of this part of K; all parts take as many turns
    const int turns = ((a.K + BK - 1) / BK + WK - 1) / WK;
    const int slice0 = wk * turns;
    const int slices = min(turns, max(0, (a.K + BK - 1) / BK - slice0));
    const auto fast = [&](int t) {
        return a.vec && (slice0 + t + 1) * BK <= a.K;
    };

    while (true) {
        int cur = -1;
        #pragma unroll
        for (int i = 0; i < (BM + 63) / 64; ++i) {
            const unsigned long long has = __ballot(left[i] >= 0);
            if (cur < 0 && has)
                cur = __builtin_amdgcn_readlane(left[i],
                                                __builtin_ctzll(has));
        }
        if (cur < 0) break;
        #pragma unroll
        for (int i = 0; i < (BM + 63) / 64; ++i)
            if (left[i] == cur) left[i] = -1;
        const __bf16* down = a.down + (long)cur * a.rank * a.K;

        const auto stage = [&](int t) {
            __bf16* image = smem + (t % BUFS) * SLICE;
            #pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const int r = (wid * PIECES + i) * 8 + lane / CH;
                const int c = (lane % CH) ^ tile_key<CH>(r);
                const __bf16* from = r < BN
                    ? down + (long)min(n0 + r, a.rank - 1) * a.K
                    : a.x + (long)min(m0 + r - BN, end - 1) * a.K;
                __bf16* to = image + (wid * PIECES + i) * 512;
                const int k = (slice0 + t) * BK + c * 8;
                if (fast(t))
                    tile_load(from + k, to);
                else
                    *reinterpret_cast<bf16x8*>(to + lane * 8) =
                        inner_load(from, k, a.K, a.vec);
            }
        };
        f32x16 acc = {};
        const unsigned base = tile_row_base<CH, 32>(tile_lds(smem), lane);
        __syncthreads();
        #pragma unroll
        for (int t = 0; t < BUFS - 1; ++t)
            if (t < slices) stage(t);
        for (int t = 0; t < turns; ++t) {
            // slice t is here; those behind it may be on their way
            if (BUFS == 4 && t + 2 < slices && fast(t + 2))
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)"
                             ::"i"(2 * PIECES) : "memory");
            else if (t + 1 < slices && fast(t + 1))
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)"
                             ::"i"(PIECES) : "memory");
            else
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            // into the buffer that every wave left before the barrier
            if (t + BUFS - 1 < slices) stage(t + BUFS - 1);
            if (t >= slices) continue;
            const unsigned at = base + (t % BUFS) * SLICE * 2;
            #pragma unroll
            for (int s = 0; s < BK / 16; ++s) {
                const v8 d = tile_row_read<__bf16, CH, 32>(
                    at + wn * 32 * BK * 2, 0, s);
                const v8 x = tile_row_read<__bf16, CH, 32>(
                    at + (BN + wm * 32) * BK * 2, 0, s);
                acc = tile_mfma(d, x, acc);
            }
        }
        if constexpr (WK > 1) {
            // the parts of K meet in LDS, in their order
            __syncthreads();
            f32x16* sums = reinterpret_cast<f32x16*>(lds)
                           + wid * 64 + lane;
            static_assert(WN * WM * (WK - 1) * 64 * 64
                          <= WK * BUFS * SLICE * 2, "room for the sums");
            if (wk > 0) sums[(wk - 1) * WN * WM * 64] = acc;
            __syncthreads();
            if (wk == 0)
                #pragma unroll
                for (int p = 0; p < WK - 1; ++p)
                    acc += sums[p * WN * WM * 64];
        }
        if (wk == 0 && id == cur) {
            const float scale = a.scales != nullptr ? a.scales[cur] : 1.0f;
            #pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int col = n0 + wn * 32 + g * 8 + hi * 4;
                TileVec<__bf16>::v4 o;
                #pragma unroll
                for (int j = 0; j < 4; ++j)
                    o[j] = f2bf(col + j < a.rank ? acc[g * 4 + j] * scale
                                                 : 0.0f);
                *reinterpret_cast<TileVec<__bf16>::v4*>(
                    a.inner + (long)row * a.rank_pad + col) = o;
            }
        }
    }
}

// Few rows, or few of each adapter: a wave takes one row and 4 inner columns,
// a block 16 of them. The matrix unit would be idle for want of rows; what
// counts is that all the adapters' rows are on their way at once.
__global__ __launch_bounds__(256) void adapter_inner_step_kernel(
        InnerArgs a) {
    if (blockIdx.x >= a.row_blocks) { pad_rows(a); return; }
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    const int row = blockIdx.x, col0 = blockIdx.y * 16 + wid * 4;
    int id = a.row_ids[row / a.rows_per_id];
    float sum[4] = {};
    if (id >= 0 && id < a.n_adapters) {
        const __bf16* x = a.x + (long)row * a.K;
        const __bf16* down = a.down + (long)id * a.rank * a.K;
        const __bf16* d[4];
        #pragma unroll
        for (int c = 0; c < 4; ++c)
            d[c] = down + (long)min(col0 + c, a.rank - 1) * a.K;
        #pragma unroll 2
        for (int k = lane * 8; k < a.K; k += 512) {
            const bf16x8 xv = inner_load(x, k, a.K, a.vec);
            #pragma unroll
            for (int c = 0; c < 4; ++c) {
                const bf16x8 dv = inner_load(d[c], k, a.K, a.vec);
                #pragma unroll
                for (int j = 0; j < 8; ++j)
                    sum[c] = fmaf(bf2f(xv[j]), bf2f(dv[j]), sum[c]);
            }
        }
        const float scale = a.scales != nullptr ? a.scales[id] : 1.0f;
        #pragma unroll
        for (int c = 0; c < 4; ++c)
            sum[c] = wave64_reduce(sum[c], SumOp()) * scale;
    }
    if (lane == 0)
        #pragma unroll
        for (int c = 0; c < 4; ++c)
            a.inner[(long)row * a.rank_pad + col0 + c] =
                f2bf(col0 + c < a.rank ? sum[c] : 0.0f);
}

// The whole projection of few rows. Bound by reading W: a block takes 16
// columns and all rows, its waves a part of K each, so that 4096 columns are
// on 256 CUs and every wave has its loads on the way before it needs one (cold,
// whole projection, us with 4 waves and with 8: 5120 to 1280 columns, 8 rows 28
// and 24; 1024 to 4096, 8 rows 13.4 and 13.4, 64 rows 18.6 and 16.6).
// The adapters' products are a short dot product for each output.
constexpr int STEP_WAVES = 8;

template <int NM>               // groups of 16 rows
__global__ __launch_bounds__(64 * STEP_WAVES) void adapter_step_kernel(
        ProductArgs a) {
    const int M = a.M, N = a.N, K = a.K;
    const AdapterRows& ad = a.ad;
    constexpr int DEPTH = 4;    // steps of 32 in flight
    __shared__ float parts[STEP_WAVES][NM][16][17];
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
    const int l15 = lane & 15, quad = lane >> 4;
    const int col0 = blockIdx.x * 16;

    const int steps = (K + 31) / 32;
    const int first = wid * steps / STEP_WAVES;
    const int last = (wid + 1) * steps / STEP_WAVES;
    const __bf16* wp = a.w + (long)min(col0 + l15, N - 1) * K + quad * 8;
    const __bf16* xp[NM];
    #pragma unroll
    for (int m = 0; m < NM; ++m)
        xp[m] = a.x + (long)min(m * 16 + l15, M - 1) * K + quad * 8;
    f32x4 acc[NM] = {};
    for (int s0 = first; s0 < last; s0 += DEPTH) {
        bf16x8 wv[DEPTH], xv[DEPTH][NM];
        #pragma unroll
        for (int s = 0; s < DEPTH; ++s) {
            // behind the wave's part nothing is loaded
            const int k = (s0 + s) * 32;
            const int end = s0 + s < last ? K - quad * 8 : 0;
            wv[s] = inner_load(wp, k, end, a.vec);
            #pragma unroll
            for (int m = 0; m < NM; ++m)
                xv[s][m] = inner_load(xp[m], k, end, a.vec);
        }
        __builtin_amdgcn_sched_barrier(0);
        #pragma unroll
        for (int s = 0; s < DEPTH; ++s)
            #pragma unroll
            for (int m = 0; m < NM; ++m)
                acc[m] = mfma_16x16x32_bf16(wv[s], xv[s][m], acc[m]);
    }
    // lane: row m * 16 + l15, columns quad * 4 ..
    #pragma unroll
    for (int m = 0; m < NM; ++m)
        #pragma unroll
        for (int r = 0; r < 4; ++r)
            parts[wid][m][l15][quad * 4 + r] = acc[m][r];
    __syncthreads();
    #pragma unroll
    for (int o = tid; o < NM * 256; o += 64 * STEP_WAVES) {
        const int row = o / 16, c = o % 16, col = col0 + c;
        if (row >= M || col >= N) continue;
        float v = 0.0f;
        #pragma unroll
        for (int p = 0; p < STEP_WAVES; ++p)
            v += parts[p][row / 16][row % 16][c];
        const int id = ad.row_ids[row / ad.rows_per_id];
        if (id >= 0 && id < ad.n_adapters) {
            const __bf16* in = ad.inner + (long)row * ad.rank_pad;
            const __bf16* up = ad.up + ((long)id * N + col) * ad.rank;
            for (int k = 0; k < ad.rank; k += 8) {
                const bf16x8 av = inner_load(in, k, ad.rank_pad, true);
                const bf16x8 bv = inner_load(up, k, ad.rank,
                                            ad.rank % 8 == 0);
                #pragma unroll
                for (int j = 0; j < 8; ++j)
                    v = fmaf(bf2f(av[j]), bf2f(bv[j]), v);
            }
        }
        if (a.bias != nullptr) v += bf2f(a.bias[col]);
        if (a.act == ACT_GELU) v = gelu_tail(v);
        else if (a.act == ACT_TANH) v = tanhf(v);
        if (a.residual != nullptr) v += bf2f(a.residual[(long)row * N + col]);
        a.out[(long)row * N + col] = f2bf(v);
    }
}

// Activation, residual and rounding of up to 8 adjacent columns.
__device__ __forceinline__ void finish8(float (&v)[8], const __bf16* residual,
                                        __bf16* out, long at, int count,
                                        bool whole, int act) {
    if (act == ACT_GELU) {
        #pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = gelu_tail(v[j]);
    } else if (act == ACT_TANH) {
        #pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = tanhf(v[j]);
    }
    if (residual != nullptr) {
        const bf16x8 r = inner_load(residual + at, 0, count, whole);
        #pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += bf2f(r[j]);
    }
    bf16x8 o;
    #pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = f2bf(v[j]);
    if (whole) {
        *reinterpret_cast<bf16x8*>(out + at) = o;
    } else {
        #pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < count) out[at + j] = o[j];
    }
}

// The whole projection of many rows, as y^T = W x^T on 32x32x16 MFMAs: a lane
// then holds columns of one row, so the row's adapter is a property of the
// lane, and four adjacent columns leave together. A block computes BN columns
// of BM rows in WN x WM waves of 32 NI columns by 32 MI rows each. Slices of
// 64 of K go to LDS by LDS-DMA, two buffers; operands are read from LDS one
// step of 16 ahead of their MFMAs, also across slices: the barrier that ends
// a slice comes before its last step, whose operands are in registers by
// then.

// Columns and rows of the block: in each XCD's contiguous share of the work,
// bands of 8 row blocks, column by column, so that the blocks that run at the
// same time share slices of both operands in that XCD's L2.
__device__ __forceinline__ void product_place(const ProductArgs& a, int& bm,
                                              int& bn) {
    const int id = xcd_contiguous(blockIdx.x, gridDim.x);
    const int band = id / (8 * a.n_blocks), first = band * 8;
    const int high = min(8, a.m_blocks - first);
    const int in = id - band * 8 * a.n_blocks;
    bm = first + in % high;
    bn = in / high;
}

template <int NI, int MI, int WN, int WM, int BK, int BUFS>
__global__ __launch_bounds__(64 * WN * WM, 2) void adapter_product_kernel(
        ProductArgs a) {
    constexpr int BN = 32 * NI * WN, BM = 32 * MI * WM, THREADS = 64 * WN * WM;
    constexpr int CH = BK / 8, STEPS = BK / 16;
    constexpr int SLICE = (BN + BM) * BK;       // one buffer: [W | x] images
    constexpr int PR = 64 / CH;                 // rows a piece of 1 KiB
    constexpr int PIECES = (BN + BM) / PR / (WN * WM);
    static_assert(BUFS == 2 || BUFS == 3, "slices that are waited for");
    typedef TileVec<__bf16>::v8 v8;
    __shared__ __attribute__((aligned(256))) __bf16 smem[BUFS * SLICE];

    const int tid = threadIdx.x, lane = tid & 63;
    const int l31 = lane & 31, hi = lane >> 5;
    const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wn = wid % WN, wm = wid / WN;
    int bm, bn;
    product_place(a, bm, bn);
    const int n0 = bn * BN, m0 = bm * BM;

    // The adapters among the block's rows, found one after another by all
    // waves alike: lane l holds those of rows l, l + 64, .. not yet found.
    int left[(BM + 63) / 64];
    #pragma unroll
    for (int i = 0; i < (BM + 63) / 64; ++i) {
        const int r = i * 64 + lane, row = m0 + r;
        const int v = r < BM && row < a.M
            ? a.ad.row_ids[row / a.ad.rows_per_id] : -1;
        left[i] = v < a.ad.n_adapters ? v : -1;
    }
    const auto next_adapter = [&] {
        int found = -1;
        #pragma unroll
        for (int i = 0; i < (BM + 63) / 64; ++i) {
            const unsigned long long has = __ballot(left[i] >= 0);
            if (found < 0 && has)
                found = __builtin_amdgcn_readlane(left[i],
                                                  __builtin_ctzll(has));
        }
        #pragma unroll
        for (int i = 0; i < (BM + 63) / 64; ++i)
            if (left[i] == found) left[i] = -1;
        return found;
    };
    // this lane's rows
    int id[MI];
    #pragma unroll
    for (int m = 0; m < MI; ++m) {
        const int row = m0 + (wm * MI + m) * 32 + l31;
        id[m] = row < a.M ? a.ad.row_ids[row / a.ad.rows_per_id] : -1;
    }
    int adapter = next_adapter();

    // this wave's pieces of a slice; rows behind the last repeat it and are
    // not stored
    const __bf16* src[PIECES];
    #pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int r = (wid * PIECES + i) * PR + lane / CH;
        const int c = (lane % CH) ^ tile_key<CH>(r);
        src[i] = (r < BN ? a.w + (long)min(n0 + r, a.N - 1) * a.K
                         : a.x + (long)min(m0 + r - BN, a.M - 1) * a.K)
                 + c * 8;
    }
    const int slices = (a.K + BK - 1) / BK;
    // the first adapter's product is staged as one slice more
    const int staged = slices + (adapter >= 0 ? 1 : 0);
    // [up | inner] from column k of the rank; columns behind the rank repeat
    // the last ones and are not used
    const auto stage_adapter = [&](int which, int k, int buf) {
        __bf16* image = smem + buf * SLICE;
        const __bf16* up = a.ad.up + (long)which * a.N * a.ad.rank;
        #pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int r = (wid * PIECES + i) * PR + lane / CH;
            const int c = k + ((lane % CH) ^ tile_key<CH>(r)) * 8;
            const __bf16* from = r < BN
                ? up + (long)min(n0 + r, a.N - 1) * a.ad.rank
                    + min(c, a.ad.rank - 8)
                : a.ad.inner + (long)min(m0 + r - BN, a.M - 1)
                    * a.ad.rank_pad + min(c, a.ad.rank_pad - 8);
            tile_load(from, image + (wid * PIECES + i) * 512);
        }
    };
    const auto fast = [&](int t) {
        return t == slices || (a.vec && (t + 1) * BK <= a.K);
    };
    const auto stage = [&](int t, int buf) {
        __bf16* image = smem + buf * SLICE;
        if (t == slices) {
            stage_adapter(adapter, 0, buf);
        } else if (fast(t)) {
            #pragma unroll
            for (int i = 0; i < PIECES; ++i)
                tile_load(src[i] + t * BK,
                          image + (wid * PIECES + i) * 512);
        } else {
            // the last part of a slice, or rows without alignment
            #pragma unroll 1
            for (int i = 0; i < PIECES; ++i) {
                const int r = (wid * PIECES + i) * PR + lane / CH;
                const int c = (lane % CH) ^ tile_key<CH>(r);
                const __bf16* row = r < BN
                    ? a.w + (long)min(n0 + r, a.N - 1) * a.K
                    : a.x + (long)min(m0 + r - BN, a.M - 1) * a.K;
                *reinterpret_cast<bf16x8*>(
                    image + (wid * PIECES + i) * 512 + lane * 8) =
                    inner_load(row, t * BK + c * 8, a.K, a.vec);
            }
        }
    };

    f32x16 acc[NI][MI] = {};
    v8 fw[2][NI], fx[2][MI];
    const unsigned lds = tile_lds(smem);
    const unsigned base = tile_row_base<CH, 32>(lds, lane);
    const auto read = [&](int buf, int step, int to) {
        const unsigned at = base + buf * SLICE * 2;
        #pragma unroll
        for (int n = 0; n < NI; ++n)
            fw[to][n] = tile_row_read<__bf16, CH, 32>(
                at + wn * NI * 32 * BK * 2, n * 32, step);
        #pragma unroll
        for (int m = 0; m < MI; ++m)
            fx[to][m] = tile_row_read<__bf16, CH, 32>(
                at + (BN + wm * MI * 32) * BK * 2, m * 32, step);
    };
    const auto multiply = [&](int from) {
        #pragma unroll
        for (int n = 0; n < NI; ++n)
            #pragma unroll
            for (int m = 0; m < MI; ++m)
                acc[n][m] = tile_mfma(fw[from][n], fx[from][m], acc[n][m]);
    };
    // Slice t has arrived for this wave, and its reads of the slice before
    // are done; behind the barrier that holds for all waves. LDS-DMA arrives
    // in order, so the pieces of the slice behind it may stay on their way.
    const auto arrive = [&](int t) {
        if (BUFS == 3 && t + 1 < staged && fast(t + 1))
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"i"(PIECES)
                         : "memory");
        else
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };

    #pragma unroll
    for (int t = 0; t < BUFS - 1; ++t)
        if (t < staged) stage(t, t);
    arrive(0);
    if (BUFS - 1 < staged) stage(BUFS - 1, BUFS - 1);
    read(0, 0, 0);
    int buf = 0;
    for (int t = 0; t < slices; ++t) {
        const int next = buf + 1 == BUFS ? 0 : buf + 1;
        #pragma unroll
        for (int step = 0; step < STEPS; ++step) {
            if (step + 1 < STEPS) {
                read(buf, step + 1, (step + 1) & 1);
            } else if (t + 1 < slices) {
                // all operands of slice t are in registers, so its buffer
                // is free once every wave is here
                arrive(t + 1);
                if (t + BUFS < staged) stage(t + BUFS, buf);
                read(next, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
            multiply(step & 1);
            __builtin_amdgcn_sched_barrier(0);
        }
        buf = next;
    }

    // ---- the adapters of the block's rows: slices of [up | inner], the next
    // one on its way while one is used
    for (int k = 0; adapter >= 0;) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const int cur = adapter, k0 = k;
        k += BK;
        if (k >= a.ad.rank) {
            adapter = next_adapter();
            k = 0;
        }
        const int next = buf + 1 == BUFS ? 0 : buf + 1;
        if (adapter >= 0) stage_adapter(adapter, k, next);
        // Other requests' rows take nothing, not even the NaN of their own
        // values times this adapter's: they keep their sums. Selected once a
        // slice, not after each step (12608 rows, 1280 to 5120 columns, rank
        // 64: 281 us by steps, 275 so; with the operands of all steps in
        // registers they no longer fit, 358).
        const int steps = min(STEPS, (a.ad.rank - k0 + 15) / 16);
        const unsigned from = base + buf * SLICE * 2;
        #pragma unroll
        for (int m = 0; m < MI; ++m) {
            if (!__any(id[m] == cur)) continue;
            f32x16 sum[NI];
            #pragma unroll
            for (int n = 0; n < NI; ++n) sum[n] = acc[n][m];
            #pragma unroll 1
            for (int step = 0; step < steps; ++step) {
                const v8 in = tile_row_read<__bf16, CH, 32>(
                    from + (BN + wm * MI * 32) * BK * 2, m * 32, step);
                #pragma unroll
                for (int n = 0; n < NI; ++n) {
                    v8 up = tile_row_read<__bf16, CH, 32>(
                        from + wn * NI * 32 * BK * 2, n * 32, step);
                    if (k0 + step * 16 + hi * 8 >= a.ad.rank) up = v8{};
                    sum[n] = tile_mfma(up, in, sum[n]);
                }
            }
            #pragma unroll
            for (int n = 0; n < NI; ++n)
                #pragma unroll
                for (int i = 0; i < 16; ++i)
                    acc[n][m][i] = id[m] == cur ? sum[n][i] : acc[n][m][i];
        }
        buf = next;
    }

    // ---- bias, activation, residual. The sums change hands through LDS, in
    // as many passes as they need, so that a thread finishes 8 adjacent
    // columns of a row and all accesses to memory are 16 B a lane. Chunk c (4
    // columns) of row r lies at c ^ r: no conflict on either side.
    constexpr int LDS = BUFS * SLICE * 2;
    constexpr int PASSES = (BN * BM * 4 + LDS - 1) / LDS;
    constexpr int MP = MI / PASSES, ROWS = 32 * MP * WM;
    static_assert(MI % PASSES == 0, "whole tiles a pass");
    constexpr int C4 = BN / 4, C8 = BN / 8;
    static_assert(THREADS % C8 == 0, "a thread keeps its columns");
    float* sums = reinterpret_cast<float*>(smem);
    const int c8 = tid % C8, col = n0 + c8 * 8;
    const bool whole = a.N % 8 == 0;
    const int count = whole ? 8 : min(8, a.N - col);
    float bias[8] = {};
    if (a.bias != nullptr && col < a.N) {
        const bf16x8 v = inner_load(a.bias + col, 0, count, whole);
        #pragma unroll
        for (int j = 0; j < 8; ++j) bias[j] = bf2f(v[j]);
    }
    #pragma unroll
    for (int pass = 0; pass < PASSES; ++pass) {
        __syncthreads();
        #pragma unroll
        for (int m = 0; m < MP; ++m) {
            const int r = (wm * MP + m) * 32 + l31;
            #pragma unroll
            for (int n = 0; n < NI; ++n)
                #pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int c = (wn * NI + n) * 8 + g * 2 + hi;
                    const f32x16& v = acc[n][pass * MP + m];
                    *reinterpret_cast<f32x4*>(
                        sums + r * BN + (c ^ (r % 16)) * 4) =
                        f32x4{v[g * 4], v[g * 4 + 1], v[g * 4 + 2],
                              v[g * 4 + 3]};
                }
        }
        __syncthreads();
        #pragma unroll 2
        for (int r = tid / C8; r < ROWS; r += THREADS / C8) {
            const int row = m0 + r / (32 * MP) * 32 * MI + pass * 32 * MP
                            + r % (32 * MP);
            if (row >= a.M || col >= a.N) continue;
            float v[8];
            #pragma unroll
            for (int q = 0; q < 2; ++q)
                *reinterpret_cast<f32x4*>(v + 4 * q) =
                    *reinterpret_cast<const f32x4*>(
                        sums + r * BN + ((2 * c8 + q) ^ (r % 16)) * 4);
            #pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += bias[j];
            finish8(v, a.residual, a.out, (long)row * a.N + col, count,
                    whole, a.act);
        }
    }
}

template <int NI, int MI, int WN, int WM, int BK, int BUFS>
void product_launch(ProductArgs& a) {
    a.n_blocks = (a.N + 32 * NI * WN - 1) / (32 * NI * WN);
    a.m_blocks = (a.M + 32 * MI * WM - 1) / (32 * MI * WM);
    hipLaunchKernelGGL((adapter_product_kernel<NI, MI, WN, WM, BK, BUFS>),
                       dim3(a.n_blocks * a.m_blocks), dim3(64 * WN * WM), 0,
                       pe_current_stream(), a);
}

// The largest tile that still fills most of the 256 CUs: larger tiles read
// less through L2 for each product, but a CU without a block does nothing.
// Measured without adapters, us, tiles in this order (columns by rows):
//   8192 x 1024 -> 2048    41  47  55  59
//   1576 x 1024 -> 4096    36  23  27  27
//   1576 x 768  -> 2304    28  18  13  14
//    512 x 1280 -> 1280    39  25  15  10
void adapter_product(ProductArgs& a) {
    const auto blocks = [&](long columns, long rows) {
        return ((a.N + columns - 1) / columns) * ((a.M + rows - 1) / rows);
    };
    if (blocks(256, 256) >= 200) product_launch<2, 4, 4, 2, 64, 2>(a);
    else if (blocks(256, 128) >= 160) product_launch<2, 2, 4, 2, 64, 3>(a);
    else if (blocks(128, 128) >= 128) product_launch<1, 2, 4, 2, 64, 3>(a);
    else product_launch<1, 1, 2, 2, 64, 2>(a);
}

// Rows that the kernels for few rows take.
constexpr int STEP_ROWS = 64;

template <int NC>
void inner_launch(const InnerArgs& a, dim3 grid) {
    if (a.vec)
        hipLaunchKernelGGL((adapter_inner_kernel<NC, true>), grid, dim3(256),
                           0, pe_current_stream(), a);
    else
        hipLaunchKernelGGL((adapter_inner_kernel<NC, false>), grid, dim3(256),
                           0, pe_current_stream(), a);
}

void adapter_inner(InnerArgs a) {
    const int pads = a.up_padded == nullptr ? 0 : (int)std::min<long>(
        256, (a.up_rows * ((a.rank + 7) / 8) + 1023) / 1024);
    // Up to 512 rows of rank 64, a wave for each row and 4 columns: it reads
    // the row's adapter alone, where the matrix unit takes all adapters of 16
    // rows in turn. Whole projection, 1280 to 1280 columns, rank 64, us with
    // it and without, rows of one adapter and of 8 mixed: 256 rows 14 and 18,
    // 18 and 62; 512 rows 17 and 18, 21 and 63; 1024 rows 23 and 20, 28 and
    // 71; 768 to 768, rank 8, 512 rows: 12 and 11, 15 and 22. The rule is that
    // of rows in order, by item; for rows of many adapters mixed one by one,
    // which it does not tell apart, this kernel would be the better one far
    // beyond 512.
    if ((long)a.M * std::max(a.rank_pad, 64) <= 512 * 64) {
        a.row_blocks = a.M;
        hipLaunchKernelGGL(adapter_inner_step_kernel,
                           dim3(a.M + pads, a.rank_pad / 16), dim3(256), 0,
                           pe_current_stream(), a);
        return;
    }
    // From about 2048 rows of rank 64 on, the way through LDS wins (12608
    // rows of 1280: rank 64 26 us against 10, rank 16 12 against 11; 3152
    // rows: rank 64 10 against 9; 1576 rows of 768, rank 8: 4.5 against 12).
    if ((long)a.M * a.rank_pad >= 2048L * 64 * (a.rank <= 32 ? 2 : 1)) {
        InnerArgs t = a;
        // blocks that end with their item have one adapter and read K once
        t.item_rows = a.rows_per_id >= 64 ? a.rows_per_id : a.M;
        t.item_blocks = (t.item_rows + 63) / 64;
        t.row_blocks = t.item_blocks * (a.M / t.item_rows);
        const int blocks = t.row_blocks + pads;
        if (a.rank <= 32)
            hipLaunchKernelGGL((adapter_inner_tile_kernel<1, 2, 2, 4>),
                               dim3(blocks, 1), dim3(256), 0,
                               pe_current_stream(), t);
        else
            hipLaunchKernelGGL((adapter_inner_tile_kernel<2, 2, 2, 4>),
                               dim3(blocks, a.rank_pad / 64), dim3(512), 0,
                               pe_current_stream(), t);
        return;
    }
    // columns a block: all of them up to 64, then 64 at a time
    a.row_blocks = (a.M + 15) / 16;
    const dim3 grid(a.row_blocks + pads, (a.rank + 63) / 64);
    if (a.rank <= 16) inner_launch<1>(a, grid);
    else if (a.rank <= 32) inner_launch<2>(a, grid);
    else inner_launch<4>(a, grid);
}

template <int NM>
void adapter_step(const ProductArgs& a) {
    hipLaunchKernelGGL((adapter_step_kernel<NM>), dim3((a.N + 15) / 16),
                       dim3(64 * STEP_WAVES), 0, pe_current_stream(), a);
}

torch::Tensor adapter_dense(const torch::Tensor& x) {
    return x.is_contiguous() &&
           reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0
        ? x : x.clone(at::MemoryFormat::Contiguous);
}

}  // namespace

torch::Tensor adapter_linear_op(
        torch::Tensor x, torch::Tensor weight, torch::Tensor down,
        torch::Tensor up, torch::Tensor ids,
        c10::optional<torch::Tensor> bias, int64_t act,
        c10::optional<torch::Tensor> residual,
        c10::optional<torch::Tensor> scales) {
    TORCH_CHECK_VALUE(x.is_cuda(), "adapter_linear: GPU tensors required");
    const c10::DeviceGuard guard(x.device());
    for (const auto* t : {&x, &weight, &down, &up})
        TORCH_CHECK_TYPE(t->scalar_type() == torch::kBFloat16,
                         "adapter_linear: x, weight, down and up must be "
                         "bfloat16");
    for (const auto* t : {&bias, &residual})
        TORCH_CHECK_TYPE(!t->has_value() ||
                         (*t)->scalar_type() == torch::kBFloat16,
                         "adapter_linear: bias and residual must be "
                         "bfloat16");
    TORCH_CHECK_TYPE(ids.scalar_type() == torch::kInt,
                     "adapter_linear: ids must be int32");
    TORCH_CHECK_TYPE(!scales.has_value() ||
                     scales->scalar_type() == torch::kFloat,
                     "adapter_linear: scales must be float32");
    bool one_device = true, grad = false;
    for (const auto* t : {&x, &weight, &down, &up, &ids}) {
        one_device = one_device && t->device() == x.device();
        grad = grad || t->requires_grad();
    }
    for (const auto* t : {&bias, &residual, &scales}) {
        if (!t->has_value()) continue;
        one_device = one_device && (*t)->device() == x.device();
        grad = grad || (*t)->requires_grad();
    }
    TORCH_CHECK_VALUE(one_device,
                      "adapter_linear: tensors on different devices");
    TORCH_CHECK_VALUE(!(grad && at::GradMode::is_enabled()),
                      "adapter_linear: inference only, an input requires a "
                      "gradient");
    TORCH_CHECK_VALUE(x.dim() >= 1 && weight.dim() == 2 && down.dim() == 3 &&
                      up.dim() == 3,
                      "adapter_linear: x must be [.., K], weight [N, K], "
                      "down [n, r, K] and up [n, N, r]");
    const int64_t K = x.size(-1), N = weight.size(0);
    const int64_t n = down.size(0), r = down.size(1);
    TORCH_CHECK_VALUE(weight.size(1) == K && down.size(2) == K &&
                      up.size(0) == n && up.size(1) == N && up.size(2) == r,
                      "adapter_linear: x ", x.sizes(), ", weight ",
                      weight.sizes(), ", down ", down.sizes(), " and up ",
                      up.sizes(), " do not match");
    TORCH_CHECK_VALUE(r <= 256, "adapter_linear: rank above 256");
    const auto lead = x.sizes().slice(0, x.dim() - 1);
    const bool by_row = ids.sizes() == lead;
    const bool by_item = x.dim() >= 2 && ids.dim() == 1 &&
                         ids.size(0) == x.size(0);
    TORCH_CHECK_VALUE(by_row || by_item,
                      "adapter_linear: ids must be one a row or one an item "
                      "of the batch, got ", ids.sizes());
    TORCH_CHECK_VALUE(!bias.has_value() ||
                      (bias->dim() == 1 && bias->size(0) == N),
                      "adapter_linear: bias must be [N]");
    auto out_sizes = x.sizes().vec();
    out_sizes.back() = N;
    TORCH_CHECK_VALUE(!residual.has_value() ||
                      residual->sizes() == torch::IntArrayRef(out_sizes),
                      "adapter_linear: residual must have the output's "
                      "shape");
    TORCH_CHECK_VALUE(!scales.has_value() ||
                      (scales->dim() == 1 && scales->size(0) == n),
                      "adapter_linear: scales must be [n]");
    TORCH_CHECK_VALUE(act >= ACT_NONE && act <= ACT_TANH,
                      "adapter_linear: unknown activation");
    int64_t M = 1;
    for (const auto s : lead) M *= s;
    TORCH_CHECK_VALUE(K > 0 && K < (1L << 31) && M < (1L << 31) &&
                      N < (1L << 31),
                      "adapter_linear: no inner columns, or too many rows");
    if (M == 0 || N == 0)
        return torch::empty(out_sizes, x.options());
    const int rank_pad = r <= 32 ? 32 : (r + 63) / 64 * 64;
    const bool any = n > 0 && r > 0;
    // A launch has less than 2^32 threads: of the inner values a block for 64
    // rows of a request, and those that pad; of few rows one for 16 columns.
    const int64_t per = by_row ? 1 : M / x.size(0);
    const int64_t tiles = per >= 64 ? (per + 63) / 64 * (M / per)
                                    : (M + 63) / 64;
    TORCH_CHECK_VALUE(
        (!any || (tiles + 256) * (r <= 32 ? 256 : 512) < (1L << 32)) &&
        (M > STEP_ROWS || (N + 15) / 16 * 64 * STEP_WAVES < (1L << 32)),
        "adapter_linear: too many rows or columns");

    const auto x2d = adapter_dense(x.reshape({M, K}));
    const auto w = adapter_dense(weight);
    const auto down_c = adapter_dense(down);
    // The products of many rows read up 8 of the rank at a time. Ranks between
    // are padded, by the kernel of the inner values: loads of single elements
    // by each block of the product cost more (12608 rows, 1280 to 5120
    // columns, rank 60: 253 us padded, 318 so), two launches more as well
    // (1000 rows, 320 to 700, rank 4: 18 us, 11 so).
    const auto up_c = adapter_dense(up);
    const bool pad_up = M > STEP_ROWS && n > 0 && r % 8 != 0;
    const int64_t up_rank = pad_up ? (r + 7) / 8 * 8 : r;
    auto up_padded = torch::empty({pad_up ? n : 0, N, up_rank}, x.options());
    const auto ids_c = ids.contiguous();
    const auto tensor_or_none = [](c10::optional<torch::Tensor>& t) {
        if (!t.has_value()) return (const __bf16*)nullptr;
        t = adapter_dense(*t);
        return reinterpret_cast<const __bf16*>(t->data_ptr());
    };
    auto inner = torch::empty({any ? M : 0, rank_pad}, x.options());
    auto out = torch::empty(out_sizes, x.options());
    ProductArgs a = {};
    a.x = reinterpret_cast<const __bf16*>(x2d.data_ptr());
    a.w = reinterpret_cast<const __bf16*>(w.data_ptr());
    a.bias = tensor_or_none(bias);
    a.residual = tensor_or_none(residual);
    a.out = reinterpret_cast<__bf16*>(out.data_ptr());
    a.M = M, a.N = N, a.K = K, a.act = act;
    a.vec = K % 8 == 0;
    a.ad.inner = reinterpret_cast<const __bf16*>(inner.data_ptr());
    a.ad.up = reinterpret_cast<const __bf16*>(
        pad_up ? up_padded.data_ptr() : up_c.data_ptr());
    a.ad.row_ids = ids_c.data_ptr<int>();
    a.ad.rows_per_id = per;
    a.ad.n_adapters = any ? n : 0;      // without any, no id is inside
    a.ad.rank = up_rank, a.ad.rank_pad = rank_pad;
    if (any) {
        InnerArgs in = {};
        in.x = a.x;
        in.down = reinterpret_cast<const __bf16*>(down_c.data_ptr());
        in.row_ids = a.ad.row_ids;
        torch::Tensor scales_c;
        if (scales.has_value()) {
            scales_c = scales->contiguous();
            in.scales = scales_c.data_ptr<float>();
        }
        in.inner = reinterpret_cast<__bf16*>(inner.data_ptr());
        in.M = M, in.K = K, in.n_adapters = n, in.rank = r;
        in.rows_per_id = a.ad.rows_per_id;
        in.rank_pad = rank_pad;
        in.vec = a.vec;
        in.up = reinterpret_cast<const __bf16*>(up_c.data_ptr());
        if (pad_up)
            in.up_padded = reinterpret_cast<__bf16*>(up_padded.data_ptr());
        in.up_rows = n * N;
        adapter_inner(in);
        HIP_CHECK_LAST();
    }
    if (M <= 16) adapter_step<1>(a);
    else if (M <= 32) adapter_step<2>(a);
    else if (M <= STEP_ROWS) adapter_step<4>(a);
    else adapter_product(a);
    HIP_CHECK_LAST();
    return out;
}
