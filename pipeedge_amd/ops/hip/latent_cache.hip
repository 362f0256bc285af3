// Latent attention, absorbed form: the projections to keys and values are
// moved to the query and output side, so every head attends to the cached
// vectors themselves, whose first R columns are also the values:
//   out[i, h] = softmax_t(scale * q[i, h] . cache[t]) cache[t][:R]
// The rows of a product are (query, head) pairs, all of one sequence, so one
// pass over the cache serves all heads; 16 heads are bound by memory, 128 by
// the matrix cores.
//
// Work is cut into tiles of 64 cached tokens, numbered through all sequences,
// and a fixed number of runs takes an equal share of them, across sequences
// where it falls so: lengths stay on the device, and ragged batches are
// balanced to within a tile. A run has a block for each group of rows; they
// are neighbours on one XCD and walk over the same tiles at the same time, so
// that one of them fetches a tile from memory and the others find it in L2.
// A run's part of one sequence is a segment; a segment that covers all tiles
// is written to the output, others leave partial sums in fp32 that a second
// kernel joins in a fixed order.
//
// Both products are transposed as in the expanded form, on 16x16x32 MFMAs: a
// wave owns 16 rows, a lane holds one row's scores, and the weights are the
// second operand as they are. One LDS image of a tile serves both products,
// read by rows for the scores and by columns, through the transposing reads,
// for the values. The accumulators take R / 4 registers and the query
// operands (R + DR) / 8. A block has up to 64 rows, one or two waves a SIMD,
// and its waves share the tokens of a tile; where two waves have the same
// rows, they take 32 tokens of a tile each and join their sums at the
// segment's end. Up to 16 rows a wave loads its own tokens, two tiles ahead,
// and waits for nobody else. 16 heads are bound by memory (64 ragged sequences
// up to 4096, 165 MB: 35 us, 4.7 TB/s, and 5 us to join), 128 heads by the
// instructions around the MFMAs and by the LDS, each fragment read from it
// feeding one MFMA (2 queries of 16 sequences of 4096 to 8192 tokens, fp16: 84
// us, 660 TFLOP/s, and 12 us to join). Two waves a SIMD with 512 columns are 15
// registers short, which go to scratch memory, outside the loop over the
// tiles.
#include <torch/extension.h>

#include <cmath>

#include <c10/core/DeviceGuard.h>

#include "mfma_tiles.h"

namespace {

struct CacheArgs {
    const void* q;                  // [B, Sq, H, R + DR]
    const void* cache;              // [pages, page size, R + DR]
    const int* table;               // [B, table_width]
    const int* lengths;             // [B]
    void* out;                      // [B, Sq, H, R]
    float* part;                    // partial sums, 16 rows by R a slot
    float2* part_stat;              // [slots][16] reference, total
    long q_b, q_s, q_h, c_p, c_t, t_b;      // strides in elements
    long pages;
    int page_size, page_shift;      // shift -1: not a power of two
    int B, H, Sq, table_width;
    int rows;                       // Sq * H
    int row_groups;                 // ceil(rows / rows a block)
    int runs, least;                // most runs, fewest tiles of one
    int tile_shift;                 // tokens a tile: 32 or 64
    float scale;                    // times log2(e)
};

// The tables are constant while the kernel runs, and read through the scalar
// cache where all lanes want the same entry: a vector load would have to wait
// for every LDS-DMA piece that is on its way before it.
typedef const __attribute__((address_space(4))) int* const_ints;
__device__ __forceinline__ const_ints as_constant(const int* p) {
    return (const_ints)(uintptr_t)p;
}

// Tiles of a sequence. A length that the table cannot hold counts as what it
// can hold; its outputs are NaN.
__device__ __forceinline__ int cache_length(const CacheArgs& a, int b) {
    const long most = (long)a.table_width * a.page_size;
    return (int)min((long)max(as_constant(a.lengths)[b], 0), most);
}
__device__ __forceinline__ int cache_tiles(const CacheArgs& a, int b) {
    return b < a.B
        ? (cache_length(a, b) + (1 << a.tile_shift) - 1) >> a.tile_shift : 0;
}

__device__ __forceinline__ int wave_scan(int v, int lane) {
    #pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int up = __shfl_up(v, d);
        if (lane >= d) v += up;
    }
    return v;
}

__device__ __forceinline__ int cache_total(const CacheArgs& a, int lane) {
    int total = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64)
        total += __builtin_amdgcn_readlane(
            wave_scan(cache_tiles(a, b0 + lane), lane), 63);
    return total;
}

// Place of tile number `at`: the sequence and the number of its first tile.
__device__ __forceinline__ void cache_find(const CacheArgs& a, int at,
                                           int lane, int& seq, int& first) {
    int before = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        const int mine = cache_tiles(a, b0 + lane);
        const int upto = wave_scan(mine, lane);
        const int end = before + upto;
        const unsigned long long past = __ballot(end > at);
        if (past) {
            const int l = __builtin_ctzll(past);
            seq = b0 + l;
            first = before + __builtin_amdgcn_readlane(upto, l)
                    - __builtin_amdgcn_readlane(mine, l);
            return;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    seq = a.B;
    first = before;
}

// No more runs than a.least tiles each are worth: a run's start, its partial
// sums and their way through memory cost about as much as a.least tiles.
__device__ __forceinline__ int run_count(const CacheArgs& a, int total) {
    return min(a.runs, max(1, total / a.least));
}
// tiles of run g: run_start(g) .. run_start(g + 1)
__device__ __forceinline__ int run_start(int total, int g, int runs) {
    return total / runs * g + min(g, total % runs);
}
// the run that has tile `at`
__device__ __forceinline__ int run_of(int total, int at, int runs) {
    const int each = total / runs, extra = total % runs;
    if (at < extra * (each + 1)) return at / (each + 1);
    return extra + (at - extra * (each + 1)) / each;
}

// The accumulators take one half of the register file. Arithmetic on them in
// a rare branch would make the compiler carry them in the other half and copy
// them back and forth in every tile.
__device__ __forceinline__ void keep_in_agprs(f32x4& v) {
    asm volatile("" : "+a"(v));
}

// Where the 8 tokens of one group lie: the address of the first, and the
// number of the last that holds one (tokens behind the last of the sequence
// are read as the last one, so that no padding reaches a product).
struct CacheGroup {
    const char* at;
    int last;
};

// WR groups of 16 rows times WT waves a group, each with its 32 tokens of a
// tile.
// GROUPED: pages hold whole groups of 8 tokens.
template <typename T, int R, int DR, int WR, int WT, bool GROUPED>
__global__ __launch_bounds__(64 * WR * WT, WR * WT > 4 ? 2 : 1)
void latent_cache_kernel(CacheArgs a) {
    // one wave on a SIMD has 512 registers, one of two has 256
    constexpr bool ONE = WR * WT <= 4;
    constexpr int AHEAD = ONE ? 8 : 2;
    constexpr int CL = R / 8, CR = DR / 8;      // chunks of a row's parts
    constexpr int NT = R / 16;                  // output tiles
    constexpr int TOKENS = 32, KEYS = TOKENS * WT;  // a wave's, a tile's
    constexpr int SUB = TOKENS / 16;            // score columns
    constexpr int GROUPS = TOKENS / 8 / WR;     // 8 tokens each, to load
    constexpr int TILE = TOKENS * (R + DR);
    // the waves of one row group load and use their tokens alone
    constexpr bool ALONE = WR == 1;
    // Buffers of a share, and how many tiles its loads run ahead: where waves
    // share tiles, behind the barrier that ends a buffer's use; a wave alone
    // loads after its own use of the buffer.
    constexpr int BUFS = WT == 1 ? 4 : 2, LEAD = ALONE ? 2 : BUFS - 1;
    constexpr int PIECES = GROUPS * CL / 8 + (GROUPS * CR + 7) / 8;
    static_assert(!ALONE || (GROUPS == 4 && PIECES < 64), "counted waits");
    typedef typename TileVec<T>::v8 v8;
    typedef RunningTop<T> softmax;
    // buffers of [latent | rope] images
    __shared__ __attribute__((aligned(256))) T smem[WT * BUFS * TILE];

    const int tid = threadIdx.x;
    const int lane = tid & 63, l15 = lane & 15, quad = lane >> 4;
    const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int group = wid % WR, share = wid / WR;
    T* const images = smem + share * BUFS * TILE;
    const unsigned lds = tile_lds(images);

    int total, seq, first;
    const int block = xcd_contiguous(blockIdx.x, gridDim.x);
    const int run = block / a.row_groups, rg = block - run * a.row_groups;
    int at, end;
    if (a.B <= 64) {
        // all sequences in one wave's lanes: their tiles are added up once
        const int mine = cache_tiles(a, lane);
        const int upto = wave_scan(mine, lane);
        total = __builtin_amdgcn_readlane(upto, 63);
        const int runs = run_count(a, total);
        at = run_start(total, run, runs);
        end = run_start(total, run + 1, runs);
        if (run >= runs || at >= end) return;
        seq = __builtin_ctzll(__ballot(upto > at));
        first = __builtin_amdgcn_readlane(upto - mine, seq);
    } else {
        total = cache_total(a, lane);
        const int runs = run_count(a, total);
        at = run_start(total, run, runs);
        end = run_start(total, run + 1, runs);
        if (run >= runs || at >= end) return;
        cache_find(a, at, lane, seq, first);
    }

    while (at < end) {
        const int len = cache_length(a, seq);
        const int tiles = (len + KEYS - 1) / KEYS;
        if (tiles == 0) { ++seq; continue; }
        const int t0 = at - first;
        const int t1 = min(tiles, end - first);

        // this lane's row and the last token that it sees
        const int row = (rg * WR + group) * 16 + l15;
        const bool live = (rg * WR + group) * 16 < a.rows;
        const int rowc = min(row, a.rows - 1);
        const int qi = rowc / a.H, h = rowc - qi * a.H;
        const int limit = len - a.Sq + qi;
        v8 bq[(R + DR) / 32];
        {
            const T* p = reinterpret_cast<const T*>(a.q) + seq * a.q_b
                         + qi * a.q_s + h * a.q_h + quad * 8;
            #pragma unroll
            for (int i = 0; i < (R + DR) / 32; ++i)
                bq[i] = *reinterpret_cast<const v8*>(p + i * 32);
        }

        // A page number that the cache does not have reads page 0 and
        // spoils the output, as does a length that the table cannot hold.
        bool bad = as_constant(a.lengths)[seq] > len;
        const const_ints table = as_constant(a.table + seq * a.t_b);
        const auto page_at = [&](int slot) {
            int page = table[slot];
            if (page < 0 || page >= a.pages) { bad = true; page = 0; }
            return reinterpret_cast<const char*>(a.cache) + page * a.c_p * 2;
        };
        const int step = (int)a.c_t * 2;        // bytes from token to token
        const auto locate = [&](int t) {
            const int tok = min(t * KEYS + share * TOKENS
                                + group * GROUPS * 8 + lane % (GROUPS * 8),
                                len - 1);
            const int slot = tok / a.page_size;
            int page = a.table[seq * a.t_b + slot];
            if (page < 0 || page >= a.pages) { bad = true; page = 0; }
            return page * a.c_p * 2
                   + (long)(tok - slot * a.page_size) * a.c_t * 2;
        };
        // The pieces of a tile that this wave loads: LP of the latent part,
        // PR rows each, and RP of the rotary part, RR rows each.
        constexpr int PR = 64 / CL, RR = 64 / CR;
        constexpr int LP = GROUPS * 8 / PR, RP = (GROUPS * 8 + RR - 1) / RR;
        // Groups of 8 tokens that never straddle a page have places that are
        // the same for all lanes and live in scalar registers. For any other
        // page size lane l has the place of token l, found one tile earlier.
        CacheGroup from[GROUPS];
        long place = 0, ahead = GROUPED ? 0 : locate(t0);
        const auto find = [&](int t) {
            if constexpr (GROUPED) {
                const int tok0 = t * KEYS + share * TOKENS
                                 + group * GROUPS * 8;
                #pragma unroll
                for (int g = 0; g < GROUPS; ++g) {
                    // behind the end, the last group once more
                    const int tok = min(tok0 + g * 8, (len - 1) & ~7);
                    const int slot = a.page_shift >= 0 ? tok >> a.page_shift
                                                       : tok / a.page_size;
                    from[g].at = page_at(slot)
                        + (long)(tok - slot * a.page_size) * a.c_t * 2;
                    from[g].last = len - 1 - tok;
                }
            } else {
                place = ahead;
                if (t + 1 < t1) ahead = locate(t + 1);
            }
        };
        const auto load = [&](int p, int buf) {
            // (recomputed for every piece: kept, they would cost registers)
            unsigned l = lane;
            asm volatile("" : "+v"(l));
            const bool rotary = p >= LP;
            const int q = rotary ? p - LP : p;
            const int row0 = q * (rotary ? RR : PR);
            T* to = images + buf * TILE + (rotary ? TOKENS * R : 0)
                    + (group * GROUPS * 8 + row0) * (rotary ? DR : R);
            const int r = row0 + (int)(rotary ? l / CR
                                              : PR == 1 ? 0 : l / CL);
            const int key = group * GROUPS * 8 + r;
            const unsigned chunk = rotary
                ? R * 2 + ((l % CR) ^ tile_key<CR>(key)) * 16
                : ((l % CL) ^ tile_key<CL>(key)) * 16;
            // half a wave loads the rotary part of one group of 32 columns
            if (rotary && GROUPS * 8 < RR && l >= 32) return;
            if constexpr (GROUPED) {
                CacheGroup f = from[row0 / 8];
                if (rotary && RR == 16 && GROUPS > 1 && l >= 32)
                    f = from[(row0 / 8 + 1) % GROUPS];
                if (!rotary && PR == 1)
                    tile_load(f.at + (long)(min(r % 8, f.last) * step),
                              chunk, to);
                else
                    tile_load(f.at + (unsigned)(min(r % 8, f.last) * step
                                                + chunk), to);
            } else {
                tile_load(reinterpret_cast<const char*>(a.cache)
                          + __shfl(place, r) + chunk, to);
            }
        };

        f32x4 acc[NT] = {};
        float top = -INFINITY, sub = 0.0f, sum = 0.0f;
        // every wave is done with the LDS of the segment before
        __syncthreads();
        const auto load_all = [&](int t) {
            if constexpr (ALONE) find(t);
            #pragma unroll
            for (int p = 0; p < PIECES; ++p) load(p, t & (BUFS - 1));
        };
        if constexpr (!ALONE)
            #pragma unroll 1
            for (int t = t0; t < min(t0 + LEAD, t1); ++t) {
                find(t);
                load_all(t);
            }
        #pragma unroll
        for (int i = 0; i < (R + DR) / 32; ++i) tile_settle(bq[i]);
        // Turn t uses tile t and loads tile t + LEAD; the first turns of a
        // wave alone only load. LDS-DMA arrives in order, so the pieces of
        // later tiles may stay on their way.
        for (int t = ALONE ? t0 - LEAD : t0; t < t1; ++t) {
            const bool more = t + LEAD < t1;
            const int later = min(t1 - 1 - t, ALONE ? 1 : LEAD - 1);
            if (!ALONE || t >= t0) {
            if (later == 2)
                asm volatile("s_waitcnt vmcnt(%0)" ::"i"(2 * PIECES)
                             : "memory");
            else if (later == 1)
                asm volatile("s_waitcnt vmcnt(%0)" ::"i"(PIECES) : "memory");
            else
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            }
            if constexpr (!ALONE) {
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                if (more) find(t + LEAD);
            }
            if (live && (!ALONE || t >= t0)) {
            const unsigned image = lds + (t & (BUFS - 1)) * TILE * 2;
            const unsigned latent = tile_row_base<CL, 16>(image, lane);
            const unsigned rope = tile_row_base<CR, 16>(
                image + TOKENS * R * 2, lane);
            const unsigned value = tile_column_base<CL, 16>(image, lane);
            const int tok0 = t * KEYS + share * TOKENS;

            // Operands are read from LDS a batch ahead of their MFMAs: one
            // wave on a SIMD has nothing else to wait with.
            f32x4 s[SUB] = {};
            v8 f[2][AHEAD];
            const auto key = [&](int j) {
                const int i = j / SUB, m = j % SUB;
                return i < R / 32
                    ? tile_row_read<T, CL, 16>(latent, m * 16, i)
                    : tile_row_read<T, CR, 16>(rope, m * 16, i - R / 32);
            };
            const auto val = [&](int j) {
                return tile_column_read<T, CL, 16>(value, j / NT * 32,
                                                   j % NT);
            };
            constexpr int KF = SUB * (R + DR) / 32, VF = SUB / 2 * NT;
            constexpr int KB = (KF + AHEAD - 1) / AHEAD;
            constexpr int VB = VF / AHEAD;
            static_assert(VF % AHEAD == 0, "whole batches");
            #pragma unroll
            for (int j = 0; j < AHEAD; ++j) f[0][j] = key(j);
            // A wave that issues a load waits until the ones before it, also
            // those of other waves, are accepted, about 24 cycles for 1 KiB:
            // they go out one by one between the batches of both products.
            constexpr int EACH = (PIECES + KB + VB - 1) / (KB + VB);
            const auto load_between = [&](int b) {
                if (!ALONE && more)
                    #pragma unroll
                    for (int p = b * EACH; p < (b + 1) * EACH; ++p)
                        if (p < PIECES) load(p, (t + LEAD) & (BUFS - 1));
            };
            #pragma unroll
            for (int b = 0; b < KB; ++b) {
                load_between(b);
                #pragma unroll
                for (int j = 0; j < AHEAD; ++j) {
                    const int k = b * AHEAD + j;
                    if (k + AHEAD < KF)
                        f[(b + 1) & 1][j] = key(k + AHEAD);
                    if (k < KF)
                        s[k % SUB] = tile_mfma(f[b & 1][j], bq[k / SUB],
                                               s[k % SUB]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            // the first values, while the weights are formed
            #pragma unroll
            for (int j = 0; j < AHEAD; ++j) f[0][j] = val(j);
            __builtin_amdgcn_sched_barrier(0);

            if (__any(limit < tok0 + TOKENS - 1)) {
                #pragma unroll
                for (int m = 0; m < SUB; ++m)
                    #pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (tok0 + m * 16 + quad * 4 + i > limit)
                            s[m][i] = -INFINITY;
            }
            float peak = -INFINITY;
            #pragma unroll
            for (int m = 0; m < SUB; ++m)
                #pragma unroll
                for (int i = 0; i < 4; ++i) peak = fmaxf(peak, s[m][i]);
            peak = fmaxf(peak, __shfl_xor(peak, 16));
            peak = fmaxf(peak, __shfl_xor(peak, 32)) * a.scale;
            if (__any(peak > top + softmax::SLACK)) {
                const float next = fmaxf(top, peak);
                const float turn = top == -INFINITY
                    ? 0.0f : __builtin_amdgcn_exp2f(top - next);
                top = next;
                sub = next == -INFINITY ? 0.0f : next - softmax::BIAS;
                sum *= turn;
                #pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if constexpr (ONE) keep_in_agprs(acc[n]);
                    acc[n] *= turn;
                    if constexpr (ONE) keep_in_agprs(acc[n]);
                }
            }
            #pragma unroll
            for (int m = 0; m < SUB; ++m)
                #pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[m][i] = __builtin_amdgcn_exp2f(
                        fmaf(s[m][i], a.scale, -sub));
                    sum += s[m][i];
                }
            v8 w[SUB / 2];
            #pragma unroll
            for (int m = 0; m < SUB; m += 2) {
                float p[8];
                #pragma unroll
                for (int j = 0; j < 8; ++j) p[j] = s[m + j / 4][j % 4];
                w[m / 2] = tile_weights<T>(p);
            }
            #pragma unroll
            for (int b = 0; b < VB; ++b) {
                load_between(KB + b);
                #pragma unroll
                for (int j = 0; j < AHEAD; ++j) {
                    const int k = b * AHEAD + j;
                    if (b + 1 < VB) f[(b + 1) & 1][j] = val(k + AHEAD);
                    acc[k % NT] = tile_mfma(f[b & 1][j], w[k / NT],
                                            acc[k % NT]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            }
            // a wave alone is done with the buffer only now; one without rows
            // does its part of the loads
            if (more && (ALONE || !live)) load_all(t + LEAD);
        }
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        // whichever wave loaded from the bad page
        if (__syncthreads_or(bad)) sum = NAN;

        if constexpr (WT == 2) {
            // the second wave of a group hands its sums to the first; the
            // barrier above ended all use of the tiles
            constexpr int STEP = 64 * WR;
            f32x4* give = reinterpret_cast<f32x4*>(smem) + group * 64 + lane;
            float2* stat = reinterpret_cast<float2*>(
                reinterpret_cast<f32x4*>(smem) + NT * STEP)
                + group * 64 + lane;
            static_assert(NT * STEP * 16 + STEP * 8 <= WT * BUFS * TILE * 2,
                          "the sums must fit in the tiles' LDS");
            if (share == 1) {
                #pragma unroll
                for (int n = 0; n < NT; ++n) give[n * STEP] = acc[n];
                *stat = make_float2(top, sum);
            }
            __syncthreads();
            if (share == 0) {
                const float2 other = *stat;
                const float next = fmaxf(top, other.x);
                // a share that saw no token has nothing to give
                const float f1 = top == -INFINITY
                    ? 0.0f : __builtin_amdgcn_exp2f(top - next);
                const float f2 = other.x == -INFINITY
                    ? 0.0f : __builtin_amdgcn_exp2f(other.x - next);
                top = next;
                sum = (sum == sum ? sum * f1 : sum)
                      + (other.y == other.y ? other.y * f2 : other.y);
                #pragma unroll
                for (int n = 0; n < NT; n += 4) {
                    f32x4 taken[4];
                    #pragma unroll
                    for (int j = 0; j < 4; ++j)
                        taken[j] = give[(n + j) * STEP];
                    __builtin_amdgcn_sched_barrier(0);
                    #pragma unroll
                    for (int j = 0; j < 4; ++j)
                        acc[n + j] = acc[n + j] * f1 + taken[j] * f2;
                }
            }
        }

        const bool whole = t0 == 0 && t1 == tiles;
        if (share == 0 && live) {
            if (whole && row < a.rows) {
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                T* out = reinterpret_cast<T*>(a.out)
                         + ((long)seq * a.rows + row) * R + quad * 4;
                #pragma unroll
                for (int n = 0; n < NT; ++n) {
                    // a row that sees nothing is zero, also where its zero
                    // weights met values that are not finite
                    typename TileVec<T>::v4 o;
                    #pragma unroll
                    for (int j = 0; j < 4; ++j)
                        o[j] = (T)(sum == 0.0f ? 0.0f : acc[n][j] * inv);
                    *reinterpret_cast<typename TileVec<T>::v4*>(
                        out + n * 16) = o;
                }
            } else if (!whole) {
                // Two slots a run: only its first segment can begin inside
                // a sequence, and of those that do not, only its last can
                // end inside one (a group of 16 rows as the lanes hold it).
                const long slot = ((long)(2 * run + (t0 == 0)) * a.row_groups
                                   + rg) * WR + group;
                f32x4* out = reinterpret_cast<f32x4*>(a.part)
                             + slot * NT * 64 + lane;
                #pragma unroll
                for (int n = 0; n < NT; ++n) out[n * 64] = acc[n];
                if (quad == 0)
                    a.part_stat[slot * 16 + l15] = make_float2(top, sum);
            }
        }
        at = first + t1;
        if (t1 == tiles) {
            first += tiles;
            ++seq;
        }
    }
}

// Joins the segments of 16 rows: out = sum 2^(top_i - top) part_i / sum
// 2^(top_i - top) sum_i. A block takes four pieces of 16 columns, its four
// waves every fourth run each, in their order, and the four meet in LDS in
// theirs. Sequences that hold nothing get zeros; whole segments are there
// already. Bound by the latency of its reads: 32 segments of a sequence are
// two rounds of loads.
template <typename T, int R>
__global__ __launch_bounds__(256) void latent_cache_join_kernel(
        CacheArgs a, int groups) {
    constexpr int NT = R / 16, PIECES = 4;
    __shared__ f32x4 sums[4][PIECES][64];
    __shared__ float2 stats[4][16];
    const int lane = threadIdx.x & 63, l15 = lane & 15, quad = lane >> 4;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int group = blockIdx.x, n0 = blockIdx.y * PIECES;
    const int seq = blockIdx.z;
    const int row = group * 16 + l15;
    // a wave writes one piece
    T* out = reinterpret_cast<T*>(a.out) + ((long)seq * a.rows + row) * R
             + (n0 + wid) * 16 + quad * 4;
    typedef typename TileVec<T>::v4 v4;
    const int tiles = cache_tiles(a, seq);
    if (tiles == 0) {
        if (row < a.rows) *reinterpret_cast<v4*>(out) = v4{};
        return;
    }
    int total = 0, first = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        const int mine = cache_tiles(a, b0 + lane);
        const int upto = wave_scan(mine, lane);
        if (seq >= b0 && seq < b0 + 64)
            first = total + __builtin_amdgcn_readlane(upto, seq - b0) - tiles;
        total += __builtin_amdgcn_readlane(upto, 63);
    }
    const int runs = run_count(a, total);
    const int g0 = run_of(total, first, runs);
    const int g1 = run_of(total, first + tiles - 1, runs);
    if (g0 == g1) return;
    // the first run begins the sequence, the others are inside it
    const auto slot_of = [&](int run) {
        return (long)(2 * run + (run == g0)) * groups + group;
    };
    float top = -INFINITY, sum = 0.0f;
    f32x4 acc[PIECES] = {};
    constexpr int BATCH = 4;
    for (int h = g0 + wid; h <= g1; h += 4 * BATCH) {
        float2 st[BATCH];
        f32x4 part[BATCH][PIECES];
        #pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            // behind the last, the last once more, without weight
            const long slot = slot_of(min(h + 4 * i, g1));
            st[i] = a.part_stat[slot * 16 + l15];
            #pragma unroll
            for (int n = 0; n < PIECES; ++n)
                part[i][n] = reinterpret_cast<const f32x4*>(a.part)[
                    (slot * NT + n0 + n) * 64 + lane];
        }
        __builtin_amdgcn_sched_barrier(0);
        #pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            if (h + 4 * i > g1) break;
            const float next = fmaxf(top, st[i].x);
            const float f0 = top == -INFINITY
                ? 0.0f : __builtin_amdgcn_exp2f(top - next);
            const float f1 = st[i].x == -INFINITY
                ? 0.0f : __builtin_amdgcn_exp2f(st[i].x - next);
            top = next;
            // a total that is not a number stays one
            sum = sum == sum ? sum * f0 : sum;
            sum += st[i].y == st[i].y ? st[i].y * f1 : st[i].y;
            #pragma unroll
            for (int n = 0; n < PIECES; ++n)
                acc[n] = acc[n] * f0 + part[i][n] * f1;
        }
    }
    #pragma unroll
    for (int n = 0; n < PIECES; ++n) sums[wid][n][lane] = acc[n];
    if (quad == 0) stats[wid][l15] = make_float2(top, sum);
    __syncthreads();
    top = -INFINITY;
    #pragma unroll
    for (int w = 0; w < 4; ++w) top = fmaxf(top, stats[w][l15].x);
    sum = 0.0f;
    f32x4 all = {};
    #pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float2 st = stats[w][l15];
        const float f = st.x == -INFINITY
            ? 0.0f : __builtin_amdgcn_exp2f(st.x - top);
        sum += st.y == st.y ? st.y * f : st.y;
        all += sums[w][wid][lane] * f;
    }
    if (row >= a.rows) return;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    v4 o;
    #pragma unroll
    for (int j = 0; j < 4; ++j)
        o[j] = (T)(sum == 0.0f ? 0.0f : all[j] * inv);
    *reinterpret_cast<v4*>(out) = o;
}

bool cache_rows_ok(const torch::Tensor& x) {
    bool ok = reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0 &&
              x.stride(-1) == 1;
    for (int64_t d = 0; d + 1 < x.dim(); ++d)
        ok = ok && (x.size(d) == 1 || x.stride(d) % 8 == 0);
    return ok;
}

template <typename T, int R, int DR, int WR, int WT>
void cache_launch_shape(const CacheArgs& a, int blocks) {
    if (a.page_size % 8 == 0)
        hipLaunchKernelGGL((latent_cache_kernel<T, R, DR, WR, WT, true>),
                           dim3(blocks), dim3(64 * WR * WT), 0,
                           pe_current_stream(), a);
    else
        hipLaunchKernelGGL((latent_cache_kernel<T, R, DR, WR, WT, false>),
                           dim3(blocks), dim3(64 * WR * WT), 0,
                           pe_current_stream(), a);
    hipLaunchKernelGGL((latent_cache_join_kernel<T, R>),
                       dim3((a.rows + 15) / 16, R / 64, a.B), dim3(256), 0,
                       pe_current_stream(), a, a.row_groups * WR);
}

template <typename T, int R, int DR>
void cache_launch(const CacheArgs& a, int block_rows, int blocks) {
    if (block_rows == 64 && a.tile_shift == 6)
        cache_launch_shape<T, R, DR, 4, 2>(a, blocks);
    else if (block_rows == 64)
        cache_launch_shape<T, R, DR, 4, 1>(a, blocks);
    else if (block_rows == 32) cache_launch_shape<T, R, DR, 2, 2>(a, blocks);
    else cache_launch_shape<T, R, DR, 1, 2>(a, blocks);
}

template <typename T>
void cache_dispatch(const CacheArgs& a, int latent, int rope, int block_rows,
                    int blocks) {
    if (latent == 512 && rope == 64)
        cache_launch<T, 512, 64>(a, block_rows, blocks);
    else if (latent == 512)
        cache_launch<T, 512, 32>(a, block_rows, blocks);
    else if (rope == 64)
        cache_launch<T, 256, 64>(a, block_rows, blocks);
    else
        cache_launch<T, 256, 32>(a, block_rows, blocks);
}

}  // namespace

torch::Tensor latent_cache_attention_op(
        torch::Tensor q, torch::Tensor cache, torch::Tensor block_table,
        torch::Tensor lengths, int64_t latent_dim, double scale) {
    TORCH_CHECK_VALUE(q.is_cuda(),
                      "latent_cache_attention: GPU tensors required");
    const c10::DeviceGuard guard(q.device());
    const auto dtype = q.scalar_type();
    TORCH_CHECK_TYPE((dtype == torch::kBFloat16 || dtype == torch::kHalf) &&
                     cache.scalar_type() == dtype,
                     "latent_cache_attention: q and cache must be both "
                     "bfloat16 or both float16");
    TORCH_CHECK_TYPE(block_table.scalar_type() == torch::kInt &&
                     lengths.scalar_type() == torch::kInt,
                     "latent_cache_attention: block_table and lengths must "
                     "be int32");
    TORCH_CHECK_VALUE(cache.device() == q.device() &&
                      block_table.device() == q.device() &&
                      lengths.device() == q.device(),
                      "latent_cache_attention: tensors on different devices");
    TORCH_CHECK_VALUE(!(at::GradMode::is_enabled() &&
                        (q.requires_grad() || cache.requires_grad())),
                      "latent_cache_attention: inference only, an input "
                      "requires a gradient");
    TORCH_CHECK_VALUE(q.dim() == 4 && cache.dim() == 3 &&
                      q.size(3) == cache.size(2),
                      "latent_cache_attention: q must be [B, Sq, H, D] and "
                      "cache [pages, page size, D], got ", q.sizes(), " and ",
                      cache.sizes());
    const int64_t B = q.size(0), Sq = q.size(1), H = q.size(2);
    const int64_t rope = q.size(3) - latent_dim;
    TORCH_CHECK_VALUE((latent_dim == 256 || latent_dim == 512) &&
                      (rope == 32 || rope == 64),
                      "latent_cache_attention: rows must be 256 or 512 "
                      "latent and 32 or 64 rotary columns, got ", latent_dim,
                      " and ", rope);
    TORCH_CHECK_VALUE(block_table.dim() == 2 && block_table.size(0) == B &&
                      lengths.dim() == 1 && lengths.size(0) == B,
                      "latent_cache_attention: block_table must be [B, P] "
                      "and lengths [B]");
    // the kernel's scale, in powers of two; zero or infinite in 32 bits it
    // would turn hidden scores into NaN
    const float scale2 = scale * 1.4426950408889634;
    TORCH_CHECK_VALUE(scale2 > 0.0f && std::isnormal(scale2),
                      "latent_cache_attention: scale must be positive and in the range of 32 "
                      "bits");
    auto out = torch::empty({B, Sq, H, latent_dim}, q.options());
    if (out.numel() == 0) return out;
    const int64_t page = cache.size(1), width = block_table.size(1);
    if (page == 0 || width == 0) {
        // nothing can be held: every length other than zero is too long
        return out.copy_(torch::where(
            lengths > 0, NAN, 0.0).reshape({B, 1, 1, 1}));
    }
    TORCH_CHECK_VALUE(cache.size(0) > 0,
                      "latent_cache_attention: the cache has no page");
    TORCH_CHECK_VALUE(cache_rows_ok(cache),
                      "latent_cache_attention: cache rows must be contiguous "
                      "and lie at multiples of 16 bytes");
    TORCH_CHECK_VALUE(page * width < (1L << 31) - 128 && B < 65536 &&
                      Sq * H < (1L << 24) && cache.stride(1) < (1L << 26),
                      "latent_cache_attention: too many tokens or rows");
    const auto qa = cache_rows_ok(q) ? q
        : q.clone(at::MemoryFormat::Contiguous);
    const auto table = block_table.size(1) > 1 && block_table.stride(1) != 1
        ? block_table.contiguous() : block_table;
    const auto len = lengths.contiguous();

    CacheArgs a = {};
    a.q = qa.data_ptr();
    a.cache = cache.data_ptr();
    a.table = table.data_ptr<int>();
    a.lengths = len.data_ptr<int>();
    a.out = out.data_ptr();
    a.q_b = qa.stride(0), a.q_s = qa.stride(1), a.q_h = qa.stride(2);
    a.c_p = cache.stride(0), a.c_t = cache.stride(1);
    a.t_b = table.stride(0);
    a.pages = cache.size(0);
    a.page_size = page;
    a.page_shift = (page & (page - 1)) == 0 ? __builtin_ctzl(page) : -1;
    a.B = B, a.H = H, a.Sq = Sq, a.table_width = width;
    a.rows = Sq * H;
    a.scale = scale2;
    const int block_rows = a.rows <= 16 ? 16 : a.rows <= 32 ? 32 : 64;
    a.row_groups = (a.rows + block_rows - 1) / block_rows;
    // LDS holds one block a CU; no more runs than there can be tiles
    const int64_t most = B * ((page * width + 63) / 64);
    TORCH_CHECK_VALUE(most < (1L << 30),
                      "latent_cache_attention: too many tokens");
    a.runs = std::min<int64_t>(std::max(256 / a.row_groups, 1), most);
    // 64 rows: two waves on a SIMD, each with half of a tile, hide more of
    // each other's latencies, but have to join at a segment's end. By the most
    // tokens that a run can have, us with one wave and with two: 2048 (32
    // tiles) 115 and 101, 1024 67 and 67, 512 47 and 52.
    const bool halves = block_rows < 64 || most >= 16 * a.runs;
    a.tile_shift = halves ? 6 : 5;
    // measured on one sequence of 8192: 64 rows 32, 30, 29, 31 us for runs of
    // 64 to 256 tokens; 16 rows of 517 tokens 13, 17, 17, 21 us
    a.least = block_rows < 64 ? 1 : halves ? 2 : 4;
    const int blocks = a.runs * a.row_groups;
    const int64_t slots = 2L * a.runs * a.row_groups;
    auto part = torch::empty({slots * block_rows * (latent_dim + 2)},
                             q.options().dtype(torch::kFloat));
    a.part = part.data_ptr<float>();
    a.part_stat = reinterpret_cast<float2*>(
        a.part + slots * block_rows * latent_dim);
    if (dtype == torch::kBFloat16)
        cache_dispatch<__bf16>(a, latent_dim, rope, block_rows, blocks);
    else
        cache_dispatch<_Float16>(a, latent_dim, rope, block_rows, blocks);
    HIP_CHECK_LAST();
    return out;
}
