// Latent attention, expanded form: each token's latent vector has been
// projected to keys and values of every head (kv), while the rotary part of
// the key is one vector a token that all heads share (k_rope):
//   s = scale * (q[:DN] . kv[:DN] + q[DN:] . k_rope),  out = softmax(s) kv[DN:]
//
// A block owns 128 query rows of one head, a wave 32 of them, and walks over
// the keys in tiles of 64. Both products are computed transposed (tokens or
// value columns as the rows, queries as the columns of 32x32x16 MFMAs), so a
// lane holds scores of one query only: softmax needs one exchange between
// the halves of a wave, and the weights are the second product's operand as
// they are, without leaving their lane. Tiles go to LDS by LDS-DMA while the
// previous one is used; the shared rotary key is staged as it is and never
// copied per head.
//
// Bound by what a wave does in turn: 40 MFMAs a tile (1280 cycles of a SIMD),
// then 32 exponentials a lane and their sums, with a second wave on the SIMD
// to fill the gaps. 4099 queries against 8198 keys, 16 heads of 128 + 64, bf16
// causal: 277 us (296 on the slowest card), 930 TFLOP/s of about 1450 that a
// large matrix product reaches (4096 tokens of 16 heads without a mask: 1030);
// without exponentials 7% less, without loads 17% less time.
#include <torch/extension.h>

#include <algorithm>
#include <cmath>

#include <c10/core/DeviceGuard.h>

#include "mfma_tiles.h"

namespace {

struct LatentArgs {
    const void* q;
    const void* kv;
    const void* k_rope;
    void* out;                  // [B, Sq, H, DN]
    float* sums;                // [parts, B, Sq, H, DN], for parts > 1
    float2* stats;              // [parts, B, Sq, H]: top and total
    const int* lengths;         // [B] or nullptr: all keys
    const int* past;            // [B] or nullptr: Sk - Sq
    long q_b, q_s, q_h, kv_b, kv_s, kv_h, r_b, r_s;   // strides in elements
    int B, H, Sq, Sk, row_blocks, parts;
    bool causal;
    float scale;                // times log2(e)
};

constexpr int KEYS = 64;        // tokens a tile
constexpr int ROWS = 128;       // queries a block

template <typename T, int DN, int DR>
__global__ __launch_bounds__(256, 2) void latent_attention_kernel(
        LatentArgs a) {
    constexpr int CN = DN / 8, CR = DR / 8;
    constexpr int NT = DN / 32;                 // output tiles a wave
    typedef typename TileVec<T>::v8 v8;
    typedef RunningTop<T> softmax;
    // two buffers of [nope | rope | value] images
    constexpr int TILE = KEYS * (2 * DN + DR);
    __shared__ __attribute__((aligned(256))) T smem[2 * TILE];

    // The last rows of all heads first: causal blocks see more keys the later
    // they are, and what starts last should be short (8192 tokens, 12 heads:
    // 320 us with head after head, 254 so). Blocks go to the 8 XCDs in turn,
    // so the blocks of a head, which read the same keys, also share an L2 if
    // the number of heads is a multiple of 8, as it mostly is.
    // An XCD's first 32 blocks go to its 32 CUs one by one, then as many more:
    // these in reverse, so that a CU's two add up to about the same (2 to 3%).
    const int heads = a.B * a.H;
    int id = blockIdx.x;
    if (a.causal) {
        const int xcd = id % 8, blocks = (gridDim.x - xcd + 7) / 8;
        int i = id / 8;
        if (i >= 32 && i < 64) i = min(blocks, 64) + 31 - i;
        id = i * 8 + xcd;
    }
    const int rest = id / heads, bh = id - rest * heads;
    const int back = rest / a.parts, part = rest - back * a.parts;
    const int b = bh / a.H, h = bh - b * a.H;
    const int q0 = (a.row_blocks - 1 - back) * ROWS;

    const int tid = threadIdx.x;
    const int lane = tid & 63, l31 = lane & 31, hi = lane >> 5;
    const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);

    int len = a.Sk, past = a.Sk - a.Sq;
    if (a.lengths) len = min(max(a.lengths[b], 0), a.Sk);
    if (a.past) past = min(max(a.past[b], -a.Sq), a.Sk);

    // the last key that this lane's query sees, -1 for padding
    const int row = q0 + wid * 32 + l31;
    const int pos = past + row;
    int limit = a.causal ? min(pos, len - 1) : len - 1;
    if (row >= a.Sq || pos >= len || pos < 0) limit = -1;
    // the same for the last live query of the block and of the wave
    const auto last_key = [&](int first, int count) {
        const int last = min(min(first + count, a.Sq) - 1, len - 1 - past);
        if (last < first || past + last < 0) return -1;
        return a.causal ? past + last : len - 1;
    };
    const int wave_last = last_key(q0 + wid * 32, 32);
    const int tiles = (last_key(q0, ROWS) + KEYS) / KEYS;

    v8 bq[(DN + DR) / 16];
    {
        const T* p = reinterpret_cast<const T*>(a.q) + b * a.q_b
                     + (long)min(row, a.Sq - 1) * a.q_s + h * a.q_h + hi * 8;
        #pragma unroll
        for (int i = 0; i < (DN + DR) / 16; ++i)
            bq[i] = *reinterpret_cast<const v8*>(p + i * 16);
    }

    const T* kv = reinterpret_cast<const T*>(a.kv) + b * a.kv_b + h * a.kv_h;
    const T* kr = reinterpret_cast<const T*>(a.k_rope) + b * a.r_b;
    // A piece's place in its tile: the lane's row and chunk, as a byte offset
    // from the tile's first token. Tokens behind the last one are read as the
    // last one: their weights are zero, and what lies in the padding cannot
    // reach the sums. That only changes the last tile's offsets.
    constexpr int NP = CN / 4, RP = CR / 4;
    unsigned kv_at[NP], r_at[RP];
    const auto place = [&](int last) {
        #pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int r = (wid + 4 * i) * (64 / CN) + lane / CN;
            const int c = (lane % CN) ^ tile_key<CN>(r);
            kv_at[i] = (unsigned)(min(r, last) * (int)a.kv_s + c * 8) * 2;
        }
        #pragma unroll
        for (int i = 0; i < RP; ++i) {
            const int r = (wid + 4 * i) * (64 / CR) + lane / CR;
            const int c = (lane % CR) ^ tile_key<CR>(r);
            r_at[i] = (unsigned)(min(r, last) * (int)a.r_s + c * 8) * 2;
        }
    };
    place(KEYS);
    const auto stage = [&](int t, int buf) {
        T* base = smem + buf * TILE;
        const int tok0 = t * KEYS;
        if (tok0 + KEYS > len) {
            tile_rare();
            place(len - 1 - tok0);
        }
        const T* k0 = kv + tok0 * a.kv_s;
        const T* r0 = kr + tok0 * a.r_s;
        #pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int p = wid + 4 * i;
            tile_load(k0, kv_at[i], base + p * 512);
            tile_load(k0 + DN, kv_at[i], base + KEYS * (DN + DR) + p * 512);
        }
        #pragma unroll
        for (int i = 0; i < RP; ++i)
            tile_load(r0, r_at[i],
                      base + KEYS * DN + (wid + 4 * i) * 512);
    };

    f32x16 acc[NT] = {};
    float top = -INFINITY, sub = 0.0f, total = 0.0f;

    const unsigned lds = tile_lds(smem);
    const int first = (long)tiles * part / a.parts;
    const int end = (long)tiles * (part + 1) / a.parts;
    if (first < end) stage(first, first & 1);
    #pragma unroll
    for (int i = 0; i < (DN + DR) / 16; ++i) tile_settle(bq[i]);
    for (int t = first; t < end; ++t) {
        const unsigned image = lds + (t & 1) * TILE * 2;
        const unsigned nope = tile_row_base<CN, 32>(image, lane);
        const unsigned rope =
            tile_row_base<CR, 32>(image + KEYS * DN * 2, lane);
        const unsigned value = tile_column_base<CN, 32>(
            image + KEYS * (DN + DR) * 2, lane);
        // this wave's part of tile t has arrived; behind the barrier all
        // parts have, and every wave is done with the other buffer
        tile_arrive();
        if (t + 1 < end) stage(t + 1, (t + 1) & 1);
        const int tok0 = t * KEYS;
        if (tok0 > wave_last) continue;

        // Keys are read from LDS a batch ahead of their MFMAs: left to itself,
        // the compiler reads the two of a step and waits for them (4096 tokens,
        // 12 heads: 112 us, 102 so).
        constexpr int AHEAD = 4, KF = 2 * (DN + DR) / 16;
        static_assert(KF % AHEAD == 0, "whole batches");
        const auto key = [&](int j) {
            const int i = j / 2, m = j % 2;
            return i < DN / 16
                ? tile_row_read<T, CN, 32>(nope, m * 32, i)
                : tile_row_read<T, CR, 32>(rope, m * 32, i - DN / 16);
        };
        f32x16 s[2] = {};
        v8 f[2][AHEAD];
        #pragma unroll
        for (int j = 0; j < AHEAD; ++j) f[0][j] = key(j);
        #pragma unroll
        for (int k = 0; k < KF; ++k) {
            const int b = k / AHEAD, j = k % AHEAD;
            if (k + AHEAD < KF) f[(b + 1) & 1][j] = key(k + AHEAD);
            s[k % 2] = tile_mfma(f[b & 1][j], bq[k / 2], s[k % 2]);
            __builtin_amdgcn_sched_barrier(0);
        }

        if (__any(limit < tok0 + KEYS - 1)) {
            tile_rare();
            #pragma unroll
            for (int m = 0; m < 2; ++m)
                #pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (tok0 + m * 32 + hi * 4 + (i & 3) + 8 * (i >> 2)
                        > limit)
                        s[m][i] = -INFINITY;
        }
        float peak = -INFINITY;
        #pragma unroll
        for (int m = 0; m < 2; ++m)
            #pragma unroll
            for (int i = 0; i < 16; ++i) peak = fmaxf(peak, s[m][i]);
        peak = fmaxf(peak, __shfl_xor(peak, 32)) * a.scale;
        if (__any(peak > top + softmax::SLACK)) {
            tile_rare();
            const float next = fmaxf(top, peak);
            const float turn = top == -INFINITY
                ? 0.0f : __builtin_amdgcn_exp2f(top - next);
            top = next;
            sub = next == -INFINITY ? 0.0f : next - softmax::BIAS;
            total *= turn;
            #pragma unroll
            for (int n = 0; n < NT; ++n)
                #pragma unroll
                for (int i = 0; i < 16; ++i) acc[n][i] *= turn;
        }
        #pragma unroll
        for (int m = 0; m < 2; ++m)
            #pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[m][i] = __builtin_amdgcn_exp2f(
                    fmaf(s[m][i], a.scale, -sub));
                total += s[m][i];
            }
        #pragma unroll
        for (int m = 0; m < 2; ++m)
            #pragma unroll
            for (int c = 0; c < 2; ++c) {
                float p[8];
                #pragma unroll
                for (int j = 0; j < 8; ++j) p[j] = s[m][8 * c + j];
                const v8 w = tile_weights<T>(p);
                #pragma unroll
                for (int n = 0; n < NT; ++n)
                    acc[n] = tile_mfma(tile_column_read<T, CN, 32>(
                        value, m * 32 + c * 16, n), w, acc[n]);
            }
    }

    total += __shfl_xor(total, 32);
    if (a.parts > 1) {
        if (row >= a.Sq) return;
        const long at = (((long)part * a.B + b) * a.Sq + row) * a.H + h;
        if (hi == 0) a.stats[at] = make_float2(top, total);
        if (total == 0.0f) return;      // not read either
        float* sums = a.sums + at * DN + hi * 4;
        #pragma unroll
        for (int n = 0; n < NT; ++n)
            #pragma unroll
            for (int g = 0; g < 4; ++g) {
                f32x4 o;
                #pragma unroll
                for (int j = 0; j < 4; ++j) o[j] = acc[n][g * 4 + j];
                *reinterpret_cast<f32x4*>(sums + n * 32 + g * 8) = o;
            }
        return;
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    if (row < a.Sq) {
        T* out = reinterpret_cast<T*>(a.out)
                 + (((long)b * a.Sq + row) * a.H + h) * DN + hi * 4;
        #pragma unroll
        for (int n = 0; n < NT; ++n)
            #pragma unroll
            for (int g = 0; g < 4; ++g) {
                typename TileVec<T>::v4 o;
                // a row that sees nothing is zero, also where its zero weights
                // met values that are not finite
                #pragma unroll
                for (int j = 0; j < 4; ++j)
                    o[j] = (T)(total == 0.0f ? 0.0f
                                             : acc[n][g * 4 + j] * inv);
                *reinterpret_cast<typename TileVec<T>::v4*>(
                    out + n * 32 + g * 8) = o;
            }
    }
}

// Joins the parts of each row, in their order: DN / 4 lanes a row.
template <typename T, int DN>
__global__ __launch_bounds__(256) void latent_join_kernel(
        const float* __restrict__ sums, const float2* __restrict__ stats,
        T* __restrict__ out, long rows, int parts) {
    constexpr int LANES = DN / 4;
    const long row = (long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    if (row >= rows) return;
    const int col = threadIdx.x % LANES * 4;
    float top = -INFINITY;
    for (int p = 0; p < parts; ++p) top = fmaxf(top, stats[p * rows + row].x);
    float total = 0.0f;
    f32x4 sum = {};
    #pragma unroll 4
    for (int p = 0; p < parts; ++p) {
        const float2 s = stats[p * rows + row];
        if (s.y == 0.0f) continue;
        const float w = __builtin_amdgcn_exp2f(s.x - top);
        total += s.y * w;
        sum += *reinterpret_cast<const f32x4*>(
            sums + (p * rows + row) * DN + col) * w;
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    typename TileVec<T>::v4 o;
    #pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = (T)(sum[j] * inv);
    *reinterpret_cast<typename TileVec<T>::v4*>(out + row * DN + col) = o;
}

// 16-byte accesses need strides and addresses of 8 elements
torch::Tensor latent_aligned(const torch::Tensor& x) {
    bool ok = reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0 &&
              x.stride(-1) == 1;
    for (int64_t d = 0; d + 1 < x.dim(); ++d)
        ok = ok && (x.size(d) == 1 || x.stride(d) % 8 == 0);
    return ok ? x : x.clone(at::MemoryFormat::Contiguous);
}

template <typename T, int DN, int DR>
void latent_launch(const LatentArgs& a, long blocks) {
    hipLaunchKernelGGL((latent_attention_kernel<T, DN, DR>), dim3(blocks),
                       dim3(256), 0, pe_current_stream(), a);
    if (a.parts == 1) return;
    const long rows = (long)a.B * a.Sq * a.H;
    const int block_rows = 256 / (DN / 4);
    hipLaunchKernelGGL((latent_join_kernel<T, DN>),
                       dim3((rows + block_rows - 1) / block_rows), dim3(256),
                       0, pe_current_stream(), a.sums, a.stats,
                       reinterpret_cast<T*>(a.out), rows, a.parts);
}

template <typename T>
void latent_dispatch(const LatentArgs& a, int nope, int rope, long blocks) {
    if (nope == 128 && rope == 64) latent_launch<T, 128, 64>(a, blocks);
    else if (nope == 128) latent_launch<T, 128, 32>(a, blocks);
    else if (rope == 64) latent_launch<T, 64, 64>(a, blocks);
    else latent_launch<T, 64, 32>(a, blocks);
}

}  // namespace

torch::Tensor latent_attention_op(
        torch::Tensor q, torch::Tensor kv, torch::Tensor k_rope, double scale,
        bool causal, c10::optional<torch::Tensor> lengths,
        c10::optional<torch::Tensor> past) {
    TORCH_CHECK_VALUE(q.is_cuda(), "latent_attention: GPU tensors required");
    const c10::DeviceGuard guard(q.device());
    const auto dtype = q.scalar_type();
    TORCH_CHECK_TYPE((dtype == torch::kBFloat16 || dtype == torch::kHalf) &&
                     kv.scalar_type() == dtype &&
                     k_rope.scalar_type() == dtype,
                     "latent_attention: q, kv and k_rope must be all bfloat16"
                     " or all float16");
    TORCH_CHECK_VALUE(kv.device() == q.device() &&
                      k_rope.device() == q.device(),
                      "latent_attention: tensors on different devices");
    TORCH_CHECK_VALUE(!(at::GradMode::is_enabled() &&
                        (q.requires_grad() || kv.requires_grad() ||
                         k_rope.requires_grad())),
                      "latent_attention: inference only, an input requires a "
                      "gradient");
    TORCH_CHECK_VALUE(q.dim() == 4 && kv.dim() == 4 && k_rope.dim() == 3,
                      "latent_attention: q and kv must be [B, S, H, D], "
                      "k_rope [B, S, D]");
    const int64_t B = q.size(0), Sq = q.size(1), H = q.size(2);
    const int64_t Sk = kv.size(1), rope = k_rope.size(2);
    const int64_t nope = q.size(3) - rope;
    TORCH_CHECK_VALUE((nope == 64 || nope == 128) &&
                      (rope == 32 || rope == 64) && kv.size(3) == 2 * nope,
                      "latent_attention: head parts must be 64 or 128 plain "
                      "and 32 or 64 rotary columns with as many values as "
                      "plain ones, got q ", q.size(3), ", kv ", kv.size(3),
                      ", k_rope ", rope);
    TORCH_CHECK_VALUE(kv.size(0) == B && k_rope.size(0) == B &&
                      kv.size(2) == H && k_rope.size(1) == Sk,
                      "latent_attention: q ", q.sizes(), ", kv ", kv.sizes(),
                      " and k_rope ", k_rope.sizes(), " do not match");
    // the kernel's scale, in powers of two; zero or infinite in 32 bits it
    // would turn hidden scores into NaN
    const float scale2 = scale * 1.4426950408889634;
    TORCH_CHECK_VALUE(scale2 > 0.0f && std::isnormal(scale2),
                      "latent_attention: scale must be positive and in the range of 32 "
                      "bits");
    for (const auto* x : {&lengths, &past}) {
        if (!x->has_value()) continue;
        TORCH_CHECK_TYPE((*x)->scalar_type() == torch::kInt,
                         "latent_attention: lengths and past must be int32");
        TORCH_CHECK_VALUE((*x)->dim() == 1 && (*x)->size(0) == B &&
                          (*x)->device() == q.device(),
                          "latent_attention: lengths and past must be one a "
                          "sequence, on the device of q");
    }
    TORCH_CHECK_VALUE(past.has_value() || !lengths.has_value() || Sq == Sk,
                      "latent_attention: lengths with fewer or more queries "
                      "than keys need past");
    auto out = torch::empty({B, Sq, H, nope}, q.options());
    if (out.numel() == 0) return out;
    if (Sk == 0) return out.zero_();
    TORCH_CHECK_VALUE(Sq < (1L << 30) && Sk < (1L << 30),
                      "latent_attention: too many tokens");
    const int64_t row_blocks = (Sq + ROWS - 1) / ROWS;
    // a launch has less than 2^32 threads
    TORCH_CHECK_VALUE(B * H * row_blocks < (1L << 24),
                      "latent_attention: too many rows");
    const auto qa = latent_aligned(q), kva = latent_aligned(kv);
    const auto ra = latent_aligned(k_rope);
    // of what the kernel reads, which may be a copy with other strides
    TORCH_CHECK_VALUE(Sk == 1 || (kva.stride(1) < (1L << 24) &&
                                  ra.stride(1) < (1L << 24)),
                      "latent_attention: tokens 32 MiB or more apart");
    torch::Tensor len_c, past_c;
    LatentArgs a = {};
    a.q = qa.data_ptr();
    a.kv = kva.data_ptr();
    a.k_rope = ra.data_ptr();
    a.out = out.data_ptr();
    if (lengths.has_value()) {
        len_c = lengths->contiguous();
        a.lengths = len_c.data_ptr<int>();
    }
    if (past.has_value()) {
        past_c = past->contiguous();
        a.past = past_c.data_ptr<int>();
    }
    a.q_b = qa.stride(0), a.q_s = qa.stride(1), a.q_h = qa.stride(2);
    a.kv_b = kva.stride(0), a.kv_s = kva.stride(1), a.kv_h = kva.stride(2);
    a.r_b = ra.stride(0), a.r_s = ra.stride(1);
    a.B = B, a.H = H, a.Sq = Sq, a.Sk = Sk, a.row_blocks = row_blocks;
    // Few blocks split the keys and a second kernel joins the parts: two
    // blocks a CU, one if all have the same work (256 blocks of 2048 tokens:
    // 57 us in one part, 62 in two; causal 54 and 50). A part has 8 tiles or
    // more, with a few rows, whose sums are cheap to pass on, 4 (us in one
    // part, with 4 and with 8 tiles a part; 16 heads: 64 rows of 8192 tokens
    // 176, 45, 34; 1 row of 517: 20, 17, 20; 4096 tokens, 4 heads: 92 to 50).
    int64_t blocks = B * H * row_blocks;
    const int64_t tiles = (Sk + KEYS - 1) / KEYS;
    a.parts = std::max<int64_t>(1, std::min((causal ? 512 : 256) / blocks,
                                            tiles / (Sq <= 32 ? 4 : 8)));
    torch::Tensor sums, stats;
    if (a.parts > 1) {
        blocks *= a.parts;
        const auto f32 = q.options().dtype(torch::kFloat);
        sums = torch::empty({a.parts, B, Sq, H, nope}, f32);
        stats = torch::empty({a.parts, B, Sq, H, 2}, f32);
        a.sums = sums.data_ptr<float>();
        a.stats = reinterpret_cast<float2*>(stats.data_ptr<float>());
    }
    a.causal = causal;
    a.scale = scale2;
    if (dtype == torch::kBFloat16)
        latent_dispatch<__bf16>(a, nope, rope, blocks);
    else
        latent_dispatch<_Float16>(a, nope, rope, blocks);
    HIP_CHECK_LAST();
    return out;
}
