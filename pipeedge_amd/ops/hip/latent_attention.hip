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
// they are, without leaving their lane. Tiles go to LDS by LDS-DMA while the previous one is used;
// the shared rotary key is staged as it is and never copied per head.
// Bound by the matrix cores and the LDS reads that feed them.
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>

#include "mfma_tiles.h"

namespace {

struct LatentArgs {
    const void* q;
    const void* kv;
    const void* k_rope;
    void* out;                  // [B, Sq, H, DN]
    const int* lengths;         // [B] or nullptr: all keys
    const int* past;            // [B] or nullptr: Sk - Sq
    long q_b, q_s, q_h, kv_b, kv_s, kv_h, r_b, r_s;   // strides in elements
    int B, H, Sq, Sk, row_blocks;
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

    const int id = xcd_contiguous(blockIdx.x, gridDim.x);
    const int bh = id / a.row_blocks;
    const int b = bh / a.H, h = bh - b * a.H;
    int rb = id - bh * a.row_blocks;
    rb = a.row_blocks - 1 - rb;
    const int q0 = rb * ROWS;

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
    if (tiles > 0) stage(0, 0);
    #pragma unroll
    for (int i = 0; i < (DN + DR) / 16; ++i) tile_settle(bq[i]);
    for (int t = 0; t < tiles; ++t) {
        const unsigned image = lds + (t & 1) * TILE * 2;
        const unsigned nope = tile_row_base<CN, 32>(image, lane);
        const unsigned rope =
            tile_row_base<CR, 32>(image + KEYS * DN * 2, lane);
        const unsigned value = tile_column_base<CN, 32>(
            image + KEYS * (DN + DR) * 2, lane);
        // this wave's part of tile t has arrived; behind the barrier all
        // parts have, and every wave is done with the other buffer
        tile_arrive();
        if (t + 1 < tiles) stage(t + 1, (t + 1) & 1);
        const int tok0 = t * KEYS;
        if (tok0 > wave_last) continue;

        f32x16 s[2] = {};
        #pragma unroll
        for (int i = 0; i < DN / 16; ++i)
            #pragma unroll
            for (int m = 0; m < 2; ++m)
                s[m] = tile_mfma(tile_row_read<T, CN, 32>(nope, m * 32, i),
                                 bq[i], s[m]);
        #pragma unroll
        for (int i = 0; i < DR / 16; ++i)
            #pragma unroll
            for (int m = 0; m < 2; ++m)
                s[m] = tile_mfma(tile_row_read<T, CR, 32>(rope, m * 32, i),
                                 bq[DN / 16 + i], s[m]);

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
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    if (row < a.Sq) {
        T* out = reinterpret_cast<T*>(a.out)
                 + (((long)b * a.Sq + row) * a.H + h) * DN + hi * 4;
        #pragma unroll
        for (int n = 0; n < NT; ++n)
            #pragma unroll
            for (int g = 0; g < 4; ++g) {
                typename TileVec<T>::v4 o;
                #pragma unroll
                for (int j = 0; j < 4; ++j)
                    o[j] = (T)(acc[n][g * 4 + j] * inv);
                *reinterpret_cast<typename TileVec<T>::v4*>(
                    out + n * 32 + g * 8) = o;
            }
    }
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
    TORCH_CHECK_VALUE(scale > 0.0 && std::isfinite(scale),
                      "latent_attention: scale must be positive");
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
    TORCH_CHECK_VALUE(kv.stride(1) < (1L << 24) &&
                      k_rope.stride(1) < (1L << 24),
                      "latent_attention: tokens more than 32 MiB apart");
    const int64_t row_blocks = (Sq + ROWS - 1) / ROWS;
    TORCH_CHECK_VALUE(B * H * row_blocks < (1L << 31),
                      "latent_attention: too many rows");
    const auto qa = latent_aligned(q), kva = latent_aligned(kv);
    const auto ra = latent_aligned(k_rope);
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
    a.causal = causal;
    a.scale = scale * 1.4426950408889634;
    if (dtype == torch::kBFloat16)
        latent_dispatch<__bf16>(a, nope, rope, B * H * row_blocks);
    else
        latent_dispatch<_Float16>(a, nope, rope, B * H * row_blocks);
    HIP_CHECK_LAST();
    return out;
}
