// Rotary positions: each pair (a, b) of a head's columns is turned by the
// angle position * frequency,
//   a' = scale * (a cos - b sin),   b' = scale * (b cos + a sin),
// with the pairs next to each other (interleaved) or half the rotated width
// apart. The turn the other way (inverse) is also the gradient.
//
// The angle is formed and reduced in 64 bits from an fp64 frequency vector
// instead of being read from a table: positions are then unbounded (a 32-bit
// product is off by a whole turn near position 2^24), nothing can be indexed
// out of range, and the trigonometry is paid once a token for all heads of
// queries and keys, which share one launch. Bound by memory: every element
// is read and written once, 16 B a lane (16411 tokens, 40 heads of 128 fp16,
// 336 MB: 73 us, 4.6 TB/s of the 5.1 that a large copy reaches; 12608 tokens,
// 24 heads of 64 bf16, 77 MB: 14.7 us).
#include <torch/extension.h>

#include <ATen/TensorUtils.h>
#include <algorithm>
#include <vector>

#include <c10/core/DeviceGuard.h>

#include "common.h"

namespace {

struct RotaryTensor {
    const void* in;
    void* out;
    long in_b, in_s, in_h;      // strides in elements
    long out_b, out_s, out_h;
    int heads;
};

struct RotaryArgs {
    RotaryTensor t[2];          // queries, keys (heads 0 = absent)
    const void* positions;      // [B * S]
    const double* freqs;        // [pairs]
    int tokens, seq;            // B * S, S
    int pairs, offset;          // rotated columns: offset .. offset + 2*pairs
    int rot_items, items;       // work items a head, in all
    int copy_lo;                // copied items below the rotated columns
    int block0, tokens_per_block;
    unsigned items_magic;       // ceil(2^32 / items)
    float scale, sign;
};

constexpr int ROTARY_THREADS = 256;

template <typename T, int VEC> struct RotaryVec {
    typedef T type __attribute__((ext_vector_type(VEC)));
};
template <typename T> struct RotaryVec<T, 1> { typedef T type; };

template <typename T, int VEC>
__device__ __forceinline__ void rotary_load(const T* p, float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        v[0] = (float)p[0];
    } else {
        const auto x =
            *reinterpret_cast<const typename RotaryVec<T, VEC>::type*>(p);
        #pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = (float)x[j];
    }
}

template <typename T, int VEC>
__device__ __forceinline__ void rotary_store(T* p, const float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        p[0] = (T)v[0];
    } else {
        typename RotaryVec<T, VEC>::type x;
        #pragma unroll
        for (int j = 0; j < VEC; ++j) x[j] = (T)v[j];
        *reinterpret_cast<typename RotaryVec<T, VEC>::type*>(p) = x;
    }
}

// One block turns tokens_per_block tokens. An item is VEC pairs, or VEC
// copied elements; a head has rot_items of the first and items - rot_items
// of the second kind (none in place). VEC 1 serves any alignment.
template <typename T, int VEC, bool INTERLEAVED, typename POS>
__global__ __launch_bounds__(ROTARY_THREADS) void rotary_kernel(
        RotaryArgs a) {
    extern __shared__ float2 turns[];       // [tokens_per_block][pairs]
    const int tok0 = (a.block0 + blockIdx.x) * a.tokens_per_block;
    const int toks = min(a.tokens_per_block, a.tokens - tok0);

    for (int i = threadIdx.x; i < toks * a.pairs; i += ROTARY_THREADS) {
        const int t = i / a.pairs, p = i - t * a.pairs;
        const double pos = (double)reinterpret_cast<const POS*>(
            a.positions)[tok0 + t];
        // in half turns, so that the reduction is exact; the remainder is
        // in [-1, 1] and 32 bits are enough from there on
        const double half_turns = pos * a.freqs[p] * 0.31830988618379067154;
        const float rest = (float)(half_turns
                                   - 2.0 * rint(half_turns * 0.5));
        float s, c;
        sincospif(rest, &s, &c);
        turns[i] = make_float2(c * a.scale, s * a.scale * a.sign);
    }
    __syncthreads();

    const int per_token = (a.t[0].heads + a.t[1].heads) * a.items;
    int tok = 0, rest = threadIdx.x;
    while (true) {
        while (rest >= per_token) { rest -= per_token; ++tok; }
        if (tok >= toks) break;
        int head = (int)__umulhi((unsigned)rest, a.items_magic);
        if (a.items == 1) head = rest;
        const int item = rest - head * a.items;
        const bool second = head >= a.t[0].heads;
        const RotaryTensor& x = a.t[second ? 1 : 0];
        if (second) head -= a.t[0].heads;
        const int b = (tok0 + tok) / a.seq;
        const int s = (tok0 + tok) - b * a.seq;
        const T* in = reinterpret_cast<const T*>(x.in) + b * x.in_b
                      + s * x.in_s + head * x.in_h;
        T* out = reinterpret_cast<T*>(x.out) + b * x.out_b
                 + s * x.out_s + head * x.out_h;
        if (item < a.rot_items) {
            const int p0 = item * VEC;
            const float2* cs = turns + tok * a.pairs + p0;
            float lo[VEC], hi[VEC];
            if (INTERLEAVED) {
                const T* p = in + a.offset + 2 * p0;
                float even_odd[2][VEC];     // columns 2*p0 .. 2*p0+2*VEC
                rotary_load<T, VEC>(p, even_odd[0]);
                rotary_load<T, VEC>(p + VEC, even_odd[1]);
                #pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    lo[j] = even_odd[(2 * j) / VEC][(2 * j) % VEC];
                    hi[j] = even_odd[(2 * j + 1) / VEC][(2 * j + 1) % VEC];
                }
            } else {
                rotary_load<T, VEC>(in + a.offset + p0, lo);
                rotary_load<T, VEC>(in + a.offset + a.pairs + p0, hi);
            }
            #pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float2 t = cs[j];
                const float x1 = lo[j] * t.x - hi[j] * t.y;
                hi[j] = hi[j] * t.x + lo[j] * t.y;
                lo[j] = x1;
            }
            if (INTERLEAVED) {
                T* p = out + a.offset + 2 * p0;
                float even_odd[2][VEC];
                #pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    even_odd[(2 * j) / VEC][(2 * j) % VEC] = lo[j];
                    even_odd[(2 * j + 1) / VEC][(2 * j + 1) % VEC] = hi[j];
                }
                rotary_store<T, VEC>(p, even_odd[0]);
                rotary_store<T, VEC>(p + VEC, even_odd[1]);
            } else {
                rotary_store<T, VEC>(out + a.offset + p0, lo);
                rotary_store<T, VEC>(out + a.offset + a.pairs + p0, hi);
            }
        } else {
            int c = item - a.rot_items;
            c = c < a.copy_lo ? c * VEC
                              : c * VEC + 2 * a.pairs;
            typedef typename RotaryVec<T, VEC>::type vec;
            *reinterpret_cast<vec*>(out + c) =
                *reinterpret_cast<const vec*>(in + c);
        }
        rest += ROTARY_THREADS;
    }
}

// Whether all addresses of one tensor allow 16-byte accesses.
bool rotary_aligned(const torch::Tensor& x, int vec) {
    if (reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 != 0) return false;
    for (int64_t d = 0; d + 1 < x.dim(); ++d)
        if (x.size(d) > 1 && x.stride(d) % vec != 0) return false;
    return true;
}

// the sizes of [.., H, D] as [B, S, H, D]
std::vector<int64_t> rotary_sizes4(const torch::Tensor& x) {
    std::vector<int64_t> sizes(4, 1);
    for (int64_t d = 0; d < x.dim(); ++d)
        sizes[std::max<int64_t>(d + 4 - x.dim(), 0)] *= x.size(d);
    return sizes;
}

// whether that is a view, the leading dimensions being one in memory
bool rotary_is_view4(const torch::Tensor& x) {
    return at::detail::computeStride(x.sizes(), x.strides(),
                                     rotary_sizes4(x)).has_value();
}

// over the same memory where it is, else a copy
torch::Tensor rotary_as4(const torch::Tensor& x) {
    return x.dim() == 4 ? x : x.reshape(rotary_sizes4(x));
}

void rotary_check(const torch::Tensor& x, const char* name) {
    TORCH_CHECK_VALUE(x.dim() >= 2, "rotary: ", name,
                      " must be [.., heads, dim]");
    TORCH_CHECK_VALUE(x.size(-1) <= 1 || x.stride(-1) == 1, "rotary: ", name,
                      " must be contiguous in its last dimension");
}

// Two heads' columns that share memory would be turned twice, in no order. A
// head's turned columns are one range of bytes, so the question is whether
// some sum of strides, each times a number in its limits, comes within that
// range's length of the distance between two heads.
struct RotaryStep {
    int64_t stride, low, high;
};

// Whether target - sum of number x stride can lie within reach of zero,
// `nonzero`: with a number other than zero. Steps by falling stride, so that
// nested layouts leave one or two numbers to try for each; what takes more
// than `tries` counts as yes.
bool rotary_reaches(const std::vector<RotaryStep>& steps, size_t at,
                    int64_t target, int64_t reach, bool nonzero, int& tries) {
    if (--tries < 0) return true;
    if (at == steps.size()) return !nonzero && std::abs(target) <= reach;
    int64_t low = -reach, high = reach;     // of what the rest can add
    for (size_t i = at + 1; i < steps.size(); ++i) {
        low += steps[i].low * steps[i].stride;
        high += steps[i].high * steps[i].stride;
    }
    const int64_t s = steps[at].stride;
    const auto down = [s](int64_t v) {
        return v >= 0 ? v / s : -((-v + s - 1) / s);
    };
    const int64_t first = std::max(steps[at].low, -down(high - target));
    const int64_t last = std::min(steps[at].high, down(target - low));
    for (int64_t n = first; n <= last; ++n)
        if (rotary_reaches(steps, at + 1, target - n * s, reach,
                           nonzero && n == 0, tries))
            return true;
    return false;
}

constexpr int ROTARY_TRIES = 1 << 14;

// both over the tensors' `width` turned columns, of equal place in the heads
bool rotary_overlaps_itself(const torch::Tensor& x, int64_t width) {
    std::vector<RotaryStep> steps;
    for (int64_t d = 0; d + 1 < x.dim(); ++d) {
        if (x.size(d) == 0) return false;
        if (x.size(d) == 1) continue;
        if (x.stride(d) == 0) return true;
        steps.push_back({x.stride(d), 1 - x.size(d), x.size(d) - 1});
    }
    std::sort(steps.begin(), steps.end(), [](const auto& a, const auto& b) {
        return a.stride > b.stride;
    });
    int tries = ROTARY_TRIES;
    return rotary_reaches(steps, 0, 0, width - 1, true, tries);
}

bool rotary_overlap(const torch::Tensor& q, const torch::Tensor& k,
                    int64_t width) {
    const int64_t size = q.element_size();
    std::vector<RotaryStep> steps;
    for (const auto* x : {&q, &k})
        for (int64_t d = 0; d + 1 < x->dim(); ++d) {
            if (x->size(d) == 0) return false;
            if (x->size(d) == 1) continue;
            const int64_t stride = x->stride(d) * size, n = x->size(d) - 1;
            auto same = std::find_if(
                steps.begin(), steps.end(),
                [stride](const auto& s) { return s.stride == stride; });
            if (same == steps.end())
                same = steps.insert(same, {stride, 0, 0});
            (x == &q ? same->high : same->low) += x == &q ? n : -n;
        }
    std::sort(steps.begin(), steps.end(), [](const auto& a, const auto& b) {
        return a.stride > b.stride;
    });
    int tries = ROTARY_TRIES;
    return rotary_reaches(
        steps, 0, static_cast<const char*>(k.data_ptr())
                      - static_cast<const char*>(q.data_ptr()),
        width * size - 1, false, tries);
}

// A launch has less than 2^32 threads, so very many tokens take several.
template <typename T, int VEC, bool INTERLEAVED>
void rotary_launch(RotaryArgs a, bool wide, int blocks, size_t lds) {
    constexpr int MOST = (int)((1L << 32) / ROTARY_THREADS) - 1;
    for (long first = 0; first < blocks; first += MOST) {
        a.block0 = first;
        const dim3 grid(std::min(blocks - a.block0, MOST));
        if (wide)
            hipLaunchKernelGGL((rotary_kernel<T, VEC, INTERLEAVED, int64_t>),
                               grid, dim3(ROTARY_THREADS), lds,
                               pe_current_stream(), a);
        else
            hipLaunchKernelGGL((rotary_kernel<T, VEC, INTERLEAVED, int32_t>),
                               grid, dim3(ROTARY_THREADS), lds,
                               pe_current_stream(), a);
    }
}

template <typename T, int WIDE>
void rotary_dispatch(const RotaryArgs& a, bool vec, bool interleaved,
                     bool wide, int blocks, size_t lds) {
    if (vec && interleaved) rotary_launch<T, WIDE, true>(a, wide, blocks, lds);
    else if (vec) rotary_launch<T, WIDE, false>(a, wide, blocks, lds);
    else if (interleaved) rotary_launch<T, 1, true>(a, wide, blocks, lds);
    else rotary_launch<T, 1, false>(a, wide, blocks, lds);
}

}  // namespace

std::tuple<torch::Tensor, c10::optional<torch::Tensor>> rotary_op(
        torch::Tensor q, torch::Tensor positions, torch::Tensor freqs,
        c10::optional<torch::Tensor> k, bool interleaved, int64_t offset,
        bool inverse, double scale, bool in_place) {
    TORCH_CHECK_VALUE(q.is_cuda(), "rotary: q must be a GPU tensor");
    const c10::DeviceGuard guard(q.device());
    const auto dtype = q.scalar_type();
    TORCH_CHECK_TYPE(dtype == torch::kBFloat16 || dtype == torch::kHalf ||
                     dtype == torch::kFloat,
                     "rotary: q must be bfloat16, float16 or float32");
    TORCH_CHECK_TYPE(positions.scalar_type() == torch::kInt ||
                     positions.scalar_type() == torch::kLong,
                     "rotary: positions must be int32 or int64");
    TORCH_CHECK_TYPE(freqs.scalar_type() == torch::kDouble &&
                     freqs.dim() == 1,
                     "rotary: freqs must be a float64 vector");
    TORCH_CHECK_VALUE(positions.device() == q.device() &&
                      freqs.device() == q.device(),
                      "rotary: tensors on different devices");
    TORCH_CHECK_VALUE(!(at::GradMode::is_enabled() &&
                        (q.requires_grad() || freqs.requires_grad() ||
                         (k.has_value() && k->requires_grad()))),
                      "rotary: inference only, an input requires a gradient");
    rotary_check(q, "q");
    const int64_t pairs = freqs.numel(), dim = q.size(-1);
    TORCH_CHECK_VALUE(pairs >= 1 && offset >= 0 && offset + 2 * pairs <= dim,
                      "rotary: columns ", offset, " to ", offset + 2 * pairs,
                      " do not fit a head of ", dim);
    TORCH_CHECK_VALUE(pairs <= 1024, "rotary: more than 2048 rotated columns");
    TORCH_CHECK_VALUE(positions.sizes() ==
                      q.sizes().slice(0, q.dim() - 2),
                      "rotary: positions must be one a token, shape ",
                      q.sizes().slice(0, q.dim() - 2),
                      ", got ", positions.sizes());
    if (k.has_value()) {
        TORCH_CHECK_TYPE(k->scalar_type() == dtype,
                         "rotary: q and k must have one type");
        TORCH_CHECK_VALUE(k->device() == q.device(),
                          "rotary: tensors on different devices");
        TORCH_CHECK_VALUE(k->dim() == q.dim() && k->size(-1) == dim &&
                          k->sizes().slice(0, q.dim() - 2) ==
                          q.sizes().slice(0, q.dim() - 2),
                          "rotary: k must match q except in its heads");
        rotary_check(*k, "k");
    }
    torch::Tensor q_out = q, k_out;
    if (in_place) {
        const int64_t width = 2 * pairs;
        TORCH_CHECK_VALUE(!rotary_overlaps_itself(q, width) &&
                          !(k.has_value() &&
                            rotary_overlaps_itself(*k, width)),
                          "rotary_: a tensor overlaps itself");
        if (k.has_value()) {
            TORCH_CHECK_VALUE(!rotary_overlap(q, *k, width),
                              "rotary_: q and k overlap");
            k_out = *k;
        }
        // a graph that has saved either has to find out, as after torch's own
        // operators (tensors made in inference mode carry no version)
        for (const auto& x : {q, k_out})
            if (x.defined() && !x.is_inference())
                x.unsafeGetTensorImpl()->bump_version();
    } else {
        q_out = torch::empty(q.sizes(), q.options());
        if (k.has_value()) k_out = torch::empty(k->sizes(), k->options());
    }
    c10::optional<torch::Tensor> k_result;
    if (k.has_value()) k_result = k_out;

    if (in_place && q.dim() > 4 &&
        !(rotary_is_view4(q) && (!k.has_value() || rotary_is_view4(*k)))) {
        // leading dimensions that are not one in memory: each by itself
        for (int64_t i = 0; i < q.size(0); ++i)
            rotary_op(q.select(0, i), positions.select(0, i), freqs,
                      k.has_value()
                          ? c10::optional<torch::Tensor>(k->select(0, i))
                          : c10::nullopt,
                      interleaved, offset, inverse, scale, true);
        return {q_out, k_result};
    }
    const auto q4 = rotary_as4(q);
    const auto k4 = k.has_value() ? rotary_as4(*k) : torch::Tensor();
    const int64_t tokens = q4.size(0) * q4.size(1);
    const int64_t heads = q4.size(2) + (k.has_value() ? k4.size(2) : 0);
    if (tokens == 0 || heads == 0) return {q_out, k_result};
    // the kernel's division by a reciprocal is exact below 2^32 / dim
    TORCH_CHECK_VALUE(tokens < (1L << 31) && heads * dim * dim < (1L << 32),
                      "rotary: too many tokens or columns");
    const auto q4_out = in_place ? q4 : rotary_as4(q_out);
    const auto k4_out = !k.has_value() || in_place
        ? k4 : rotary_as4(k_out);

    const int wide = dtype == torch::kFloat ? 4 : 8;
    bool vec = pairs % wide == 0 && offset % wide == 0 && dim % wide == 0 &&
        rotary_aligned(q4, wide) && rotary_aligned(q4_out, wide);
    if (k.has_value())
        vec = vec && rotary_aligned(k4, wide) && rotary_aligned(k4_out, wide);

    RotaryArgs a = {};
    const auto fill = [](RotaryTensor& t, const torch::Tensor& in,
                         const torch::Tensor& out) {
        t.in = in.data_ptr();
        t.out = out.data_ptr();
        t.in_b = in.stride(0), t.in_s = in.stride(1), t.in_h = in.stride(2);
        t.out_b = out.stride(0), t.out_s = out.stride(1);
        t.out_h = out.stride(2);
        t.heads = in.size(2);
    };
    fill(a.t[0], q4, q4_out);
    if (k.has_value()) fill(a.t[1], k4, k4_out);
    const auto pos = positions.contiguous();
    const auto freqs_c = freqs.contiguous();
    a.positions = pos.data_ptr();
    a.freqs = freqs_c.data_ptr<double>();
    a.tokens = tokens;
    a.seq = q4.size(1);
    a.pairs = pairs;
    a.offset = offset;
    const int v = vec ? wide : 1;
    a.rot_items = pairs / v;
    a.copy_lo = offset / v;
    a.items = a.rot_items + (in_place ? 0 : (dim - 2 * pairs) / v);
    a.items_magic = (unsigned)(((1UL << 32) + a.items - 1) / a.items);
    a.scale = scale;
    a.sign = inverse ? -1.0f : 1.0f;
    // three items a thread: enough blocks to fill the chip at a microbatch,
    // and the trigonometry of a block is about one pair a thread
    const long per_token = heads * a.items;
    long tpb = (3 * ROTARY_THREADS + per_token - 1) / per_token;
    tpb = std::min<long>(tpb, std::max<long>(1, 2048 / pairs));
    a.tokens_per_block = std::min<long>(tpb, tokens);
    const int blocks = (tokens + a.tokens_per_block - 1) / a.tokens_per_block;
    const size_t lds = a.tokens_per_block * pairs * sizeof(float2);
    const bool long_pos = pos.scalar_type() == torch::kLong;
    if (dtype == torch::kBFloat16)
        rotary_dispatch<__bf16, 8>(a, vec, interleaved, long_pos, blocks, lds);
    else if (dtype == torch::kHalf)
        rotary_dispatch<_Float16, 8>(a, vec, interleaved, long_pos, blocks,
                                     lds);
    else
        rotary_dispatch<float, 4>(a, vec, interleaved, long_pos, blocks, lds);
    HIP_CHECK_LAST();
    return {q_out, k_result};
}
