// Projection with low-rank adapters of many requests,
//   y = act(x W^T + b + s_i (x A_i^T) B_i^T) + residual,   i = id of the row,
// in two launches: the inner values s_i x A_i^T of all rows, and the shared
// GEMM, which adds their products with B_i to its accumulators before its
// epilogue (gemm.hip), so y is written once and W is read as without
// adapters. The inner values are rounded to bf16 once, as the operand of the
// second product; the sums before and after stay in fp32.
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>

#include "adapter.h"
#include "common.h"

std::tuple<torch::Tensor, torch::Tensor> gemm_bf16(
        torch::Tensor a2d, torch::Tensor b,
        c10::optional<torch::Tensor> bias, int64_t act,
        c10::optional<torch::Tensor> residual2d, int64_t tile,
        c10::optional<torch::Tensor> ln_stats,
        c10::optional<torch::Tensor> ln_s,
        c10::optional<torch::Tensor> ln_c, double ln_eps, bool want_stats,
        const AdapterRows* adapters);

namespace {

struct InnerArgs {
    const __bf16* x;            // [M][K]
    const __bf16* down;         // [n][rank][K]
    const int* row_ids;
    const float* scales;        // [n] or nullptr
    __bf16* inner;              // [M][rank_pad]
    int M, K, rows_per_id, n_adapters, rank, rank_pad;
    bool vec;                   // rows lie at multiples of 16 bytes
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

// Many rows: a block takes 16 rows by 16 * NC inner columns, its 4 waves a
// quarter of K each, for each adapter among the rows; the waves' sums meet in
// LDS and rows keep those of their own adapter.
template <int NC>
__global__ __launch_bounds__(256) void adapter_inner_kernel(InnerArgs a) {
    __shared__ float parts[4][NC][64][4];
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
    const int l15 = lane & 15, quad = lane >> 4;
    const int row0 = blockIdx.x * 16, col0 = blockIdx.y * 16 * NC;
    const int row = row0 + l15;
    int id = row < a.M ? a.row_ids[row / a.rows_per_id] : -1;
    if (id >= a.n_adapters) id = -1;

    const int steps = (a.K + 31) / 32;
    const int first = wid * steps / 4, last = (wid + 1) * steps / 4;
    const __bf16* x = a.x + (long)min(row, a.M - 1) * a.K + quad * 8;
    f32x4 mine[NC] = {};
    unsigned long long left = __ballot(id >= 0);
    while (left) {
        const int cur = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
        left &= ~__ballot(id == cur);
        const unsigned rows = (unsigned)__ballot(id == cur) >> (quad * 4);
        const __bf16* down = a.down + (long)cur * a.rank * a.K + quad * 8;
        f32x4 acc[NC] = {};
        for (int s = first; s < last; ++s) {
            const int k = s * 32;
            const bf16x8 xa = inner_load(x, k, a.K - quad * 8, a.vec);
            #pragma unroll
            for (int n = 0; n < NC; ++n) {
                const int c = min(col0 + n * 16 + l15, a.rank - 1);
                acc[n] = mfma_16x16x32_bf16(
                    xa, inner_load(down + (long)c * a.K, k,
                                   a.K - quad * 8, a.vec), acc[n]);
            }
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
    for (int n = wid; n < NC; n += 4) {
        const int col = col0 + n * 16 + l15;
        if (col >= a.rank_pad) continue;
        #pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int out_row = row0 + quad * 4 + r;
            const int out_id = __shfl(id, quad * 4 + r);
            if (out_row >= a.M) continue;
            float v = parts[0][n][lane][r] + parts[1][n][lane][r]
                      + parts[2][n][lane][r] + parts[3][n][lane][r];
            if (a.scales != nullptr && out_id >= 0) v *= a.scales[out_id];
            if (out_id < 0 || col >= a.rank) v = 0.0f;
            a.inner[(long)out_row * a.rank_pad + col] = f2bf(v);
        }
    }
}

// Few rows: a wave takes one row and 4 inner columns, a block 16 of them. The
// matrix unit would be idle for want of rows; what counts is that all the
// adapters' rows are on their way at once.
__global__ __launch_bounds__(256) void adapter_inner_step_kernel(
        InnerArgs a) {
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
// on 256 CUs and every wave has its loads on the way before it needs one.
// The adapters' products are a short dot product for each output.
constexpr int STEP_WAVES = 4;

template <int NM>               // groups of 16 rows
__global__ __launch_bounds__(64 * STEP_WAVES) void adapter_step_kernel(
        const __bf16* __restrict__ x, const __bf16* __restrict__ w,
        const __bf16* __restrict__ bias, const __bf16* __restrict__ residual,
        __bf16* __restrict__ out, AdapterRows ad, int M, int N, int K,
        int act, bool vec) {
    constexpr int DEPTH = 4;    // steps of 32 in flight
    __shared__ float parts[STEP_WAVES][NM][16][17];
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
    const int l15 = lane & 15, quad = lane >> 4;
    const int col0 = blockIdx.x * 16;

    const int steps = (K + 31) / 32;
    const int first = wid * steps / STEP_WAVES;
    const int last = (wid + 1) * steps / STEP_WAVES;
    const __bf16* wp = w + (long)min(col0 + l15, N - 1) * K + quad * 8;
    const __bf16* xp[NM];
    #pragma unroll
    for (int m = 0; m < NM; ++m)
        xp[m] = x + (long)min(m * 16 + l15, M - 1) * K + quad * 8;
    f32x4 acc[NM] = {};
    for (int s0 = first; s0 < last; s0 += DEPTH) {
        bf16x8 wv[DEPTH], xv[DEPTH][NM];
        #pragma unroll
        for (int s = 0; s < DEPTH; ++s) {
            // behind the wave's part nothing is loaded
            const int k = (s0 + s) * 32;
            const int end = s0 + s < last ? K - quad * 8 : 0;
            wv[s] = inner_load(wp, k, end, vec);
            #pragma unroll
            for (int m = 0; m < NM; ++m)
                xv[s][m] = inner_load(xp[m], k, end, vec);
        }
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
            const __bf16* in = reinterpret_cast<const __bf16*>(ad.inner)
                               + (long)row * ad.rank_pad;
            const __bf16* up = reinterpret_cast<const __bf16*>(ad.up)
                               + ((long)id * N + col) * ad.rank;
            for (int k = 0; k < ad.rank; k += 8) {
                const bf16x8 a = inner_load(in, k, ad.rank_pad, true);
                const bf16x8 b = inner_load(up, k, ad.rank,
                                            ad.rank % 8 == 0);
                #pragma unroll
                for (int j = 0; j < 8; ++j)
                    v = fmaf(bf2f(a[j]), bf2f(b[j]), v);
            }
        }
        if (bias != nullptr) v += bf2f(bias[col]);
        if (act == ACT_GELU) v = gelu_f(v);
        else if (act == ACT_TANH) v = tanhf(v);
        if (residual != nullptr) v += bf2f(residual[(long)row * N + col]);
        out[(long)row * N + col] = f2bf(v);
    }
}

// Rows that the kernels for few rows take.
constexpr int STEP_ROWS = 64;

void adapter_inner(const InnerArgs& a) {
    const dim3 block(256);
    if (a.M <= STEP_ROWS) {
        hipLaunchKernelGGL(adapter_inner_step_kernel,
                           dim3(a.M, a.rank_pad / 16), block, 0,
                           pe_current_stream(), a);
        return;
    }
    // columns a block: all of them up to 64, then 64 at a time
    const int rows = (a.M + 15) / 16;
    if (a.rank_pad <= 32)
        hipLaunchKernelGGL((adapter_inner_kernel<2>), dim3(rows, 1), block, 0,
                           pe_current_stream(), a);
    else
        hipLaunchKernelGGL((adapter_inner_kernel<4>),
                           dim3(rows, (a.rank_pad + 63) / 64), block, 0,
                           pe_current_stream(), a);
}

template <int NM>
void adapter_step(const torch::Tensor& x, const torch::Tensor& w,
                  const __bf16* bias, const __bf16* residual,
                  torch::Tensor& out, const AdapterRows& rows, int act) {
    const int M = x.size(0), N = w.size(0), K = x.size(1);
    hipLaunchKernelGGL((adapter_step_kernel<NM>), dim3((N + 15) / 16),
                       dim3(64 * STEP_WAVES), 0, pe_current_stream(),
                       reinterpret_cast<const __bf16*>(x.data_ptr()),
                       reinterpret_cast<const __bf16*>(w.data_ptr()), bias,
                       residual, reinterpret_cast<__bf16*>(out.data_ptr()),
                       rows, M, N, K, act, K % 8 == 0);
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
    TORCH_CHECK_VALUE(K > 0 && M < (1L << 31) && N < (1L << 31),
                      "adapter_linear: no inner columns, or too many rows");
    if (M == 0 || N == 0)
        return torch::empty(out_sizes, x.options());

    const auto x2d = adapter_dense(x.reshape({M, K}));
    const auto w = adapter_dense(weight);
    c10::optional<torch::Tensor> res2d;
    if (residual.has_value()) res2d = residual->reshape({M, N});
    if (n == 0 || r == 0)
        return std::get<0>(gemm_bf16(x2d, w, bias, act, res2d, 0,
                                     c10::nullopt, c10::nullopt, c10::nullopt,
                                     1e-12, false, nullptr))
            .reshape(out_sizes);
    const auto down_c = adapter_dense(down), up_c = adapter_dense(up);
    const auto ids_c = ids.contiguous();
    const int rank_pad = (r + 31) / 32 * 32;
    auto inner = torch::empty({M, rank_pad}, x.options());
    InnerArgs in = {};
    in.x = reinterpret_cast<const __bf16*>(x2d.data_ptr());
    in.down = reinterpret_cast<const __bf16*>(down_c.data_ptr());
    in.row_ids = ids_c.data_ptr<int>();
    torch::Tensor scales_c;
    if (scales.has_value()) {
        scales_c = scales->contiguous();
        in.scales = scales_c.data_ptr<float>();
    }
    in.inner = reinterpret_cast<__bf16*>(inner.data_ptr());
    in.M = M, in.K = K, in.n_adapters = n, in.rank = r;
    in.rows_per_id = by_row ? 1 : M / x.size(0);
    in.rank_pad = rank_pad;
    in.vec = K % 8 == 0;
    adapter_inner(in);
    HIP_CHECK_LAST();
    const AdapterRows rows = {inner.data_ptr(), up_c.data_ptr(),
                              ids_c.data_ptr<int>(), in.rows_per_id, (int)n,
                              (int)r, rank_pad};
    if (M <= STEP_ROWS) {
        auto out = torch::empty(out_sizes, x.options());
        const auto pointer = [](c10::optional<torch::Tensor>& t) {
            if (!t.has_value()) return (const __bf16*)nullptr;
            t = t->contiguous();
            return reinterpret_cast<const __bf16*>(t->data_ptr());
        };
        const auto* b = pointer(bias);
        const auto* res = pointer(res2d);
        if (M <= 16) adapter_step<1>(x2d, w, b, res, out, rows, act);
        else if (M <= 32) adapter_step<2>(x2d, w, b, res, out, rows, act);
        else adapter_step<4>(x2d, w, b, res, out, rows, act);
        HIP_CHECK_LAST();
        return out;
    }
    return std::get<0>(gemm_bf16(x2d, w, bias, act, res2d, 0, c10::nullopt,
                                 c10::nullopt, c10::nullopt, 1e-12, false,
                                 &rows)).reshape(out_sizes);
}
