// Losses over the logits of a vocabulary, and their gradients by the logits.
//
//   x = logits / temperature (one row of V values per token),  lse = log sum_j exp(x_j),  lp = x_id - lse
//   dL/dlogits_j = (c / temperature) (1[j = id] - exp(x_j - lse)),  c = dL/dlp of that token
//
// A token counts if its mask (where there is one) is not zero and its id is not negative.  The row of one that does not count
// is not read, whatever it holds; its lp is zero and its gradient's row is written as zeros.  An id beyond the vocabulary makes
// lp and the row's gradient NaN.
//
// A row is kept as two numbers, stats = (top, sum): top = max_j logits_j, sum = sum_j exp((logits_j - top) / temperature).
// lp = (logits_id - top) / temperature - log(sum) and p_j = exp((logits_j - top) / temperature) / sum then have the accuracy of
// fp32 at any offset of the logits, which x - lse with lse rounded to fp32 does not.
//
// No sum depends on an order that changes from run to run: rows are added up by one workgroup in 64 bits.
#include "wkv6_common.h"
#include "wkv6_kernels.h"

namespace wkv6 {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kFinish = 1024;        // threads of the one workgroup that adds up
constexpr int kCountBlocks = 256;    // at most
constexpr double kLog2e = 1.44269504088896340736;

// exp(d / temperature) as a power of two.  log2(e) / temperature rounded to fp32 is off by up to 2^-24 of itself, the same way in
// every element: lp would be off by as much times the mean of d, over a whole text hundreds of times that.  `low` is what the rounding left.
struct Scale {
    float high, low;
    __device__ __forceinline__ explicit Scale(float inv_temperature) {
        const double s = kLog2e * inv_temperature;
        high = (float)s;
        low = (float)(s - high);
    }
    __device__ __forceinline__ float exp(float d) const { return __builtin_amdgcn_exp2f(__builtin_fmaf(d, high, d * low)); }
};

__device__ __forceinline__ bool counts(const LossRows &a, int64_t row, int64_t id) {
    return id >= 0 && (a.mask == nullptr || a.mask[row] != 0);
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
    return v;
}
template <typename S> __device__ __forceinline__ S wave_sum(S v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
// Over the workgroup, for every thread; `part`: one value per wave in LDS that nothing else is read from meanwhile.
template <int kW> __device__ __forceinline__ float block_max(float v, float *part) {
    v = wave_max(v);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int i = 1; i < kW; ++i) v = fmaxf(v, part[i]);
    return v;
}
template <int kW, typename S> __device__ __forceinline__ S block_sum(S v, S *part) {
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int i = 1; i < kW; ++i) v += part[i];
    return v;
}

// Counted tokens of each text, and of each workgroup's texts together: tokens, and texts that have any.
__global__ __launch_bounds__(kThreads) void count_kernel(LossRows a, LossCounts c) {
    __shared__ int part[2][kWaves];
    int64_t tokens = 0, texts = 0;
    int turn = 0;
    for (int64_t b = blockIdx.x; b < a.B; b += gridDim.x, turn ^= 1) {
        int n = 0;
        for (int64_t t = threadIdx.x; t < a.T; t += kThreads) n += counts(a, b * a.T + t, a.ids[b * a.T + t]);
        n = block_sum<kWaves>(n, part[turn]);
        if (threadIdx.x == 0) c.by_text[b] = n;
        tokens += n;
        texts += n > 0;
    }
    if (threadIdx.x == 0) c.tokens[blockIdx.x] = (int)tokens, c.texts[blockIdx.x] = (int)texts;
}

// The weight of each of text b's tokens in the loss.
__device__ __forceinline__ float weight_of(const LossCounts &c, int64_t b, int reduction) {
    if (reduction == kLossSum) return 1.f;
    const int *of = reduction == kLossMean ? c.tokens : c.texts;
    int64_t n = 0;
    for (int i = threadIdx.x & 63; i < c.blocks; i += 64) n += of[i];
    n = wave_sum(n);
    const double all = reduction == kLossMean ? (double)n : (double)n * c.by_text[b];
    return all > 0. ? (float)(1. / all) : 0.f;
}

// What a loss makes of one token's lp: its weighted terms, for the finishing kernel to add up, and c.
__device__ __forceinline__ float row_terms(const LossRows &a, const LossTerms &l, int64_t row, double exact, float w) {
    const int64_t rows = a.B * a.T;
    const float lp = (float)exact;
    if (l.kind == kLossCrossEntropy) {
        l.terms[row] = -lp * w;
        return lp == lp ? -w : lp;
    }
    const int64_t b = row / a.T, t = row % a.T;
    const float A = l.advantages[b * l.adv_stride_b + t * l.adv_stride_t];
    const float ratio = l.old_logps ? expf(lp - l.old_logps[row]) : 1.f + (lp - lp);   // (the sampling model is this one: NaN stays NaN)
    const float free = ratio * A, held = fminf(fmaxf(ratio, 1.f - l.clip_low), 1.f + l.clip_high) * A;
    const bool clipped = free > held;
    float kl = 0.f, by_lp = clipped ? 0.f : -free;
    if (l.ref_logps) {
        const float e = l.ref_logps[row] - lp, g = expm1f(e);   // (small where the models agree: neither term is formed from 1)
        kl = g - e;
        by_lp -= l.kl_weight * g;
    }
    l.terms[row] = (l.kl_weight * kl - (clipped ? held : free)) * w;
    l.terms[rows + row] = kl * w;
    l.terms[2 * rows + row] = clipped ? w : 0.f;
    return by_lp * w;
}

// top, sum and lp of every row, and what the loss makes of it.
template <typename T> __global__ __launch_bounds__(kThreads) void rows_kernel(LossRows a, LossCounts n, LossTerms l) {
    __shared__ float part_max[kWaves], part_sum[kWaves];
    const int64_t row = blockIdx.x, b = row / a.T;
    const int64_t id = a.ids[row];
    if (!counts(a, row, id)) {
        if (threadIdx.x == 0) {
            if (a.logps) a.logps[row] = 0.f;
            if (a.exact) a.exact[row] = 0.;
            if (a.stats) a.stats[2 * row] = 0.f, a.stats[2 * row + 1] = 1.f;
            if (l.coef) l.coef[row] = 0.f;
            for (int i = 0; i < l.count; ++i) l.terms[i * a.B * a.T + row] = 0.f;
        }
        return;
    }
    const T *x = static_cast<const T *>(a.logits) + b * a.stride_b + row % a.T * a.stride_t;
    float top = -INFINITY;
    for (int64_t j = threadIdx.x; j < a.V; j += kThreads) top = fmaxf(top, load1(x + j));
    top = block_max<kWaves>(top, part_max);
    const Scale scale(a.inv_temperature);
    float sum = 0.f;
    for (int64_t j = threadIdx.x; j < a.V; j += kThreads) sum += scale.exp(load1(x + j) - top);
    sum = block_sum<kWaves>(sum, part_sum);
    if (threadIdx.x < 64) {
        const double lp = id < a.V ? (double)(load1(x + id) - top) * a.inv_temperature - log((double)sum) : NAN;
        const float w = l.kind == kLossNone ? 0.f : weight_of(n, b, l.reduction);
        if (threadIdx.x == 0) {
            if (a.logps) a.logps[row] = (float)lp;
            if (a.exact) a.exact[row] = lp;
            if (a.stats) a.stats[2 * row] = top, a.stats[2 * row + 1] = sum;
            if (l.kind != kLossNone) {
                const float c = row_terms(a, l, row, lp, w);
                if (l.coef) l.coef[row] = c;
            }
        }
    }
}

// The sums of up to three arrays of terms.
__global__ __launch_bounds__(kFinish) void finish_kernel(int64_t rows, LossTerms l) {
    __shared__ double part[3][kFinish / 64];
    for (int i = 0; i < l.count; ++i) {
        double s = 0.;
        for (int64_t r = threadIdx.x; r < rows; r += kFinish) s += l.terms[i * rows + r];
        s = block_sum<kFinish / 64>(s, part[i]);
        if (threadIdx.x == 0) (i == 0 ? l.loss[0] : l.means[i - 1]) = (float)s;
    }
}

// Pairs of texts (b and b + P), a wave each: log probabilities of whole texts in 64 bits (sums over thousands of tokens, of
// which a small difference is wanted), the loss of their difference, and c of either text's tokens.
__global__ __launch_bounds__(kFinish) void preference_kernel(LossRows a, PreferenceTerms l) {
    __shared__ double part[kFinish / 64];
    const int lane = threadIdx.x & 63;
    const int64_t P = a.B / 2;
    double loss = 0.;
    for (int64_t b = threadIdx.x >> 6; b < P; b += kFinish / 64) {
        double s[2], len[2];
        for (int i = 0; i < 2; ++i) {
            const int64_t first = (b + i * P) * a.T;
            double v = 0.;
            int64_t n = 0;
            for (int64_t t = lane; t < a.T; t += 64) {
                v += a.exact[first + t];
                n += counts(a, first + t, a.ids[first + t]);
            }
            n = wave_sum(n);
            len[i] = l.average && n > 0 ? 1. / (double)n : 1.;
            s[i] = wave_sum(v) * len[i];
            if (lane == 0) l.text_logps[b + i * P] = (float)s[i];
        }
        double d = s[0] - s[1], by_d;
        if (l.ref_logps) d -= (double)l.ref_logps[b] - (double)l.ref_logps[b + P];
        if (l.kind == kPreferenceSigmoid) {
            const double z = l.beta * d, soft = log1p(exp(-fabs(z))), up = 1. / (1. + exp(-z));
            // (1 - e) softplus(-z) + e softplus(z)
            loss += soft + (1. - l.label_smoothing) * fmax(-z, 0.);
            if (l.label_smoothing > 0.) loss += l.label_smoothing * fmax(z, 0.);
            by_d = l.beta * (up - (1. - l.label_smoothing));
        } else if (l.kind == kPreferenceHinge) {
            const double z = 1. - l.beta * d;
            loss += z <= 0. ? 0. : z;
            by_d = z <= 0. ? 0. : -l.beta + 0. * z;
        } else {
            const double z = d - 0.5 / l.beta;
            loss += z * z;
            by_d = 2. * z;
        }
        if (lane == 0 && l.coef) {
            l.coef[b] = (float)(by_d * len[0] / (double)P);
            l.coef[b + P] = (float)(-by_d * len[1] / (double)P);
        }
    }
    if (lane != 0) loss = 0.;
    loss = block_sum<kFinish / 64>(loss, part);
    if (threadIdx.x == 0) l.loss[0] = (float)(loss / (double)P);
}

template <typename T> __global__ __launch_bounds__(kThreads) void grad_kernel(LossRows a, LossGrad g) {
    const float up = g.upstream ? *g.upstream : 1.f;
    if (g.is_there && up == 1.f) return;
    const int64_t row = blockIdx.x, b = row / a.T, t = row % a.T;
    const int64_t id = a.ids[row];
    T *out = static_cast<T *>(g.grad) + row * a.V;
    if (!counts(a, row, id)) {
        for (int64_t j = threadIdx.x; j < a.V; j += kThreads) store1(out + j, 0.f);
        return;
    }
    const T *x = static_cast<const T *>(a.logits) + b * a.stride_b + t * a.stride_t;
    float c = g.coef[b * g.coef_stride_b + t * g.coef_stride_t] * up * a.inv_temperature;
    if (id >= a.V) c = NAN;
    const float top = a.stats[2 * row], norm = 1.f / a.stats[2 * row + 1];
    const Scale scale(a.inv_temperature);
    for (int64_t j = threadIdx.x; j < a.V; j += kThreads) {
        const float p = scale.exp(load1(x + j) - top) * norm;
        store1(out + j, c * ((j == id ? 1.f : 0.f) - p));
    }
}

template <typename F> hipError_t by_type(int dtype, F &&f) {
    if (dtype == kBF16) f(bf16_t{});
    else if (dtype == kF16) f(f16_t{});
    else f(float{});
    return hipGetLastError();
}

}  // namespace

// three terms for each token and the counts, or lp in 64 bits
size_t loss_workspace_bytes(int64_t B, int64_t T) {
    return (size_t)(3 * B * T) * sizeof(float) + (size_t)(B + 2 * kCountBlocks) * sizeof(int);
}

hipError_t loss_rows(hipStream_t st, int dtype, LossRows a, LossTerms l, void *grad, void *workspace) {
    LossCounts n{};
    const int64_t rows = a.B * a.T;
    if (l.kind != kLossNone) {
        l.terms = static_cast<float *>(workspace);
        l.count = l.kind == kLossPolicy ? 3 : 1;
        n.by_text = reinterpret_cast<int *>(l.terms + 3 * rows);
        n.tokens = n.by_text + a.B;
        n.texts = n.tokens + kCountBlocks;
        n.blocks = (int)(a.B < kCountBlocks ? a.B : kCountBlocks);
        hipLaunchKernelGGL(count_kernel, dim3(n.blocks), dim3(kThreads), 0, st, a, n);
    }
    hipError_t e = by_type(dtype, [&](auto t) {
        hipLaunchKernelGGL((rows_kernel<decltype(t)>), dim3((unsigned)rows), dim3(kThreads), 0, st, a, n, l);
    });
    if (e != hipSuccess || l.kind == kLossNone) return e;
    hipLaunchKernelGGL(finish_kernel, dim3(1), dim3(kFinish), 0, st, rows, l);
    if (!grad) return hipGetLastError();
    return loss_grad(st, dtype, a, LossGrad{l.coef, a.T, 1, nullptr, 0, grad});
}

hipError_t loss_preference(hipStream_t st, LossRows a, PreferenceTerms l) {
    hipLaunchKernelGGL(preference_kernel, dim3(1), dim3(kFinish), 0, st, a, l);
    return hipGetLastError();
}

hipError_t loss_grad(hipStream_t st, int dtype, LossRows a, LossGrad g) {
    return by_type(dtype, [&](auto t) {
        hipLaunchKernelGGL((grad_kernel<decltype(t)>), dim3((unsigned)(a.B * a.T)), dim3(kThreads), 0, st, a, g);
    });
}

}  // namespace wkv6
