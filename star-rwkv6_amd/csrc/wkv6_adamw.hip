// One step of AdamW over many tensors, with gradients clipped by their common norm and moments held in 32 bits or in 8.
//
//   g' = g * max_norm / max(norm, max_norm)                 norm: over all tensors, in 64 bits, always added up in the same order
//   m  = b1 m + (1 - b1) g',   v = b2 v + (1 - b2) g'^2
//   p  = p (1 - lr wd) - (lr / (1 - b1^t)) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Moments in 8 bits: m and r = sqrt(v) as float8 (4 exponent bits, 3 mantissa bits) under one scale for each 256 elements, the
// largest magnitude among them over 448.  (The root, because the format's range of 2^18 then holds a range of 2^36 in v.)  A
// decay of 0.999 changes r by far less than the format's step of an eighth, so rounding to the nearest would leave r where it
// is for ever; it is rounded to one of its two neighbours with the probabilities that keep the mean instead.  The 16 random
// bits for each come from a hash of seed, step, tensor and element: the same call gives the same result.  p is formed from
// the moments before they are rounded, and no r > 0 is rounded to 0.
#include "wkv6_common.h"
#include "wkv6_kernels.h"

namespace wkv6 {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kGroup = 48;          // tensors of one launch: they travel in its arguments, which hold 4 KB
constexpr int kChunk = 4096;        // elements of one workgroup
constexpr int kScaleBlock = 256;    // elements that share a scale
constexpr int kNormBlocks = 1024;   // of a group, at most

struct Group {
    AdamwTensor t[kGroup];
    int first[kGroup + 1];   // chunk at which a tensor begins
    int count;
    int number;              // of the first tensor in the call's list
};

// What a step is done with, worked out once on the device.
struct Plan {
    float clip, decay, rate, root, skip;   // rate = lr / (1 - b1^t), root = 1 / sqrt(1 - b2^t)
    uint32_t key;
};

__device__ __forceinline__ uint32_t mix(uint32_t x) {
    x = (x ^ (x >> 16)) * 0xBB67AE85u;   // (fractions of the roots of 3 and 5, as odd numbers)
    x = (x ^ (x >> 15)) * 0x9E3779B9u;
    return x ^ (x >> 16);
}

template <typename S> __device__ __forceinline__ S block_sum(S v, S *part) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[0];
    for (int i = 1; i < kWaves; ++i) v += part[i];
    return v;
}
__device__ __forceinline__ float block_top(float v, float *part) {   // of magnitudes; NaN if one is
    uint32_t b = __float_as_uint(v);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) b = max(b, (uint32_t)__shfl_xor((int)b, d));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = __uint_as_float(b);
    __syncthreads();
    b = __float_as_uint(part[0]);
    for (int i = 1; i < kWaves; ++i) b = max(b, __float_as_uint(part[i]));
    return __uint_as_float(b);
}

__device__ __forceinline__ int tensor_of(const Group &g, int chunk) {
    int lo = 0, hi = g.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (g.first[mid] <= chunk) lo = mid; else hi = mid;
    }
    return lo;
}

template <typename T> __global__ __launch_bounds__(kThreads) void norm_kernel(Group g, double *partial) {
    __shared__ double part[kWaves];
    double s = 0.;
    for (int chunk = blockIdx.x; chunk < g.first[g.count]; chunk += gridDim.x) {
        const int k = tensor_of(g, chunk);
        const int64_t first = (int64_t)(chunk - g.first[k]) * kChunk, n = min((int64_t)kChunk, g.t[k].numel - first);
        const T *x = static_cast<const T *>(g.t[k].grad) + first;
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const double v = load1(x + i);
            s += v * v;
        }
    }
    s = block_sum(s, part);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

__global__ __launch_bounds__(kThreads) void norm_finish_kernel(const double *partial, int64_t partials, float *norm) {
    __shared__ double part[kWaves];
    double s = 0.;
    for (int64_t i = threadIdx.x; i < partials; i += kThreads) s += partial[i];
    s = block_sum(s, part);
    if (threadIdx.x == 0) *norm = (float)sqrt(s);
}

__global__ void plan_kernel(AdamwStep a, Plan *plan) {
    Plan p;
    const double norm = a.grad_norm ? (double)*a.grad_norm : 0.;
    p.clip = a.max_grad_norm > 0. ? (float)(norm <= a.max_grad_norm ? 1. : a.max_grad_norm / norm) : 1.f;
    p.skip = a.skip_nonfinite && !(norm <= 3.402823466e38) ? 1.f : 0.f;
    const int64_t t = *a.step + 1;
    if (p.skip == 0.f) *a.step = t;
    const double lr = a.lr_device ? (double)*a.lr_device : a.lr;
    p.decay = (float)(1. - lr * a.weight_decay);
    p.rate = (float)(lr / (1. - pow(a.beta1, (double)t)));
    p.root = (float)(1. / sqrt(1. - pow(a.beta2, (double)t)));
    p.key = a.seed * 0x9E3779B9u + (uint32_t)t * 0xBB67AE85u;
    *plan = p;
}

struct Rates {
    float b1, c1, b2, c2, eps;
};

__device__ __forceinline__ uint8_t to_float8(float x, uint32_t random16) {
    // 2^-120 brings the exponents of the two formats together, below float8's smallest normal number too
    const uint32_t bits = __float_as_uint(fabsf(x) * 0x1p-120f) + (random16 << 4);
    return (uint8_t)min(bits >> 20, 0x7Eu);
}
__device__ __forceinline__ float from_float8(uint8_t c) {
    const float x = __uint_as_float((uint32_t)(c & 0x7F) << 20) * 0x1p120f;
    return c & 0x80 ? -x : x;
}

template <typename T, int kBits> __global__ __launch_bounds__(kThreads) void step_kernel(Group g, Rates r, const Plan *plan) {
    __shared__ float part[kWaves];
    const Plan q = *plan;
    if (q.skip != 0.f) return;
    const int chunk = blockIdx.x, k = tensor_of(g, chunk);
    const AdamwTensor t = g.t[k];
    const uint32_t key = mix(q.key + (uint32_t)(g.number + k));
    const int64_t first = (int64_t)(chunk - g.first[k]) * kChunk, end = min(first + kChunk, t.numel);
    T *p = static_cast<T *>(t.param);
    for (int64_t at = first; at < end; at += kThreads) {
        const int64_t i = at + threadIdx.x;
        const bool in = i < end;
        const float grad = in ? load1(static_cast<const T *>(t.grad) + i) * q.clip : 0.f;
        float m = 0.f, v = 0.f;
        float2 scale = make_float2(0.f, 0.f);
        if (kBits == 8) {
            scale = *reinterpret_cast<const float2 *>(t.scales + 2 * (at / kScaleBlock));
            if (in) {
                m = from_float8(static_cast<const uint8_t *>(t.exp_avg)[i]) * scale.x;
                v = from_float8(static_cast<const uint8_t *>(t.exp_avg_sq)[i]) * scale.y;
                v *= v;
            }
        } else if (in) {
            m = static_cast<const float *>(t.exp_avg)[i];
            v = static_cast<const float *>(t.exp_avg_sq)[i];
        }
        m = m * r.b1 + grad * r.c1;
        v = v * r.b2 + grad * grad * r.c2;
        const float root = sqrtf(v);
        if (in) {
            float w = t.master ? t.master[i] : load1(p + i);
            w = w * q.decay - m * q.rate / (root * q.root + r.eps);
            if (t.master) t.master[i] = w;
            store1(p + i, w);
        }
        if (kBits == 8) {
            const float top_m = block_top(in ? fabsf(m) : 0.f, part), top_r = block_top(in ? root : 0.f, part);
            const float sm = top_m < 0x1p-100f ? 0x1p-100f : top_m, sr = top_r < 0x1p-100f ? 0x1p-100f : top_r;
            if (threadIdx.x == 0) *reinterpret_cast<float2 *>(t.scales + 2 * (at / kScaleBlock)) = make_float2(sm * (1.f / 448.f), sr * (1.f / 448.f));
            if (in) {
                const uint32_t h = mix((uint32_t)i * 0x9E3779B9u + key);
                const uint8_t cm = to_float8(m * (448.f / sm), h & 0xFFFF);
                uint8_t cr = to_float8(root * (448.f / sr), h >> 16);
                if (cr == 0 && root > 0.f) cr = 1;
                static_cast<uint8_t *>(t.exp_avg)[i] = cm | (m < 0.f ? 0x80 : 0);
                static_cast<uint8_t *>(t.exp_avg_sq)[i] = cr;
            }
        } else if (in) {
            static_cast<float *>(t.exp_avg)[i] = m;
            static_cast<float *>(t.exp_avg_sq)[i] = v;
        }
    }
}

// The tensors in groups that one launch takes: f(group, its chunks).
template <typename F> void by_group(int64_t count, const AdamwTensor *tensors, F &&f) {
    for (int64_t at = 0; at < count;) {
        Group g;
        g.number = (int)at;
        g.first[0] = 0;
        for (g.count = 0; g.count < kGroup && at < count; ++g.count, ++at) {
            const int64_t chunks = (tensors[at].numel + kChunk - 1) / kChunk;
            if (g.first[g.count] + chunks > 0x3fffffff) break;   // (chunks are numbered in 32 bits; one tensor has at most 2^28)
            g.t[g.count] = tensors[at];
            g.first[g.count + 1] = g.first[g.count] + (int)chunks;
        }
        if (g.first[g.count] > 0) f(g, g.first[g.count]);
    }
}

template <typename F> hipError_t by_type(int dtype, F &&f) {
    if (dtype == kBF16) f(bf16_t{});
    else if (dtype == kF16) f(f16_t{});
    else f(float{});
    return hipGetLastError();
}

}  // namespace

// (a group ends early only before more than 2^30 chunks: twice the groups are more than enough)
size_t grad_norm_workspace_bytes(int64_t count) {
    return (size_t)(2 * ((count + kGroup - 1) / kGroup)) * kNormBlocks * sizeof(double);
}

hipError_t grad_norm(hipStream_t st, int dtype, int64_t count, const AdamwTensor *tensors, float *norm, void *workspace) {
    return by_type(dtype, [&](auto t) {
        double *partial = static_cast<double *>(workspace);
        int64_t partials = 0;
        by_group(count, tensors, [&](const Group &g, int chunks) {
            const int blocks = chunks < kNormBlocks ? chunks : kNormBlocks;
            hipLaunchKernelGGL((norm_kernel<decltype(t)>), dim3(blocks), dim3(kThreads), 0, st, g, partial + partials);
            partials += blocks;
        });
        hipLaunchKernelGGL(norm_finish_kernel, dim3(1), dim3(kThreads), 0, st, partial, partials, norm);
    });
}

size_t adamw_workspace_bytes(int64_t) { return 256; }

hipError_t adamw_step(hipStream_t st, int dtype, int moment_bits, int64_t count, const AdamwTensor *tensors, const AdamwStep &s, void *workspace) {
    Plan *plan = static_cast<Plan *>(workspace);
    const Rates r{(float)s.beta1, (float)(1. - s.beta1), (float)s.beta2, (float)(1. - s.beta2), (float)s.eps};
    return by_type(dtype, [&](auto t) {
        hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(1), 0, st, s, plan);
        by_group(count, tensors, [&](const Group &g, int chunks) {
            if (moment_bits == 8) hipLaunchKernelGGL((step_kernel<decltype(t), 8>), dim3(chunks), dim3(kThreads), 0, st, g, r, plan);
            else hipLaunchKernelGGL((step_kernel<decltype(t), 32>), dim3(chunks), dim3(kThreads), 0, st, g, r, plan);
        });
    });
}

}  // namespace wkv6
