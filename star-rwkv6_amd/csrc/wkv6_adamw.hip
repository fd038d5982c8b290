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
//
// Bound by memory: 28 bytes a parameter with everything in fp32, 10 with bf16 parameters and 8-bit moments (whose some 60 vector operations a parameter
// take two thirds of the time), and the gradient once more for the norm.  490 M parameters in 150 tensors: step 2.43 ms and norm 0.32 ms in fp32
// (5.6 and 6.1 TB/s; elements of a wave's load without gaps, past the caches 10 % faster than through them), 0.98 and 0.18 ms in bf16 with 8 bits; steps of
// bf16 parameters with masters 2.2 ms (6.3 TB/s) and with 8 bits 1.4 (5.5).  Some 1 M parameters in 36 tensors: one launch of 9.5 us.
#include "wkv6_common.h"
#include "wkv6_kernels.h"
#include "wkv6_pieces.h"

#include <math.h>

#include <type_traits>

namespace wkv6 {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kGroup = 60;          // tensors of one launch: they travel in its arguments, which hold 4 KB
constexpr int kChunk = 4096;        // elements that a workgroup takes at a time, 16 to a thread in pieces that lie next to each other
constexpr int kScaleBlock = 256;    // elements that share a scale
// Workgroups of a launch at most, which go from chunk to chunk.  Of step_kernel four or five stand on a compute unit at a time (84 to 115 registers), of norm_kernel eight:
// of 2048 some stand at once and the others follow, and launches of no more than stand at once are no faster.  490 M parameters, fp32 / bf16 with 8 bits, clipped, in us: 1024
// 2824 / 1182, 1280 2762 / 1167, 2048 2760 / 1142, 4096 2748 / 1138, 8192 2738 / 1291.
constexpr int kBlocks = 2048;
constexpr int kFinish = 1024;       // threads of the one workgroup that adds up
constexpr int64_t kPastBytes = 160 << 20;   // of all tensors of a call

struct Group {
    AdamwTensor t[kGroup];
    int first[kGroup + 1];   // chunk at which a tensor begins
    int count;
    int number;              // of the first tensor in the call's list
    int last;                // whether nothing of the call follows
};

// What a step is done with.
struct Plan {
    float clip, decay, rate, root;   // rate = lr / (1 - b1^t), root = 1 / sqrt(1 - b2^t)
    uint32_t key;
    int skip;
};
struct Rates {
    float b1, c1, b2, c2, eps;
};
static_assert(sizeof(Group) + sizeof(Rates) + sizeof(AdamwStep) <= 4096, "a launch's arguments");

__device__ __forceinline__ uint32_t mix(uint32_t x) {
    x = (x ^ (x >> 16)) * 0xBB67AE85u;   // (fractions of the roots of 3 and 5, as odd numbers)
    x = (x ^ (x >> 15)) * 0x9E3779B9u;
    return x ^ (x >> 16);
}

template <int kW> __device__ __forceinline__ double block_sum(double v, double *part) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[0];
    for (int i = 1; i < kW; ++i) v += part[i];
    return v;
}

__device__ __forceinline__ int tensor_of(const Group &g, int chunk) {
    int lo = 0, hi = g.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (g.first[mid] <= chunk) lo = mid; else hi = mid;
    }
    return lo;
}

template <typename F> void either(bool which, F &&f) {   // f(true) or f(false), for code that is compiled for either
    if (which) f(std::true_type{});
    else f(std::false_type{});
}

template <typename T> __global__ __launch_bounds__(kThreads) void norm_kernel(Group g, double *partial) {
    constexpr int kEach = 16 / sizeof(T), kItems = kChunk / kThreads / kEach;
    __shared__ double part[kWaves];
    double s = 0.;
    for (int chunk = blockIdx.x; chunk < g.first[g.count]; chunk += gridDim.x) {
        const int k = tensor_of(g, chunk);
        const int64_t first = (int64_t)(chunk - g.first[k]) * kChunk;
        const T *x = static_cast<const T *>(g.t[k].grad) + first;
        const int n = (int)min((int64_t)kChunk, g.t[k].numel - first);
        Piece<T, kEach> held[kItems];
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
            const int at = (i * kThreads + threadIdx.x) * kEach;
            held[i].template load<false>(x + at, n - at);
        }
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
            float v[kEach];
            unpack(held[i], v);
#pragma unroll
            for (int e = 0; e < kEach; ++e) s = __builtin_fma((double)v[e], (double)v[e], s);
        }
    }
    s = block_sum<kWaves>(s, part);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

__global__ __launch_bounds__(kFinish) void norm_finish_kernel(const double *partial, int64_t partials, float *norm) {
    __shared__ double part[kFinish / 64];
    double s = 0.;
    for (int64_t r = threadIdx.x; r < partials; r += 8 * kFinish) {
        double x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = r + i * kFinish < partials ? partial[r + i * kFinish] : 0.;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += x[i];
    }
    s = block_sum<kFinish / 64>(s, part);
    if (threadIdx.x == 0) *norm = (float)sqrt(s);
}

__device__ Plan plan_of(const AdamwStep &a) {
    Plan p;
    const double norm = a.grad_norm ? (double)*a.grad_norm : 0.;
    p.clip = a.max_grad_norm > 0. ? (float)(norm <= a.max_grad_norm ? 1. : a.max_grad_norm / norm) : 1.f;
    p.skip = a.skip_nonfinite && !(norm <= 3.402823466e38);
    // (the upper half counts workgroups while a step is under way, see below)
    const uint32_t t = (uint32_t)__hip_atomic_load(a.step, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1;
    const double lr = a.lr_device ? (double)*a.lr_device : a.lr;
    p.decay = (float)(1. - lr * a.weight_decay);
    p.rate = (float)(lr / -expm1((double)t * a.log_beta1));
    p.root = (float)(1. / sqrt(-expm1((double)t * a.log_beta2)));
    p.key = a.seed * 0x9E3779B9u + t * 0xBB67AE85u;
    return p;
}

// The largest of 32 or 64 neighbouring lanes' magnitudes; NaN if one is.
template <int kLanes> __device__ __forceinline__ float top_of(float v) {
    uint32_t b = __float_as_uint(v);
    b = max(b, (uint32_t)__builtin_amdgcn_mov_dpp((int)b, 0xB1, 0xF, 0xF, true));    // quad_perm [1,0,3,2]
    b = max(b, (uint32_t)__builtin_amdgcn_mov_dpp((int)b, 0x4E, 0xF, 0xF, true));    // quad_perm [2,3,0,1]
    b = max(b, (uint32_t)__builtin_amdgcn_mov_dpp((int)b, 0x141, 0xF, 0xF, true));   // row_half_mirror
    b = max(b, (uint32_t)__builtin_amdgcn_mov_dpp((int)b, 0x140, 0xF, 0xF, true));   // row_mirror
    b = max(b, (uint32_t)__shfl_xor((int)b, 16));
    if (kLanes == 64) b = max(b, (uint32_t)__shfl_xor((int)b, 32));
    return __uint_as_float(b);
}

// The float8 below or above |x|, above with the probability that keeps the mean.  2^-120 brings the exponents of the two formats together,
// below float8's smallest normal number too: what float8 holds are the upper bits, the random number rounds by its carry.
__device__ __forceinline__ uint32_t to_float8(float x, uint32_t random16) {
    return min((__float_as_uint(fabsf(x) * 0x1p-120f) + (random16 << 4)) >> 20, 0x7Eu);
}

// The square root rounded to the nearest, of anything from 2^-96 on (below, to one unit in the last place): the instruction's is off by one unit at
// most, and the sign of x - s t for it and a neighbour t says which one is nearer.
__device__ __forceinline__ float root_of(float x) {
    const float s = __builtin_amdgcn_sqrtf(x);
    const float below = __uint_as_float(__float_as_uint(s) - 1), above = __uint_as_float(__float_as_uint(s) + 1);
    const float r = __builtin_fmaf(-below, s, x) <= 0.f ? below : s;
    return __builtin_fmaf(-above, s, x) > 0.f ? above : r;
}

__device__ __forceinline__ void new_moments32(float g, float &m, float &v, float &root, const Rates &r, float clip) {
    g *= clip;
    m = m * r.b1 + g * r.c1;
    v = v * r.b2 + g * g * r.c2;
    root = __builtin_amdgcn_sqrtf(v);
}
// Moments that will be held in 8 bits: every product, sum and root is rounded by itself, to the nearest.  Where one lies next to a value of float8
// the last bit decides which one it becomes, and the next step starts from there: so the result is that of the formula's operations
// in fp32, one after the other, and not of what a compiler joins.
__device__ __forceinline__ void new_moments8(float g, float &m, float &v, float &root, float2 scale, const Rates &r, float clip) {
#pragma clang fp contract(off)
    g *= clip;
    const float m0 = m * scale.x, r0 = v * scale.y;
    m = m0 * r.b1 + g * r.c1;
    v = r0 * r0 * r.b2 + g * g * r.c2;
    root = root_of(v);
}

template <typename T, int kBits, bool kMaster, bool kPast>
__device__ __forceinline__ void step_chunk(const AdamwTensor &t, const Rates &r, const Plan &q, uint32_t key, int64_t first) {
    typedef std::conditional_t<kBits == 8, uint8_t, float> M;
    // Neighbouring lanes' pieces lie next to each other, so what one load of a wave reaches has no gaps if a piece has at most 16 bytes: pieces of
    // 4 elements where there is something in fp32 (AdamW over 490 M fp32 parameters 2.84 ms with pieces of 8)
    constexpr int kEach = kBits == 8 && sizeof(T) == 2 && !kMaster ? 8 : 4, kItems = kChunk / kThreads / kEach;
    Piece<T, kEach> g8[kItems], p8[kItems];
    Piece<M, kEach> m8[kItems], v8[kItems];
    Piece<float, kEach> w8[kMaster ? kItems : 1];
    float2 scale[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        const int64_t at = first + (i * kThreads + (int)threadIdx.x) * kEach;
        const int n = (int)min((int64_t)kEach, t.numel - at);
        g8[i].template load<kPast>(static_cast<const T *>(t.grad) + at, n);
        if (kMaster) w8[i].template load<kPast>(t.master + at, n);
        else p8[i].template load<kPast>(static_cast<const T *>(t.param) + at, n);
        m8[i].template load<kPast>(static_cast<const M *>(t.exp_avg) + at, n);
        v8[i].template load<kPast>(static_cast<const M *>(t.exp_avg_sq) + at, n);
        if (kBits == 8) scale[i] = n > 0 ? *reinterpret_cast<const float2 *>(t.scales + 2 * (at / kScaleBlock)) : make_float2(0.f, 0.f);
    }
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        const int64_t at = first + (i * kThreads + (int)threadIdx.x) * kEach;
        const int n = (int)min((int64_t)kEach, t.numel - at);
        float g[kEach], w[kEach], m[kEach], v[kEach], root[kEach];
        unpack(g8[i], g);
        unpack(m8[i], m);
        unpack(v8[i], v);
        if constexpr (kMaster) unpack(w8[i], w);
        else unpack(p8[i], w);
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            if constexpr (kBits == 8) new_moments8(g[e], m[e], v[e], root[e], scale[i], r, q.clip);
            else new_moments32(g[e], m[e], v[e], root[e], r, q.clip);
            // (root and reciprocal to one unit in the last place of fp32; correctly rounded ones take some twenty operations more)
            w[e] = w[e] * q.decay - m[e] * q.rate * __builtin_amdgcn_rcpf(root[e] * q.root + r.eps);
        }
        if constexpr (kMaster) {
            pack(w, w8[i]);
            w8[i].template store<kPast>(t.master + at, n);
        }
        pack(w, p8[i]);
        p8[i].template store<kPast>(static_cast<T *>(t.param) + at, n);
        if constexpr (kBits == 8) {
            float top_m = 0.f, top_r = 0.f;
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                // (as bits: NaN is the largest; elements behind the tensor's end were loaded as zeros and stay zeros)
                top_m = __uint_as_float(max(__float_as_uint(top_m), __float_as_uint(m[e]) & 0x7fffffffu));
                top_r = __uint_as_float(max(__float_as_uint(top_r), __float_as_uint(root[e])));
            }
            top_m = top_of<kScaleBlock / kEach>(top_m), top_r = top_of<kScaleBlock / kEach>(top_r);
            const float sm = top_m < 0x1p-100f ? 0x1p-100f : top_m, sr = top_r < 0x1p-100f ? 0x1p-100f : top_r;
            if (threadIdx.x % (kScaleBlock / kEach) == 0 && n > 0)
                *reinterpret_cast<float2 *>(t.scales + 2 * (at / kScaleBlock)) = make_float2(sm * (1.f / 448.f), sr * (1.f / 448.f));
            const float im = 1.f / sm * 448.f, ir = 1.f / sr * 448.f;
            const uint32_t start = (uint32_t)at * 0x9E3779B9u + key;
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                const uint32_t h = mix(start + (uint32_t)e * 0x9E3779B9u);
                const uint32_t cm = to_float8(m[e] * im, h & 0xFFFF) | (__float_as_uint(m[e]) >> 24 & 0x80u);
                uint32_t cr = to_float8(root[e] * ir, h >> 16);
                cr = root[e] > 0.f ? max(cr, 1u) : cr;   // (a denominator is never rounded to zero)
                if (e % 4 == 0) m8[i].r[e / 4] = cm, v8[i].r[e / 4] = cr;
                else m8[i].r[e / 4] |= cm << (8 * (e % 4)), v8[i].r[e / 4] |= cr << (8 * (e % 4));
            }
        } else {
            pack(m, m8[i]);
            pack(v, v8[i]);
        }
        m8[i].template store<kPast>(static_cast<M *>(t.exp_avg) + at, n);
        v8[i].template store<kPast>(static_cast<M *>(t.exp_avg_sq) + at, n);
    }
}

// kMaster: some tensor has a master.
template <typename T, int kBits, bool kMaster, bool kPast>
__global__ __launch_bounds__(kThreads) void step_kernel(Group g, Rates r, AdamwStep a) {
    __shared__ Plan plan;
    if (threadIdx.x == 0) plan = plan_of(a);
    __syncthreads();
    const Plan q = plan;
    if (q.skip) return;
    for (int chunk = blockIdx.x; chunk < g.first[g.count]; chunk += gridDim.x) {
        const int k = tensor_of(g, chunk);
        const AdamwTensor t = g.t[k];
        const uint32_t key = mix(q.key + (uint32_t)(g.number + k));
        const int64_t first = (int64_t)(chunk - g.first[k]) * kChunk;
        if (kMaster && t.master) step_chunk<T, kBits, kMaster, kPast>(t, r, q, key, first);
        else step_chunk<T, kBits, false, kPast>(t, r, q, key, first);
    }
    // The step count moves on when the last workgroup has read it: the workgroups that have are counted in its upper half.
    if (!g.last || threadIdx.x != 0) return;
    auto *step = reinterpret_cast<unsigned long long *>(a.step);
    const unsigned long long was = __hip_atomic_fetch_add(step, 1ull << 32, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (was >> 32 == gridDim.x - 1) __hip_atomic_store(step, (was & 0xffffffffull) + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The tensors in groups that one launch takes: f(group, workgroups).  At least one group, also where there is nothing in any tensor.
template <typename F> void by_group(int64_t count, const AdamwTensor *tensors, F &&f) {
    Group g;
    for (int64_t at = 0;;) {
        g.number = (int)at;
        g.first[0] = 0;
        for (g.count = 0; g.count < kGroup && at < count; ++g.count, ++at) {
            const int64_t chunks = (tensors[at].numel + kChunk - 1) / kChunk;
            if (g.first[g.count] + chunks > 0x3fffffff) break;   // (chunks are numbered in 32 bits; one tensor has at most 2^28)
            g.t[g.count] = tensors[at];
            g.first[g.count + 1] = g.first[g.count] + (int)chunks;
        }
        g.last = at >= count;
        const int chunks = g.first[g.count];
        if (chunks > 0 || g.last) f(g, chunks < 1 ? 1 : chunks < kBlocks ? chunks : kBlocks);
        if (g.last) return;
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
    return (size_t)(2 * ((count + kGroup - 1) / kGroup)) * kBlocks * sizeof(double);
}

hipError_t grad_norm(hipStream_t st, int dtype, int64_t count, const AdamwTensor *tensors, float *norm, void *workspace) {
    return by_type(dtype, [&](auto t) {
        double *partial = static_cast<double *>(workspace);
        int64_t partials = 0;
        by_group(count, tensors, [&](const Group &g, int blocks) {
            hipLaunchKernelGGL((norm_kernel<decltype(t)>), dim3(blocks), dim3(kThreads), 0, st, g, partial + partials);
            partials += blocks;
        });
        hipLaunchKernelGGL(norm_finish_kernel, dim3(1), dim3(kFinish), 0, st, partial, partials, norm);
    });
}

hipError_t adamw_step(hipStream_t st, int dtype, int moment_bits, int64_t count, const AdamwTensor *tensors, const AdamwStep &s) {
    const Rates r{(float)s.beta1, (float)(1. - s.beta1), (float)s.beta2, (float)(1. - s.beta2), (float)s.eps};
    AdamwStep a = s;
    a.log_beta1 = log(s.beta1), a.log_beta2 = log(s.beta2);   // (of 0: -inf, and the power 0)
    int64_t bytes = 0;
    bool master = false;
    for (int64_t i = 0; i < count; ++i) {
        bytes += tensors[i].numel * ((dtype == kF32 ? 4 : 2) * 2 + moment_bits / 4 + (tensors[i].master ? 4 : 0));
        master |= tensors[i].master != nullptr;
    }
    return by_type(dtype, [&](auto t) {
        either(moment_bits == 8, [&](auto eight) {
            either(master, [&](auto any) {
                either(bytes >= kPastBytes, [&](auto past) {
                    by_group(count, tensors, [&](const Group &g, int blocks) {
                        hipLaunchKernelGGL((step_kernel<decltype(t), eight.value ? 8 : 32, any.value, past.value>), dim3(blocks), dim3(kThreads), 0, st, g, r, a);
                    });
                });
            });
        });
    });
}

}  // namespace wkv6
