// Norm over a token's channels, with the residual addition before it, and its gradients.
//
//   s = x + add  (rounded to x's type: what the layers after this one see),   m = mean(s),   q = 1 / sqrt(mean((s - m)^2) + eps)
//   y = (s - m) q w + b
//   backward, with h = (s - m) q and g' = g w:  ds = q (g' - mean(g') - h mean(g' h)) + what arrives at s,   dw = sum over tokens of g h,   db = sum of g
//
// A row is held in registers, by a wave up to 16 channels to a lane, by 256 to 1024 threads beyond: it is read once, and the squares are of differences from the mean
// that is already known (a sum of squares less the square of the sum loses what is small beside the mean).  Sums are fp32 within a row; those over
// rows are fp32 within the rows that a wave takes one after the other, fp64 over the workgroups, always in the same order.
//
// Bound by memory: 8192 rows of 2048, stream in fp32, branches in bf16, with the addition 37 us forward and 46 backward (5.4 and 5.8 TB/s, some of it in the
// caches), the sums over rows 5 more; 32768 rows of 4096 bf16 192 and 214 us (5.6 and 5.0 TB/s; a copy runs at 5.1).  Reading or writing past the caches: the same
// forward, 5 to 15 % slower backward.  One row of 2048: a launch of 4 us.
#include "wkv6_common.h"
#include "wkv6_kernels.h"
#include "wkv6_pieces.h"

namespace wkv6 {
namespace {

constexpr int kThreads = 256;
constexpr int kFinish = 1024;
constexpr int64_t kMostBlocks = 1 << 20;   // of a launch, whose threads are counted in 32 bits

template <int kT> __device__ __forceinline__ float row_sum(float v, float *part) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    if (kT == 64) return v;
    __syncthreads();   // (the last sum has been read)
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int i = 1; i < kT / 64; ++i) v += part[i];
    return v;
}

// Elements of a row from `at` on that a piece of kE there has, or more.  kWhole: rows are whole pieces, without the code for single elements.
template <int kE, bool kWhole> __device__ __forceinline__ int left(int C, int at) { return !kWhole ? C - at : at < C ? kE : 0; }

// kE of the weights or biases, of type kBF16, kF16 or kF32, as fp32; `none` where there are none.
template <int kE> __device__ __forceinline__ void load_params(const void *p, int type, int at, int n, float none, float (&o)[kE]) {
    if (!p) {
#pragma unroll
        for (int e = 0; e < kE; ++e) o[e] = none;
    } else if (type == kF32) {
        Piece<float, kE> b;
        b.template load<false>(static_cast<const float *>(p) + at, n);
        unpack(b, o);
    } else if (type == kBF16) {
        Piece<bf16_t, kE> b;
        b.template load<false>(static_cast<const bf16_t *>(p) + at, n);
        unpack(b, o);
    } else {
        Piece<f16_t, kE> b;
        b.template load<false>(static_cast<const f16_t *>(p) + at, n);
        unpack(b, o);
    }
}

template <typename S, typename Y, int kT, int kVecs, bool kWhole>
__global__ __launch_bounds__(kT == 64 ? kThreads : kT) void norm_kernel(NormArgs a, int64_t first_block) {
    constexpr int kE = 16 / sizeof(S), kRows = kT == 64 ? kThreads / 64 : 1;
    __shared__ float part[kT / 64];
    const int C = (int)a.C, tid = threadIdx.x % kT;
    const int64_t block = first_block + blockIdx.x, row = kT == 64 ? block * kRows + __builtin_amdgcn_readfirstlane(threadIdx.x / 64) : block;
    if (kT == 64 && row >= a.rows) return;
    const S *x = static_cast<const S *>(a.x) + row * a.x_stride;
    const Y *add = static_cast<const Y *>(a.add) + row * a.add_stride;
    Piece<S, kE> xs[kVecs];
    Piece<Y, kE> as[kVecs];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) xs[i].template load<false>(x + (i * kT + tid) * kE, left<kE, kWhole>(C, (i * kT + tid) * kE));
    if (a.add) {
#pragma unroll
        for (int i = 0; i < kVecs; ++i) as[i].template load<false>(add + (i * kT + tid) * kE, left<kE, kWhole>(C, (i * kT + tid) * kE));
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            float v[kE], w[kE];
            unpack(xs[i], v);
            unpack(as[i], w);
#pragma unroll
            for (int e = 0; e < kE; ++e) v[e] += w[e];
            pack(v, xs[i]);
            xs[i].template store<false>(static_cast<S *>(a.total) + row * C + (i * kT + tid) * kE, left<kE, kWhole>(C, (i * kT + tid) * kE));
        }
    }
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        float v[kE];
        unpack(xs[i], v);   // (zero behind the row's end)
#pragma unroll
        for (int e = 0; e < kE; ++e) sum += v[e];
    }
    const float mean = row_sum<kT>(sum, part) / (float)C;
    float squares = 0.f;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        float v[kE];
        unpack(xs[i], v);
#pragma unroll
        for (int e = 0; e < kE; ++e) {
            const float d = (i * kT + tid) * kE + e < C ? v[e] - mean : 0.f;
            squares += d * d;
        }
    }
    const float rstd = 1.f / sqrtf(row_sum<kT>(squares, part) / (float)C + a.eps);
    if (tid == 0 && a.stats) *reinterpret_cast<float2 *>(a.stats + 2 * row) = make_float2(mean, rstd);
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        const int at = (i * kT + tid) * kE;
        float v[kE], w[kE], b[kE];
        load_params<kE>(a.weight, a.param_type, at, left<kE, kWhole>(C, at), 1.f, w);
        load_params<kE>(a.bias, a.param_type, at, left<kE, kWhole>(C, at), 0.f, b);
        unpack(xs[i], v);
#pragma unroll
        for (int e = 0; e < kE; ++e) v[e] = (v[e] - mean) * rstd * w[e] + b[e];
        Piece<Y, kE> y;
        pack(v, y);
        y.template store<false>(static_cast<Y *>(a.y) + row * C + at, left<kE, kWhole>(C, at));
    }
}

template <typename S, typename Y, int kT, int kVecs, bool kWhole>
__global__ __launch_bounds__(kT == 64 ? kThreads : kT) void norm_backward_kernel(NormGrad a, float *partial) {
    constexpr int kE = 16 / sizeof(S), kRows = kT == 64 ? kThreads / 64 : 1;
    __shared__ float part[kT / 64];
    const int C = (int)a.C, tid = threadIdx.x % kT, wave = kT == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x / 64) : 0;
    float dw[kVecs][kE], db[kVecs][kE], w[kVecs][kE];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        const int at = (i * kT + tid) * kE;
        load_params<kE>(a.weight, a.param_type, at, left<kE, kWhole>(C, at), 1.f, w[i]);
#pragma unroll
        for (int e = 0; e < kE; ++e) dw[i][e] = db[i][e] = 0.f;
    }
    const float over = 1.f / (float)C;
    for (int64_t row = (int64_t)blockIdx.x * kRows + wave; row < a.rows; row += (int64_t)gridDim.x * kRows) {
        const S *s = static_cast<const S *>(a.total) + row * a.total_stride;
        const Y *gy = static_cast<const Y *>(a.gy) + row * C;
        Piece<S, kE> ss[kVecs], ts[kVecs];
        Piece<Y, kE> gs[kVecs];
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            const int at = (i * kT + tid) * kE;
            ss[i].template load<false>(s + at, left<kE, kWhole>(C, at));
            gs[i].template load<false>(gy + at, left<kE, kWhole>(C, at));
        }
        if (a.gtotal) {
#pragma unroll
            for (int i = 0; i < kVecs; ++i) {
                const int at = (i * kT + tid) * kE;
                ts[i].template load<false>(static_cast<const S *>(a.gtotal) + row * C + at, left<kE, kWhole>(C, at));
            }
        }
        const float2 stats = *reinterpret_cast<const float2 *>(a.stats + 2 * row);
        const float mean = stats.x, rstd = stats.y;
        float sum = 0.f, dot = 0.f;
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            float v[kE], g[kE];
            unpack(ss[i], v);
            unpack(gs[i], g);   // (zero behind the row's end)
#pragma unroll
            for (int e = 0; e < kE; ++e) {
                const bool in = (i * kT + tid) * kE + e < C;
                const float h = in ? (v[e] - mean) * rstd : 0.f, gw = in ? g[e] * w[i][e] : 0.f;
                dw[i][e] += g[e] * h;
                db[i][e] += g[e];
                sum += gw;
                dot += gw * h;
            }
        }
        sum = row_sum<kT>(sum, part) * over;
        dot = row_sum<kT>(dot, part) * over;
        if (!a.gx && !a.gadd) continue;
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            const int at = (i * kT + tid) * kE;
            float v[kE], g[kE], t[kE];
            unpack(ss[i], v);
            unpack(gs[i], g);
            if (a.gtotal) unpack(ts[i], t);
#pragma unroll
            for (int e = 0; e < kE; ++e) {
                const float h = (v[e] - mean) * rstd;
                v[e] = rstd * (g[e] * w[i][e] - sum - h * dot);
                if (a.gtotal) v[e] += t[e];
            }
            if (a.gx) {
                Piece<S, kE> o;
                pack(v, o);
                o.template store<false>(static_cast<S *>(a.gx) + row * C + at, left<kE, kWhole>(C, at));
            }
            if (a.gadd) {
                Piece<Y, kE> o;
                pack(v, o);
                o.template store<false>(static_cast<Y *>(a.gadd) + row * C + at, left<kE, kWhole>(C, at));
            }
        }
    }
    if (!partial) return;
    float *out = partial + (int64_t)blockIdx.x * 2 * C;
    if constexpr (kT == 64) {
        extern __shared__ float sums[];   // of the four waves
#pragma unroll
        for (int i = 0; i < kVecs; ++i)
#pragma unroll
            for (int e = 0; e < kE; ++e) {
                const int at = (i * 64 + tid) * kE + e;
                if (at < C) sums[wave * 2 * C + at] = dw[i][e], sums[wave * 2 * C + C + at] = db[i][e];
            }
        __syncthreads();
        for (int at = threadIdx.x; at < 2 * C; at += kThreads) {
            float v = sums[at];
#pragma unroll
            for (int k = 1; k < kRows; ++k) v += sums[k * 2 * C + at];
            out[at] = v;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kVecs; ++i)
#pragma unroll
            for (int e = 0; e < kE; ++e) {
                const int at = (i * kT + tid) * kE + e;
                if (at < C) out[at] = dw[i][e], out[C + at] = db[i][e];
            }
    }
}

__device__ __forceinline__ void store_param(void *p, int type, int64_t at, float v) {
    if (type == kF32) store1(static_cast<float *>(p) + at, v);
    else if (type == kBF16) store1(static_cast<bf16_t *>(p) + at, v);
    else store1(static_cast<f16_t *>(p) + at, v);
}

// The sums over workgroups of 64 columns of (weight's gradient, bias's gradient): 4 columns to a lane, 64 workgroups' sums at a time.
__global__ __launch_bounds__(kFinish) void norm_finish_kernel(NormGrad a, const float *partial, int blocks) {
    constexpr int kW = kFinish / 64, kAtOnce = 4, kEach = 4;
    __shared__ double part[kW][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t width = 2 * a.C, column = (int64_t)blockIdx.x * 64 + lane % 16 * kEach;
    const int n = (int)min(width - column, (int64_t)kEach);
    double s[kEach] = {};
    for (int first = wave * 4 + lane / 16; first < blocks; first += kAtOnce * kW * 4) {
        Piece<float, kEach> b[kAtOnce];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            const int row = first + k * kW * 4;
            b[k].template load<false>(partial + min(row, blocks - 1) * width + column, row < blocks ? n : 0);
        }
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            float v[kEach];
            unpack(b[k], v);
#pragma unroll
            for (int e = 0; e < kEach; ++e) s[e] += v[e];
        }
    }
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        s[e] += __shfl_xor(s[e], 16);
        s[e] += __shfl_xor(s[e], 32);
        if (lane < 16) part[wave][lane * kEach + e] = s[e];
    }
    __syncthreads();
    const int64_t mine = (int64_t)blockIdx.x * 64 + threadIdx.x;
    if (threadIdx.x >= 64 || mine >= width) return;
    double sum = 0.;
    for (int i = 0; i < kW; ++i) sum += part[i][threadIdx.x];
    void *out = mine < a.C ? a.gweight : a.gbias;
    if (out) store_param(out, a.param_type, mine < a.C ? mine : mine - a.C, (float)sum);
}

template <int T, int V, bool W> struct Shape {
    static constexpr int threads = T, vecs = V;
    static constexpr bool whole = W;
};

// By the number of channels: threads that a row is spread over, and 16-byte pieces of the stream's type to a thread.  (Few to a thread: the backward's sums and the
// weights take three registers a channel.  8192 rows of 2048, a stream in fp32 and branches in bf16,
// backward, in us: 64 threads to a row 61 to 74, 128 49, 256 47.)
template <int kE, bool kWhole, typename F> void by_width(int64_t C, F &&f) {
    if (C <= 64 * 8) f(Shape<64, 8 / kE, kWhole>{});
    else if (C <= 64 * 16) f(Shape<64, 16 / kE, kWhole>{});
    else if (C <= 256 * 8) f(Shape<256, 8 / kE, kWhole>{});
    else if (C <= 256 * 16) f(Shape<256, 16 / kE, kWhole>{});
    else if (C <= 256 * 32) f(Shape<256, 32 / kE, kWhole>{});
    else if (C <= 512 * 32) f(Shape<512, 32 / kE, kWhole>{});
    else f(Shape<1024, 32 / kE, kWhole>{});
}
template <typename S, typename F> void by_width(int64_t C, F &&f) {
    constexpr int kE = 16 / sizeof(S);
    if (C % kE == 0) by_width<kE, true>(C, f);
    else by_width<kE, false>(C, f);
}

// The types of the stream and of the branches, what is added to it and what comes out: one, or a stream in fp32 with branches in 16 bits.
template <typename F> hipError_t by_types(int stream, int branch, F &&f) {
    if (stream == kBF16) f(bf16_t{}, bf16_t{});
    else if (stream == kF16) f(f16_t{}, f16_t{});
    else if (branch == kF32) f(float{}, float{});
    else if (branch == kBF16) f(float{}, bf16_t{});
    else f(float{}, f16_t{});
    return hipGetLastError();
}

// Two workgroups to a compute unit at most: each leaves 2 C sums in the workspace, which another launch adds up.
int backward_blocks(int64_t rows, int64_t C) {
    const int64_t at_once = C <= 64 * 16 ? kThreads / 64 : 1, all = (rows + at_once - 1) / at_once;
    return (int)(all < 512 ? all : 512);
}

}  // namespace

hipError_t layer_norm(hipStream_t st, int dtype, int branch_dtype, const NormArgs &a) {
    return by_types(dtype, branch_dtype, [&](auto s, auto y) {
        by_width<decltype(s)>(a.C, [&](auto shape) {
            constexpr int kT = decltype(shape)::threads;
            const int64_t blocks = kT == 64 ? (a.rows + kThreads / 64 - 1) / (kThreads / 64) : a.rows;
            for (int64_t first = 0; first < blocks; first += kMostBlocks)
                hipLaunchKernelGGL((norm_kernel<decltype(s), decltype(y), kT, decltype(shape)::vecs, decltype(shape)::whole>),
                                   dim3((unsigned)(blocks - first < kMostBlocks ? blocks - first : kMostBlocks)), dim3(kT == 64 ? kThreads : kT), 0, st, a, first);
        });
    });
}

size_t layer_norm_backward_workspace_bytes(int64_t rows, int64_t C) { return (size_t)backward_blocks(rows, C) * 2 * C * sizeof(float); }

hipError_t layer_norm_backward(hipStream_t st, int dtype, int branch_dtype, const NormGrad &a, void *workspace) {
    const bool params = a.gweight || a.gbias;
    float *partial = params ? static_cast<float *>(workspace) : nullptr;
    const int blocks = backward_blocks(a.rows, a.C);
    const hipError_t e = by_types(dtype, branch_dtype, [&](auto s, auto y) {
        by_width<decltype(s)>(a.C, [&](auto shape) {
            constexpr int kT = decltype(shape)::threads;
            hipLaunchKernelGGL((norm_backward_kernel<decltype(s), decltype(y), kT, decltype(shape)::vecs, decltype(shape)::whole>), dim3(blocks),
                               dim3(kT == 64 ? kThreads : kT), kT == 64 ? kThreads / 64 * 2 * a.C * sizeof(float) : 0, st, a, partial);
        });
    });
    if (e != hipSuccess || !params) return e;
    hipLaunchKernelGGL(norm_finish_kernel, dim3((unsigned)((2 * a.C + 63) / 64)), dim3(kFinish), 0, st, a, partial, blocks);
    return hipGetLastError();
}

}  // namespace wkv6
