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
// No sum depends on an order that changes from run to run: terms of rows are added up in 64 bits, in stretches of rows that depend on their number alone.
//
// Bound by memory.  A loss whose c is known when a row's sums are (cross entropy, the clipped policy loss) reads a row once, into registers, and
// writes its gradient from there: two passes over the logits instead of three (8192 rows of 65536 bf16: 390 us, 5.5 TB/s, where copying as
// much takes 432).  The preference loss's c needs both whole texts, so its gradient reads the logits again (16 x 1024 rows: 955 us, 5.6 TB/s of three
// passes; grouping the pairs so that the second reading might find them in the last-level cache, with the next pairs' rows in the same launch or
// in one of their own, took as long).  Sums alone reach 6.2 to 7 TB/s (8192 rows of 65536 bf16, three quarters of which count: 134 us).
#include "wkv6_common.h"
#include "wkv6_kernels.h"

#include <type_traits>

namespace wkv6 {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kFinish = 1024;        // threads of the one workgroup that adds up
constexpr int kCountBlocks = 256;    // at most
constexpr int kStretches = 256;      // of a great many rows
// Of up to so many rows every row's threads count the tokens for themselves, a launch less; beyond, each row's reading of all ids takes longer than the launch.  All
// kernels of a cross entropy over V 1000, in us, counted by the rows / ahead: 64 rows 10.2 / 14.2, 512 12.2 / 14.2, 1024 14.6 / 14.4 (and the host's 2 us for a launch), 2048
// 19.5 / 15.6, 8192 71 / 23.
constexpr int kFewRows = 1024;
constexpr int64_t kMostBlocks = 1 << 21;   // of a launch: it counts its threads in 32 bits
constexpr int kGradVecs = 8;         // vectors of a thread in the gradient's own pass
// A gradient of this size and more is written past the caches.  Cross entropy, log probabilities with their backward, and the latter with a reader
// of the gradient behind it, in us, written into / past them: 128 MiB 63 / 66, 78 / 78, 106 / 120; 192 MiB 89 / 89, 119 / 108, 178 / 171; 2 GiB (8 pairs
// of texts) 1110 / 1000.
constexpr int64_t kPastBytes = 160 << 20;
constexpr double kLog2e = 1.44269504088896340736;

// exp(d / temperature) as a power of two.  (1 / temperature is in 64 bits, here and in lp.)  log2(e) / temperature rounded to fp32 is off by up to 2^-24 of itself, the same way in
// every element: lp would be off by as much times the mean of d, over a whole text hundreds of times that.  `low` is what the
// rounding left; the gradient, whose elements are rounded one by one, does without.  (`high` is rounded down and `low` positive: with d = -inf
// the two products are -inf both, and not two infinities of different signs.)
struct Scale {
    float high, low;
    __device__ __forceinline__ explicit Scale(double inv_temperature) {
        const double s = kLog2e * inv_temperature;
        high = (float)s;
        if ((double)high >= s) high = __uint_as_float(__float_as_uint(high) - 1);
        low = fmaxf((float)(s - high), 0x1p-149f);
    }
    __device__ __forceinline__ float exp(float d) const { return __builtin_amdgcn_exp2f(__builtin_fmaf(d, high, d * low)); }
    __device__ __forceinline__ float exp_once(float d) const { return __builtin_amdgcn_exp2f(d * high); }
};

// 16 bytes of a row as they sit in memory, at any element's address.
template <typename T> struct Vec;
template <> struct Vec<bf16_t> {
    typedef uint32_t raw __attribute__((ext_vector_type(4), aligned(2)));
    static constexpr int kN = 8;
    static constexpr uint32_t kNone = 0xFF80FF80u;   // -inf
    static __device__ __forceinline__ void unpack(const uint32_t (&r)[4], float (&o)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) o[2 * i] = __uint_as_float(r[i] << 16), o[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
    }
    static __device__ __forceinline__ void pack(const float (&v)[8], uint32_t (&r)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
    }
};
template <> struct Vec<f16_t> {
    typedef uint32_t raw __attribute__((ext_vector_type(4), aligned(2)));
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    static constexpr int kN = 8;
    static constexpr uint32_t kNone = 0xFC00FC00u;
    static __device__ __forceinline__ void unpack(const uint32_t (&r)[4], float (&o)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const h2 h = __builtin_bit_cast(h2, r[i]);
            o[2 * i] = (float)h[0], o[2 * i + 1] = (float)h[1];
        }
    }
    static __device__ __forceinline__ void pack(const float (&v)[8], uint32_t (&r)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = __builtin_bit_cast(uint32_t, (h2){to_f16(v[2 * i]), to_f16(v[2 * i + 1])});
    }
};
template <> struct Vec<float> {
    typedef uint32_t raw __attribute__((ext_vector_type(4), aligned(4)));
    static constexpr int kN = 4;
    static constexpr uint32_t kNone = 0xFF800000u;
    static __device__ __forceinline__ void unpack(const uint32_t (&r)[4], float (&o)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = __uint_as_float(r[i]);
    }
    static __device__ __forceinline__ void pack(const float (&v)[4], uint32_t (&r)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = __float_as_uint(v[i]);
    }
};
template <typename T> struct Bits {
    uint32_t r[4];
    // kPast: past the caches
    template <bool kPast> __device__ __forceinline__ void load(const T *p) {
        typename Vec<T>::raw v;
        if (kPast) v = __builtin_nontemporal_load(reinterpret_cast<const typename Vec<T>::raw *>(p));
        else v = *reinterpret_cast<const typename Vec<T>::raw *>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = v[i];
    }
    // Keeps the compiler from holding the unpacked values of one pass over the registers for the next, at twice the registers.
    __device__ __forceinline__ void again() {
#pragma unroll
        for (int i = 0; i < 4; ++i) asm("" : "+v"(r[i]));
    }
    __device__ __forceinline__ void none() { r[0] = r[1] = r[2] = r[3] = Vec<T>::kNone; }
    __device__ __forceinline__ void zero() { r[0] = r[1] = r[2] = r[3] = 0; }
    template <bool kPast> __device__ __forceinline__ void store(T *p) const {
        typename Vec<T>::raw v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = r[i];
        if (kPast) __builtin_nontemporal_store(v, reinterpret_cast<typename Vec<T>::raw *>(p));
        else *reinterpret_cast<typename Vec<T>::raw *>(p) = v;
    }
};

// How a row of V elements is taken: `full` vectors from its first 16-byte boundary on (loads across such boundaries are allowed, but slower: cross
// entropy of 10682 rows of 50257 bf16 488 us with them, 410 without), and up to 14 single elements before and behind, one to a thread.
template <typename T> struct Cut {
    int head, full, singles;
    __device__ __forceinline__ Cut(const T *x, int V) {
        head = min(V, (int)((16 - reinterpret_cast<uintptr_t>(x) % 16) % 16 / sizeof(T)));
        full = (V - head) / Vec<T>::kN;
        singles = V - full * Vec<T>::kN;
    }
    __device__ __forceinline__ int single(int i) const { return i < head ? i : full * Vec<T>::kN + i; }
    // whether element id is a single one, and which; or its vector
    __device__ __forceinline__ int single_of(int id) const { return id < head ? id : id >= head + full * Vec<T>::kN ? id - full * Vec<T>::kN : -1; }
    __device__ __forceinline__ int vector_of(int id) const { return (id - head) / Vec<T>::kN; }
};

__device__ __forceinline__ bool counts(const LossRows &a, int64_t row, int64_t id) {
    return id >= 0 && (a.mask == nullptr || a.mask[row] != 0);
}

// A wave's folds: across neighbours within 16 lanes by DPP, then over the four rows of lanes.
template <int kCtrl> __device__ __forceinline__ float moved(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), kCtrl, 0xF, 0xF, true));
}
__device__ __forceinline__ float lane_of(float v, int lane) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane)); }
__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, moved<0xB1>(v));    // quad_perm [1,0,3,2]
    v = fmaxf(v, moved<0x4E>(v));    // quad_perm [2,3,0,1]
    v = fmaxf(v, moved<0x141>(v));   // row_half_mirror
    v = fmaxf(v, moved<0x140>(v));   // row_mirror
    return fmaxf(fmaxf(lane_of(v, 0), lane_of(v, 16)), fmaxf(lane_of(v, 32), lane_of(v, 48)));
}
__device__ __forceinline__ float wave_sum(float v) {
    v += moved<0xB1>(v);
    v += moved<0x4E>(v);
    v += moved<0x141>(v);
    v += moved<0x140>(v);
    return (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
}
template <typename S> __device__ __forceinline__ S wave_sum(S v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
// Over the workgroup, for every thread; `part`: one value per wave in LDS that nothing else is read from meanwhile.
template <int kW> __device__ __forceinline__ float block_max(float v, float *part) {
    v = wave_max(v);
    if (kW == 1) return v;
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int i = 1; i < kW; ++i) v = fmaxf(v, part[i]);
    return v;
}
template <int kW, typename S> __device__ __forceinline__ S block_sum(S v, S *part) {
    v = wave_sum(v);
    if (kW == 1) return v;
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int i = 1; i < kW; ++i) v += part[i];
    return v;
}

// Counted tokens among n, by all threads of a workgroup.  (One token after the other to a thread would wait for two loads each: four go
// together, 6 us for 8 texts of 1024 tokens before, 4 now.)
__device__ __forceinline__ int count_tokens(const LossRows &a, int64_t first, int64_t n, int *part) {
    const int64_t *ids = a.ids + first;
    const uint8_t *mask = a.mask ? a.mask + first : nullptr;
    int sum = 0;
    for (int64_t t = threadIdx.x; t < n; t += 4 * kFinish) {
        int64_t id[4];
        uint8_t m[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool in = t + i * kFinish < n;
            id[i] = in ? ids[t + i * kFinish] : -1;
            m[i] = in && mask ? mask[t + i * kFinish] : 1;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += id[i] >= 0 && m[i] != 0;
    }
    return block_sum<kFinish / 64>(sum, part);
}

// Counted tokens of each text, and in how many texts of a workgroup's there are any.
__global__ __launch_bounds__(kFinish) void count_texts_kernel(LossRows a, LossCounts c) {
    __shared__ int part[2][kFinish / 64];
    int texts = 0, turn = 0;
    for (int64_t b = blockIdx.x; b < a.B; b += gridDim.x, turn ^= 1) {
        const int n = count_tokens(a, b * a.T, a.T, part[turn]);
        if (threadIdx.x == 0) c.by_text[b] = n;
        texts += n > 0;
    }
    if (threadIdx.x == 0) c.partial[blockIdx.x] = texts;
}

// Counted tokens of all texts, a stretch of them to each workgroup.
__global__ __launch_bounds__(kFinish) void count_kernel(LossRows a, LossCounts c, int64_t stretch) {
    __shared__ int part[kFinish / 64];
    const int64_t first = blockIdx.x * stretch, end = a.B * a.T;
    const int n = count_tokens(a, first, first + stretch < end ? stretch : end - first, part);
    if (threadIdx.x == 0) c.partial[blockIdx.x] = n;
}

// The weight of each of text b's tokens in the loss, from counts that were taken ahead.
__device__ __forceinline__ float weight_of(const LossCounts &c, int64_t b, int reduction) {
    if (reduction == kLossSum) return 1.f;
    int64_t n = 0;
    for (int i = threadIdx.x & 63; i < c.blocks; i += 64) n += c.partial[i];
    n = wave_sum(n);
    const double all = reduction == kLossMean ? (double)n : (double)n * c.by_text[b];
    return all > 0. ? (float)(1. / all) : 0.f;
}
// The same where no counts were taken: of few tokens in all, every kT threads count for themselves.
template <int kT> __device__ __forceinline__ float weight_of_few(const LossRows &a, int *part) {
    int n = 0;
    for (int t = threadIdx.x % kT; t < (int)(a.B * a.T); t += kT) n += counts(a, t, a.ids[t]);
    n = block_sum<kT / 64>(n, part);
    return n > 0 ? (float)(1. / (double)n) : 0.f;
}

// What a loss makes of one token's lp: its weighted terms, for the finishing kernel to add up, and c.
__device__ __forceinline__ float row_terms(const LossRows &a, const LossTerms &l, int64_t row, double exact, float w) {
#pragma clang fp contract(off)   // (left to itself the compiler joins other products and sums in the kernel with the gradient than in the one without)
    const int64_t rows = a.B * a.T;
    // (as this call returns it, in fp32 like the other models': a model beside its own log probabilities has ratios of 1 and a KL term of 0 to the last bit)
    const float lp = (float)exact;
    if (l.kind == kLossCrossEntropy) {
        l.terms[row] = -lp * w;
        return lp == lp ? -w : lp;
    }
    const int64_t b = row / a.T, t = row % a.T;
    const float A = l.advantages[b * l.adv_stride_b + t * l.adv_stride_t];
    const float ratio = l.old_logps ? expf(lp - l.old_logps[row]) : lp == lp ? 1.f : lp;   // (the sampling model is this one: only NaN stays NaN)
    // (exp of a finite difference that fp32 cannot hold, times an advantage of 0: 0 and no NaN)
    const bool beyond = A == 0.f && ratio == INFINITY && lp - l.old_logps[row] < INFINITY;
    const float free = beyond ? 0.f : ratio * A, held = fminf(fmaxf(ratio, 1.f - l.clip_low), 1.f + l.clip_high) * A;
    const bool clipped = free > held;
    float kl = 0.f, by_lp = clipped ? 0.f : -free;
    if (l.ref_logps) {
        const float e = l.ref_logps[row] - lp, g = expm1f(e);   // (small where the models agree: neither term is formed from 1)
        kl = g == INFINITY ? g : g - e;                         // (e may be infinite too)
        // (a weight of 0: the term is reported and takes no part, infinite as it may be)
        if (l.kl_weight != 0.f) by_lp -= l.kl_weight * g;
    }
    const float penalty = l.kl_weight != 0.f ? l.kl_weight * kl : 0.f;
    l.terms[row] = (penalty - (clipped ? held : free)) * w;
    l.terms[rows + row] = kl * w;
    l.terms[2 * rows + row] = clipped ? w : 0.f;
    return by_lp * w;
}

// f(true) or f(false), for code that is compiled for either
template <typename F> __device__ __forceinline__ void either(bool which, F &&f) {
    if (which) f(std::true_type{});
    else f(std::false_type{});
}

// Zeros over a row of the gradient.
template <typename T, int kT> __device__ __forceinline__ void zero_row(T *out, int V) {
    constexpr int kN = Vec<T>::kN;
    const Cut<T> cut(out, V);
    Bits<T> z;
    z.zero();
    for (int j = threadIdx.x % kT; j < cut.full; j += kT) z.template store<true>(out + cut.head + (int64_t)j * kN);
    if ((int)(threadIdx.x % kT) < cut.singles) store1(out + cut.single(threadIdx.x % kT), 0.f);
}

// c / temperature (1[j = id] - p_j) for one vector of a row, from its logits.
template <typename T> __device__ __forceinline__ void gradient(Bits<T> &b, const Scale &scale, float top, float minus_c_norm) {
    float v[Vec<T>::kN];
    Vec<T>::unpack(b.r, v);
#pragma unroll
    for (int e = 0; e < Vec<T>::kN; ++e) v[e] = scale.exp_once(v[e] - top) * minus_c_norm;
    Vec<T>::pack(v, b.r);
}
template <typename T> __device__ __forceinline__ float gradient(float x, const Scale &scale, float top, float minus_c_norm) {
    return scale.exp_once(x - top) * minus_c_norm;
}

// top, sum and lp of every row, and what the loss makes of it; with kGrad the gradient by the row too, while its logits are at hand.
// kT threads take a row: a workgroup, or each of a workgroup's four waves.  kHold: the row is read once, into registers (kVecs vectors of 16
// bytes to a thread); otherwise a thread goes through its part of it with a running maximum and sum, kVecs vectors at a time, and the gradient reads it
// again.  The single elements before and behind the whole vectors are one more each to the first threads.
// (Not better: one workgroup to a compute unit that loads each register's vector of the next row as soon as the gradient has left it, 494 us for 375 at
// 8192 rows of 65536 bf16 and 10 % slower beyond: two workgroups that read and compute in turn do as much, and their registers suffice.)
constexpr int waves_per_simd(int threads, int vecs) { return threads == 1024 && vecs <= 8 ? 8 : 4; }

template <typename T, int kT, int kVecs, bool kHold, bool kGrad>
__global__ __launch_bounds__(kT == 64 ? kThreads : kT, waves_per_simd(kT, kVecs)) void rows_kernel(LossRows a, LossCounts n, LossTerms l, LossGrad g, int64_t first_block) {
    constexpr int kN = Vec<T>::kN, kW = kT / 64;
    __shared__ float part_max[kW], part_sum[kW], part_c;
    __shared__ int part_n[kW];
    const int64_t block = first_block + blockIdx.x, row = kT == 64 ? block * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / 64) : block, b = row / a.T;
    if (kT == 64 && row >= a.B * a.T) return;
    const int64_t id = a.ids[row];
    const int V = (int)a.V, tid = threadIdx.x % kT;
    T *out = kGrad ? static_cast<T *>(g.grad) + row * V : nullptr;
    if (!counts(a, row, id)) {
        if (tid == 0) {
            if (a.logps) a.logps[row] = 0.f;
            if (a.exact) a.exact[row] = 0.;
            if (a.stats) a.stats[2 * row] = 0.f, a.stats[2 * row + 1] = 1.f;
            if (l.coef) l.coef[row] = 0.f;
            for (int i = 0; i < l.count; ++i) l.terms[i * a.B * a.T + row] = 0.f;
        }
        if (kGrad) zero_row<T, kT>(out, V);
        return;
    }
    // (before the row is loaded: its registers are not free later)
    const bool few = l.reduction == kLossMean && n.blocks == 0 && l.kind != kLossNone;
    float w = few ? weight_of_few<kT>(a, part_n) : 0.f;
    const T *x = static_cast<const T *>(a.logits) + b * a.stride_b + row % a.T * a.stride_t;
    const Cut<T> cut(x, V);
    const int full = cut.full;
    const T *vectors = x + cut.head;
    T *out_vectors = out + cut.head;
    const Scale scale(a.inv_temperature);
    Bits<T> held[kVecs];
    const float single = tid < cut.singles ? load1(x + cut.single(tid)) : -INFINITY;
    float top, sum;
    if (kHold) {
        either(kGrad || !a.stats, [&](auto past) {   // (read once, or once more by a backward)
#pragma unroll
            for (int i = 0; i < kVecs; ++i) {
                if (i * kT + tid < full) held[i].template load<past.value>(vectors + (int64_t)(i * kT + tid) * kN);
                else held[i].none();
            }
        });
    }
    if (!few) w = l.kind == kLossNone ? 0.f : weight_of(n, b, l.reduction);
    const float stands = id < V ? load1(x + id) : NAN;
    if (kHold) {
        top = single;
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            float v[kN];
            Vec<T>::unpack(held[i].r, v);
#pragma unroll
            for (int e = 0; e < kN; ++e) top = fmaxf(top, v[e]);
        }
        top = block_max<kW>(top, part_max);
        sum = scale.exp(single - top);
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            float v[kN];
            held[i].again();
            Vec<T>::unpack(held[i].r, v);
#pragma unroll
            for (int e = 0; e < kN; ++e) sum += scale.exp(v[e] - top);
        }
    } else {
        float mine = single;
        sum = single == -INFINITY ? 0.f : scale.exp(single - single);
        either(!kGrad && !a.stats, [&](auto past) {
            for (int first = tid; first < full; first += kVecs * kT) {
                float most = mine;
#pragma unroll
                for (int i = 0; i < kVecs; ++i) {
                    if (first + i * kT < full) held[i].template load<past.value>(vectors + (int64_t)(first + i * kT) * kN);
                    else held[i].none();
                }
#pragma unroll
                for (int i = 0; i < kVecs; ++i) {
                    float v[kN];
                    Vec<T>::unpack(held[i].r, v);
#pragma unroll
                    for (int e = 0; e < kN; ++e) most = fmaxf(most, v[e]);
                }
                const float from = most == -INFINITY ? 0.f : most;   // (-inf less -inf is no number)
                sum *= scale.exp(mine - from);
                mine = most;
#pragma unroll
                for (int i = 0; i < kVecs; ++i) {
                    float v[kN];
                    held[i].again();
                    Vec<T>::unpack(held[i].r, v);
#pragma unroll
                    for (int e = 0; e < kN; ++e) sum += scale.exp(v[e] - from);
                }
            }
        });
        top = block_max<kW>(mine, part_max);
        sum = sum == 0.f && top != -INFINITY ? 0.f : sum * scale.exp(mine - top);   // (a thread without elements)
    }
    sum = block_sum<kW>(sum, part_sum);
    float c = id < V ? -w : NAN;   // the cross entropy's: lp does not come into it
    if (tid < 64) {
        const double lp = __builtin_fma((double)(stands - top), a.inv_temperature, -log((double)sum));
        if (tid == 0) {
            if (l.kind != kLossNone) c = row_terms(a, l, row, lp, w);
            if (a.logps) a.logps[row] = (float)lp;
            if (a.exact) a.exact[row] = lp;
            if (a.stats) a.stats[2 * row] = top, a.stats[2 * row + 1] = sum;
            if (l.coef) l.coef[row] = c;
            if (kT > 64) part_c = c;
        }
    }
    if (!kGrad) return;
    if (l.kind != kLossCrossEntropy) {
        if (kT == 64) {
            c = lane_of(c, 0);
        } else {
            __syncthreads();
            c = part_c;
        }
    }
    c *= (float)a.inv_temperature;
    const float norm = 1.f / sum, factor = -c * norm;
    if (kHold) {
        either(g.past, [&](auto past) {
#pragma unroll
            for (int i = 0; i < kVecs; ++i) {
                held[i].again();
                gradient<T>(held[i], scale, top, factor);
                if (i * kT + tid < full) held[i].template store<past.value>(out_vectors + (int64_t)(i * kT + tid) * kN);
            }
        });
    } else {
        for (int first = tid; first < full; first += kVecs * kT) {
#pragma unroll
            for (int i = 0; i < kVecs; ++i)
                if (first + i * kT < full) held[i].template load<false>(vectors + (int64_t)(first + i * kT) * kN);
#pragma unroll
            for (int i = 0; i < kVecs; ++i) {
                if (first + i * kT >= full) continue;
                gradient<T>(held[i], scale, top, factor);
                held[i].template store<true>(out_vectors + (int64_t)(first + i * kT) * kN);
            }
        }
    }
    if (tid < cut.singles) store1(out + cut.single(tid), gradient<T>(single, scale, top, factor));
    // the element that stands there, by the thread whose store it was in
    if (id >= V) return;
    const int lone = cut.single_of((int)id), owner = lone >= 0 ? lone : cut.vector_of((int)id) % kT;
    if (tid == owner) store1(out + id, c + scale.exp_once(stands - top) * factor);
}

// v[first], v[first + stride], .. below `end`, added up in 64 bits, eight loads on their way at a time.
template <typename S> __device__ __forceinline__ double strided_sum(const S *v, int64_t first, int64_t end, int stride) {
    double s = 0.;
    for (int64_t r = first; r < end; r += 8 * stride) {
        S x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = r + i * stride < end ? v[r + i * stride] : S(0);
#pragma unroll
        for (int i = 0; i < 8; ++i) s += (double)x[i];
    }
    return s;
}

// The sums of up to three arrays of terms: all of an array by one workgroup, or of a great many rows a stretch by each of kStretches, into `sums`.
__global__ __launch_bounds__(kFinish) void finish_kernel(int64_t rows, LossTerms l, double *sums, int64_t stretch) {
    __shared__ double part[kFinish / 64];
    const int i = blockIdx.y;
    const int64_t first = blockIdx.x * stretch, end = first + stretch < rows ? first + stretch : rows;
    const double s = block_sum<kFinish / 64>(strided_sum(l.terms + i * rows, first + threadIdx.x, end, kFinish), part);
    if (threadIdx.x != 0) return;
    if (gridDim.x > 1) sums[i * kStretches + blockIdx.x] = s;
    else (i == 0 ? l.loss[0] : l.means[i - 1]) = (float)s;
}
__global__ __launch_bounds__(kStretches) void finish_stretches_kernel(LossTerms l, const double *sums, int stretches) {
    __shared__ double part[kStretches / 64];
    const int i = blockIdx.x;
    const double s = block_sum<kStretches / 64>((int)threadIdx.x < stretches ? sums[i * kStretches + threadIdx.x] : 0., part);
    if (threadIdx.x == 0) (i == 0 ? l.loss[0] : l.means[i - 1]) = (float)s;
}

// Pairs of texts (b and b + P), a workgroup each: log probabilities of whole texts in 64 bits (sums over thousands of tokens, of
// which a small difference is wanted), the loss of their difference, and c of either text's tokens.
__global__ __launch_bounds__(kFinish) void pairs_kernel(LossRows a, PreferenceTerms l, int64_t first_pair) {
    __shared__ double part[2][kFinish / 64];
    __shared__ int count[2][kFinish / 64];
    const int half = kFinish / 2, i = threadIdx.x / half;   // the first half of the threads takes the chosen text
    const int64_t P = a.B / 2, pair = first_pair + blockIdx.x, b = pair + i * P, first = b * a.T;
    double v = wave_sum(strided_sum(a.exact + first, threadIdx.x % half, a.T, half));
    int n = 0;
    if (l.average)
        for (int64_t t = threadIdx.x % half; t < a.T; t += half) n += counts(a, first + t, a.ids[first + t]);
    n = wave_sum(n);
    if ((threadIdx.x & 63) == 0) part[i][threadIdx.x % half / 64] = v, count[i][threadIdx.x % half / 64] = n;
    __syncthreads();
    if (threadIdx.x != 0) return;
    double s[2], len[2];
    for (int k = 0; k < 2; ++k) {
        v = 0., n = 0;
        for (int w = 0; w < half / 64; ++w) v += part[k][w], n += count[k][w];
        len[k] = n > 0 ? 1. / n : 1.;
        s[k] = v * len[k];
        l.text_logps[pair + k * P] = (float)s[k];
    }
    double d = s[0] - s[1], by_d, loss;
    if (l.ref_logps) d -= (double)l.ref_logps[pair] - (double)l.ref_logps[pair + P];
    if (l.kind == kPreferenceSigmoid) {
        const double z = l.beta * d, soft = log1p(exp(-fabs(z))), up = 1. / (1. + exp(-z));
        // (1 - e) softplus(-z) + e softplus(z)
        loss = soft + (1. - l.label_smoothing) * fmax(-z, 0.);
        if (l.label_smoothing > 0.) loss += l.label_smoothing * fmax(z, 0.);
        by_d = l.beta * (up - (1. - l.label_smoothing));
    } else if (l.kind == kPreferenceHinge) {
        const double z = 1. - l.beta * d;
        loss = z <= 0. ? 0. : z;
        by_d = z <= 0. ? 0. : z == z ? -l.beta : z;
    } else {
        const double z = d - 0.5 / l.beta;
        loss = z * z;
        by_d = 2. * z;
    }
    if (P == 1) l.loss[0] = (float)loss;
    else l.by_pair[pair] = loss / (double)P;
    if (l.coef) {
        l.coef[pair] = (float)(by_d * len[0] / (double)P);
        l.coef[pair + P] = (float)(-by_d * len[1] / (double)P);
    }
}

__global__ __launch_bounds__(kFinish) void pairs_finish_kernel(int64_t P, PreferenceTerms l) {
    __shared__ double part[kFinish / 64];
    const double s = block_sum<kFinish / 64>(strided_sum(l.by_pair, threadIdx.x, P, kFinish), part);
    if (threadIdx.x == 0) l.loss[0] = (float)s;
}

// The gradient by the logits from stats and c, a pass of its own: kGradVecs vectors of a row to a thread, some workgroups to a row.  No sums, so nothing
// waits but for its own loads: 12288 rows of 65536 bf16 read and 16384 written in 668 us, 5.6 TB/s.
template <typename T, int kT> __device__ __forceinline__ void grad_piece(const LossRows &a, const LossGrad &g, float up, int64_t row, int piece) {
    constexpr int kN = Vec<T>::kN;
    const int64_t b = row / a.T, t = row % a.T;
    const int64_t id = a.ids[row];
    const int V = (int)a.V, tid = threadIdx.x % kT, first = piece * (kGradVecs * kT) + tid;
    const T *x = static_cast<const T *>(a.logits) + b * a.stride_b + t * a.stride_t;
    T *out = static_cast<T *>(g.grad) + row * V;
    const Cut<T> cut(x, V);
    const bool lone = piece == 0 && tid < cut.singles;
    if (!counts(a, row, id)) {
        Bits<T> z;
        z.zero();
#pragma unroll
        for (int i = 0; i < kGradVecs; ++i)
            if (first + i * kT < cut.full) z.template store<true>(out + cut.head + (int64_t)(first + i * kT) * kN);
        if (lone) store1(out + cut.single(tid), 0.f);
        return;
    }
    Bits<T> held[kGradVecs];
#pragma unroll
    for (int i = 0; i < kGradVecs; ++i)
        if (first + i * kT < cut.full) held[i].template load<false>(x + cut.head + (int64_t)(first + i * kT) * kN);
    float c = g.coef[b * g.coef_stride_b + t * g.coef_stride_t] * up;
    if (id >= V) c = NAN;
    c *= (float)a.inv_temperature;
    const float top = a.stats[2 * row], norm = 1.f / a.stats[2 * row + 1], factor = -c * norm;
    const Scale scale(a.inv_temperature);
    either(g.past, [&](auto past) {
#pragma unroll
        for (int i = 0; i < kGradVecs; ++i) {
            if (first + i * kT >= cut.full) continue;
            gradient<T>(held[i], scale, top, factor);
            held[i].template store<past.value>(out + cut.head + (int64_t)(first + i * kT) * kN);
        }
    });
    if (lone) store1(out + cut.single(tid), gradient<T>(load1(x + cut.single(tid)), scale, top, factor));
    // the element that stands there, by the thread whose store it was in
    if (id >= V) return;
    const int j = cut.single_of((int)id), v = cut.vector_of((int)id);
    const bool mine = j >= 0 ? lone && tid == j : v % kT == tid && v / (kGradVecs * kT) == piece;
    if (mine) store1(out + id, c + scale.exp_once(load1(x + id) - top) * factor);
}

// kT threads, a workgroup or one of its waves, take a piece.  (The last rows come first: those are the ones that a pass over all rows before this
// one may have left in the last-level cache.)
template <typename T, int kT> __global__ __launch_bounds__(kThreads) void grad_kernel(LossRows a, LossGrad g, int pieces, int64_t rows) {
    const float up = g.upstream ? *g.upstream : 1.f;
    if (g.is_there && up == 1.f) return;
    constexpr int kTogether = kThreads / kT;
    for (int64_t i = (int64_t)blockIdx.x * kTogether + __builtin_amdgcn_readfirstlane(threadIdx.x / kT); i < rows * pieces; i += (int64_t)gridDim.x * kTogether)
        grad_piece<T, kT>(a, g, up, rows - 1 - i / pieces, (int)(i % pieces));
}

template <typename F> hipError_t by_type(int dtype, F &&f) {
    if (dtype == kBF16) f(bf16_t{});
    else if (dtype == kF16) f(f16_t{});
    else f(float{});
    return hipGetLastError();
}

}  // namespace

// three terms for each token, sums of stretches of them and the counts; or lp in 64 bits and a loss for each pair
size_t loss_workspace_bytes(int64_t B, int64_t T) {
    return (size_t)(3 * B * T + 1) / 2 * 2 * sizeof(float) + 3 * kStretches * sizeof(double) + (size_t)(B + kCountBlocks) * sizeof(int);
}

namespace {

// Whether the gradient is written past the caches: from the size on that they do not hold for whoever reads it next.
bool past_the_caches(int dtype, const LossRows &a) { return a.B * a.T * a.V * (dtype == kF32 ? 4 : 2) >= kPastBytes; }

template <int kT, int kVecs, bool kHold> struct Shape {
    static constexpr int threads = kT, vecs = kVecs;
    static constexpr bool hold = kHold;
};

// f(shape) of the smallest one that holds a row of n vectors.  Cross entropy with its gradient of 1 GiB of bf16 logits, in us, this shape / the next
// one up: V 20000 411 / 445, 32000 361 / 406 (1024 x 4), 50257 410 / 488 (1024 x 8, rows not from a boundary).  Two workgroups of 512 threads share a compute
// unit where one of 1024 fills it, so that one reads while the other computes and writes: V 73000 420 / 500 (1024 x 10), 98000 452 / 492 (1024 x
// 13); fp32 logits, half as many to a byte, gain nothing by it (V 40000 759 / 725).
template <typename T, typename F> void by_length(int64_t n, F &&f) {
    if (n <= 64 * 1) return f(Shape<64, 1, true>{});
    if (n <= 64 * 2) return f(Shape<64, 2, true>{});
    if (n <= 64 * 4) return f(Shape<64, 4, true>{});
    if (n <= 64 * 8) return f(Shape<64, 8, true>{});
    if (n <= 256 * 4) return f(Shape<256, 4, true>{});
    if (n <= 256 * 6) return f(Shape<256, 6, true>{});
    if (n <= 256 * 8) return f(Shape<256, 8, true>{});
    if (n <= 256 * 10) return f(Shape<256, 10, true>{});
    if (n <= 512 * 6) return f(Shape<512, 6, true>{});
    if (n <= 512 * 8) return f(Shape<512, 8, true>{});
    if (n <= 1024 * 5) return f(Shape<1024, 5, true>{});
    if (n <= 1024 * 6) return f(Shape<1024, 6, true>{});
    if (n <= 1024 * 7) return f(Shape<1024, 7, true>{});
    if (n <= 1024 * 8) return f(Shape<1024, 8, true>{});
    if constexpr (sizeof(T) == 2) {
        if (n <= 512 * 18) return f(Shape<512, 18, true>{});
        if (n <= 512 * 20) return f(Shape<512, 20, true>{});
        if (n <= 512 * 22) return f(Shape<512, 22, true>{});
        if (n <= 512 * 24) return f(Shape<512, 24, true>{});
    } else {
        if (n <= 1024 * 10) return f(Shape<1024, 10, true>{});
    }
    if (n <= 1024 * 13) return f(Shape<1024, 13, true>{});
    if (n <= 1024 * 16) return f(Shape<1024, 16, true>{});
    if (n <= 1024 * 20) return f(Shape<1024, 20, true>{});
    f(Shape<1024, 4, false>{});
}
// ... where nothing but the row's sums is wanted of it: from 16384 16-bit logits on a row is better gone through than held (8192 rows of 65536 bf16
// 200 us held by 1024 threads, 157 gone through by 512), down to 4096 the wave that holds a row does without LDS and barriers.
template <typename F> void by_length_alone(int64_t n, F &&f) {
    if (n <= 64 * 1) f(Shape<64, 1, true>{});
    else if (n <= 64 * 2) f(Shape<64, 2, true>{});
    else if (n <= 64 * 4) f(Shape<64, 4, true>{});
    else if (n <= 64 * 8) f(Shape<64, 8, true>{});
    else if (n <= 256 * 4) f(Shape<256, 4, true>{});
    else if (n <= 256 * 6) f(Shape<256, 6, true>{});
    else if (n <= 256 * 8) f(Shape<256, 8, true>{});
    else if (n <= 512 * 8) f(Shape<256, 4, false>{});
    else f(Shape<512, 4, false>{});
}

template <typename F> void in_launches(int64_t blocks, F &&f) {
    for (int64_t first = 0; first < blocks; first += kMostBlocks) f(first, (unsigned)(blocks - first < kMostBlocks ? blocks - first : kMostBlocks));
}

template <typename T, typename S, bool kGrad> void launch_rows(hipStream_t st, S, const LossRows &a, const LossCounts &n, const LossTerms &l, const LossGrad &g) {
    const int64_t rows = a.B * a.T;
    const bool waves = S::threads == 64;
    in_launches(waves ? (rows + kWaves - 1) / kWaves : rows, [&](int64_t first, unsigned blocks) {
        hipLaunchKernelGGL((rows_kernel<T, S::threads, S::vecs, S::hold, kGrad>), dim3(blocks), dim3(waves ? kThreads : S::threads), 0, st, a, n, l, g, first);
    });
}

}  // namespace

hipError_t loss_rows(hipStream_t st, int dtype, LossRows a, LossTerms l, void *grad, void *workspace) {
    LossCounts n{};
    const int64_t rows = a.B * a.T;
    double *sums = nullptr;
    if (l.kind != kLossNone) {
        l.terms = static_cast<float *>(workspace);
        l.count = l.kind == kLossPolicy ? 3 : 1;
        sums = reinterpret_cast<double *>(l.terms + (3 * rows + 1) / 2 * 2);
        n.partial = reinterpret_cast<int *>(sums + 3 * kStretches);
        n.by_text = n.partial + kCountBlocks;
        if (l.reduction == kLossMeanOfTexts) {
            n.blocks = (int)(a.B < kCountBlocks ? a.B : kCountBlocks);
            hipLaunchKernelGGL(count_texts_kernel, dim3(n.blocks), dim3(kFinish), 0, st, a, n);
        } else if (l.reduction == kLossMean && rows > kFewRows) {
            int64_t stretch = 2 * kFinish;
            if (rows > stretch * kCountBlocks) stretch = (rows + kCountBlocks - 1) / kCountBlocks;
            n.blocks = (int)((rows + stretch - 1) / stretch);
            hipLaunchKernelGGL(count_kernel, dim3(n.blocks), dim3(kFinish), 0, st, a, n, stretch);
        }
    }
    hipError_t e = by_type(dtype, [&](auto t) {
        using T = decltype(t);
        const int64_t vecs = a.V / Vec<T>::kN;
        const LossGrad g{nullptr, 0, 0, nullptr, 0, grad, past_the_caches(dtype, a)};
        if (l.kind == kLossNone) by_length_alone(vecs, [&](auto s) { launch_rows<T, decltype(s), false>(st, s, a, n, l, g); });
        else if (!grad) by_length<T>(vecs, [&](auto s) { launch_rows<T, decltype(s), false>(st, s, a, n, l, g); });
        else by_length<T>(vecs, [&](auto s) { launch_rows<T, decltype(s), true>(st, s, a, n, l, g); });
    });
    if (e != hipSuccess || l.kind == kLossNone) return e;
    // (one workgroup adds 65536 values in 19 us; stretches and their sums take 9, at four times as many too)
    const int64_t stretch = rows <= 32768 ? rows : (rows + kStretches - 1) / kStretches;
    hipLaunchKernelGGL(finish_kernel, dim3((unsigned)((rows + stretch - 1) / stretch), l.count), dim3(kFinish), 0, st, rows, l, sums, stretch);
    if (rows > 32768) hipLaunchKernelGGL(finish_stretches_kernel, dim3(l.count), dim3(kStretches), 0, st, l, sums, (int)((rows + stretch - 1) / stretch));
    return hipGetLastError();
}

hipError_t loss_grad(hipStream_t st, int dtype, LossRows a, LossGrad g) {
    g.past = past_the_caches(dtype, a);
    return by_type(dtype, [&](auto t) {
        using T = decltype(t);
        const auto launch = [&](auto threads) {
            const int64_t per = (int64_t)kGradVecs * threads.value * Vec<T>::kN, pieces = (a.V + per - 1) / per, rows = a.B * a.T;
            const int64_t all = (rows * pieces * threads.value + kThreads - 1) / kThreads;
            // (most often there is nothing to do where a forward has written the gradient: 32768 workgroups took 9 us to find that out)
            const int64_t most = g.is_there ? 2048 : kMostBlocks;
            hipLaunchKernelGGL((grad_kernel<T, threads.value>), dim3((unsigned)(all < most ? all : most)), dim3(kThreads), 0, st, a, g, (int)pieces, rows);
        };
        // (a short row leaves most of a workgroup idle, a wave with more than four vectors to a lane has few others beside it: 512 MiB of rows by workgroups /
        // by waves, in us, bf16 V 1000 471 / 186, 2048 245 / 166, 4000 175 / 183; fp32 V 1000 521 / 435, 2048 367 / 421)
        if (a.V <= 64 * 4 * Vec<T>::kN) launch(std::integral_constant<int, 64>{});
        else launch(std::integral_constant<int, kThreads>{});
    });
}

hipError_t loss_preference(hipStream_t st, int dtype, LossRows a, PreferenceTerms l) {
    const int64_t P = a.B / 2;
    l.by_pair = a.exact + a.B * a.T;
    const hipError_t e = loss_rows(st, dtype, a, LossTerms{}, nullptr, nullptr);
    if (e != hipSuccess) return e;
    in_launches(P, [&](int64_t pair, unsigned blocks) { hipLaunchKernelGGL(pairs_kernel, dim3(blocks), dim3(kFinish), 0, st, a, l, pair); });
    if (P > 1) hipLaunchKernelGGL(pairs_finish_kernel, dim3(1), dim3(kFinish), 0, st, P, l);   // (4 us behind a large kernel)
    return hipGetLastError();
}

}  // namespace wkv6
