// Rows of a table by token, scaled, and the table's gradient.
//
//   out[i] = scale W[ids[i]]                            (zeros where ids[i] < 0, NaN where ids[i] >= V)
//   gW[v]  = scale sum over the places i with ids[i] = v of g[i]
//
// The gradient adds up rows in the order of their places and uses no atomics: the same call gives the same bits.  The places are sorted by token (stable,
// 9 bits at a time), and stretches of equal length of the sorted list, however often a token occurs, are added up side by side.  A token's
// run that reaches over an end of a stretch leaves its part there in the workspace, and another launch adds such parts in order.  Most of the table belongs to
// no token of the call: it is set to zero by other workgroups of the launch that sorts.
//
// Bound by memory, the table's zeros before all: 8192 tokens, 65536 x 2048 in fp32: rows 19 us (7.0 TB/s), zeros with the sorting behind them 91 (5.9 TB/s), sums 19, what reaches over
// stretches 7.  1665 tokens of 50277 x 777 fp16: 6, 18, 10 and 4.  One token: a launch of 4 us.  All 8192 tokens alike: the parts of 512 stretches are added one
// after the other, 50 us more.
#include "wkv6_common.h"
#include "wkv6_kernels.h"
#include "wkv6_pieces.h"

#include <math.h>

#include <algorithm>

namespace wkv6 {
namespace {

constexpr int kThreads = 256;
constexpr int kDigit = 9, kBins = 1 << kDigit;
constexpr int64_t kMostBlocks = 1 << 20;   // of a launch, whose threads are counted in 32 bits

// ---- the rows ----

template <typename W, typename O> __global__ __launch_bounds__(kThreads) void embedding_kernel(EmbeddingArgs a, int64_t first_block) {
    constexpr int kE = 16 / sizeof(W), kAtOnce = 8;
    const int lane = threadIdx.x & 63;
    const int64_t row = (first_block + blockIdx.x) * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    if (row >= a.N) return;
    const int64_t id = a.ids[row];
    const W *w = static_cast<const W *>(a.weight) + (id >= 0 && id < a.V ? id : 0) * a.stride;
    O *out = static_cast<O *>(a.out) + row * a.C;
    const bool held = id >= 0 && id < a.V;
    const float other = id < 0 ? 0.f : NAN;
    for (int64_t first = 0; first < a.C; first += 64 * kE * kAtOnce) {
        Piece<W, kE> b[kAtOnce];
        const int left = (int)min(a.C - first, (int64_t)(64 * kE * kAtOnce));
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) b[i].template load<false>(w + first + (i * 64 + lane) * kE, held ? left - (i * 64 + lane) * kE : 0);
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            float v[kE];
            unpack(b[i], v);
#pragma unroll
            for (int e = 0; e < kE; ++e) v[e] = held ? v[e] * a.scale : other;
            Piece<O, kE> o;
            pack(v, o);
            o.template store<false>(out + first + (i * 64 + lane) * kE, left - (i * 64 + lane) * kE);
        }
    }
}

// ---- places sorted by token ----

// A token as a sorting key: V for what takes no part.
__device__ __forceinline__ uint32_t key_of(const EmbeddingGrad &a, int64_t i) {
    const int64_t id = a.ids[i];
    return id < 0 || id >= a.V || id == a.padding_id ? (uint32_t)a.V : (uint32_t)id;
}

// Lanes of this wave, among those that take part, with this lane's digit.
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, bool part) {
    uint64_t m = __ballot(part);
#pragma unroll
    for (int b = 0; b < kDigit; ++b) {
        const uint64_t ones = __ballot((digit >> b) & 1);
        m &= (digit >> b) & 1 ? ones : ~ones;
    }
    return m;
}

// The place of each item among those of its digit that its wave has seen; counts: kBins of the wave's own, zero before.
template <int kItems> __device__ __forceinline__ void rank(const uint32_t (&digit)[kItems], int count, int lane, volatile uint32_t *counts, uint32_t (&place)[kItems]) {
#pragma unroll
    for (int r = 0; r < kItems; ++r) {
        if (r * 64 >= count) break;
        const bool part = r * 64 + lane < count;
        const uint64_t same = same_digit(digit[r], part), below = same & ((1ull << lane) - 1);
        const uint32_t before = part ? counts[digit[r]] : 0;
        place[r] = before + (uint32_t)__popcll(below);
        __builtin_amdgcn_wave_barrier();
        if (part && below == 0) counts[digit[r]] = before + (uint32_t)__popcll(same);
        __builtin_amdgcn_wave_barrier();
    }
}

// Exclusive sums over kBins values by the first kBins threads of a workgroup; all threads call it.
__device__ __forceinline__ uint32_t bins_before(uint32_t mine, uint32_t *part) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t v = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t up = __shfl_up(v, d);
        if (lane >= d) v += up;
    }
    if (lane == 63 && wave < kBins / 64) part[wave] = v;
    __syncthreads();
    uint32_t before = v - mine;
    for (int i = 0; i < min(wave, kBins / 64); ++i) before += part[i];
    return before;
}

// Zeros by all threads of `blocks` workgroups, of which this is number `block`, each in a stretch of its own and past the caches.  (2048 workgroups' 512 MiB beside the sorting of 8192
// tokens 93 us, strided over the whole 122; through the caches 79, but the sums behind it then take 36 us instead of 19.)
__device__ __forceinline__ void zero(char *p, int64_t count, int64_t block, int64_t blocks) {
    typedef uint32_t vec __attribute__((ext_vector_type(4)));
    const int64_t head = min(count, (int64_t)(-(uintptr_t)p & 15)), whole = (count - head) / 16, tail = count - head - whole * 16;
    vec *v = reinterpret_cast<vec *>(p + head);
    const int64_t each = (whole + blocks - 1) / blocks, end = min(whole, (block + 1) * each);
    for (int64_t i = block * each + threadIdx.x; i < end; i += blockDim.x) __builtin_nontemporal_store((vec)(0), v + i);
    if (block == 0 && threadIdx.x < head) p[threadIdx.x] = 0;
    if (block == 0 && threadIdx.x < tail) p[count - tail + threadIdx.x] = 0;
}

constexpr int kSmallThreads = 1024, kSmallItems = 16, kSmall = kSmallThreads * kSmallItems;   // places that one workgroup sorts in its LDS ...
constexpr int kSmallKeyBits = 18;   // ... with tokens that fit beside a place's 14 bits
static_assert(kSmall <= 1 << (32 - kSmallKeyBits), "an item is one word");

__global__ __launch_bounds__(kSmallThreads) void sort_small_kernel(EmbeddingGrad a, int bits, int64_t table_bytes, uint32_t *keys, uint32_t *places) {
    constexpr int kW = kSmallThreads / 64, kPlace = 32 - kSmallKeyBits;
    __shared__ uint32_t items[kSmall], counts[kW][kBins], part[kBins / 64], start[kBins];
    if (blockIdx.x > 0) {
        zero(static_cast<char *>(a.gweight), table_bytes, blockIdx.x - 1, gridDim.x - 1);
        return;
    }
    const int N = (int)a.N, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int each = (N + kW * 64 - 1) / (kW * 64) * 64, first = wave * each, count = max(0, min(each, N - first));   // this wave's items
    for (int i = tid; i < N; i += kSmallThreads) items[i] = key_of(a, i) << kPlace | (uint32_t)i;
    for (int shift = kPlace; shift < kPlace + bits; shift += kDigit) {
        for (int i = tid; i < kW * kBins; i += kSmallThreads) (&counts[0][0])[i] = 0;
        __syncthreads();
        uint32_t item[kSmallItems], digit[kSmallItems], place[kSmallItems];
#pragma unroll
        for (int r = 0; r < kSmallItems; ++r) {
            item[r] = r * 64 + lane < count ? items[first + r * 64 + lane] : 0;
            digit[r] = item[r] >> shift & (kBins - 1);
        }
        rank<kSmallItems>(digit, count, lane, counts[wave], place);
        __syncthreads();
        uint32_t total = 0;
        if (tid < kBins)
            for (int w = 0; w < kW; ++w) {
                const uint32_t n = counts[w][tid];
                counts[w][tid] = total;
                total += n;
            }
        const uint32_t before = bins_before(total, part);
        if (tid < kBins) start[tid] = before;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kSmallItems; ++r)
            if (r * 64 + lane < count) items[start[digit[r]] + counts[wave][digit[r]] + place[r]] = item[r];
        __syncthreads();
    }
    for (int i = tid; i < N; i += kSmallThreads) {
        keys[i] = items[i] >> kPlace;
        places[i] = items[i] & ((1u << kPlace) - 1);
    }
}

// Any number of places: tiles of kTile, three launches for every 9 bits.
constexpr int kTileItems = 16, kTileWaves = kThreads / 64, kTile = kThreads * kTileItems;

__device__ __forceinline__ void load_tile(const EmbeddingGrad &a, const uint32_t *keys, int64_t first, int count, int lane, int shift, uint32_t (&key)[kTileItems],
                                          uint32_t (&digit)[kTileItems]) {
#pragma unroll
    for (int r = 0; r < kTileItems; ++r) {
        key[r] = r * 64 + lane >= count ? 0 : keys ? keys[first + r * 64 + lane] : key_of(a, first + r * 64 + lane);
        digit[r] = key[r] >> shift & (kBins - 1);
    }
}

// How many items of each digit a tile has: counts[digit][tile].  keys null: the first round, from the tokens themselves; the workgroups behind the tiles' set
// the table to zero then.
__global__ __launch_bounds__(kThreads) void sort_count_kernel(EmbeddingGrad a, const uint32_t *keys, int shift, int tiles, uint32_t *counts, int64_t table_bytes) {
    __shared__ uint32_t bins[kBins];
    if ((int)blockIdx.x >= tiles) {
        zero(static_cast<char *>(a.gweight), table_bytes, blockIdx.x - tiles, gridDim.x - tiles);
        return;
    }
    for (int i = threadIdx.x; i < kBins; i += kThreads) bins[i] = 0;
    __syncthreads();
    const int64_t first = (int64_t)blockIdx.x * kTile;
    const int count = (int)min(a.N - first, (int64_t)kTile);
    for (int i = threadIdx.x; i < count; i += kThreads) atomicAdd(&bins[(keys ? keys[first + i] : key_of(a, first + i)) >> shift & (kBins - 1)], 1u);
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads) counts[(int64_t)i * tiles + blockIdx.x] = bins[i];
}

// counts[digit][tile] become the sums over the tiles before, totals[digit] the sum over all; a workgroup to a digit.
__global__ __launch_bounds__(kThreads) void sort_sum_kernel(int tiles, uint32_t *counts, uint32_t *totals) {
    __shared__ uint32_t part[kThreads / 64];
    uint32_t *mine = counts + (int64_t)blockIdx.x * tiles;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t carry = 0;
    for (int first = 0; first < tiles; first += kThreads) {
        const int at = first + threadIdx.x;
        const uint32_t n = at < tiles ? mine[at] : 0;
        uint32_t v = n;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t up = __shfl_up(v, d);
            if (lane >= d) v += up;
        }
        __syncthreads();
        if (lane == 63) part[wave] = v;
        __syncthreads();
        uint32_t before = carry + v - n;
        for (int i = 0; i < wave; ++i) before += part[i];
        for (int i = 0; i < kThreads / 64; ++i) carry += part[i];
        if (at < tiles) mine[at] = before;
    }
    if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

__global__ __launch_bounds__(kThreads) void sort_place_kernel(EmbeddingGrad a, const uint32_t *keys, const uint32_t *places, int shift, int tiles, const uint32_t *counts,
                                                              const uint32_t *totals, uint32_t *new_keys, uint32_t *new_places) {
    __shared__ uint32_t seen[kTileWaves][kBins], start[kBins], part[kTileWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    for (int i = tid; i < kTileWaves * kBins; i += kThreads) (&seen[0][0])[i] = 0;
    __syncthreads();
    const int64_t tile = (int64_t)blockIdx.x * kTile, first = tile + wave * (kTile / kTileWaves);
    const int count = (int)max((int64_t)0, min(a.N - first, (int64_t)(kTile / kTileWaves)));
    uint32_t key[kTileItems], digit[kTileItems], place[kTileItems];
    load_tile(a, keys, first, count, lane, shift, key, digit);
    rank<kTileItems>(digit, count, lane, seen[wave], place);
    // where each digit's items of this tile begin: two digits to a thread, next to each other
    uint32_t total[kBins / kThreads], mine = 0;
#pragma unroll
    for (int k = 0; k < kBins / kThreads; ++k) {
        total[k] = totals[tid * (kBins / kThreads) + k];
        mine += total[k];
    }
    uint32_t v = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t up = __shfl_up(v, d);
        if (lane >= d) v += up;
    }
    if (lane == 63) part[wave] = v;
    __syncthreads();
    uint32_t before = v - mine;
    for (int i = 0; i < wave; ++i) before += part[i];
#pragma unroll
    for (int k = 0; k < kBins / kThreads; ++k) {
        const int bin = tid * (kBins / kThreads) + k;
        uint32_t at = before + counts[(int64_t)bin * tiles + blockIdx.x];
        for (int w = 0; w < kTileWaves; ++w) {
            const uint32_t n = seen[w][bin];
            seen[w][bin] = at;
            at += n;
        }
        before += total[k];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kTileItems; ++r) {
        if (r * 64 + lane >= count) continue;
        const uint32_t to = seen[wave][digit[r]] + place[r];
        new_keys[to] = key[r];
        new_places[to] = keys ? places[first + r * 64 + lane] : (uint32_t)(first + r * 64 + lane);
    }
}

// ---- the sums ----

// What the sums of stretches leave for the runs that reach over their ends: of stretch s the sum of the run that came in at its beginning, at 2 s, and of the
// one that goes on behind its end and began in it, at 2 s + 1.
struct Sorted {
    const uint32_t *keys, *places;
    float *partial;    // (stretches, 2, C)
    int stretch;       // places of a stretch
    int64_t stretches;
};

template <typename W, int kE> __device__ __forceinline__ void store_row(const EmbeddingGrad &a, uint32_t key, int64_t at, int n, const float (&sum)[kE]) {
    float v[kE];
#pragma unroll
    for (int e = 0; e < kE; ++e) v[e] = sum[e] * a.scale;
    Piece<W, kE> o;
    pack(v, o);
    o.template store<false>(static_cast<W *>(a.gweight) + (int64_t)key * a.C + at, n);
}

// kT threads (a wave of a workgroup, or a workgroup) take a stretch, kVecs pieces of 16 bytes of a row to a thread; blockIdx.y is the part of the row.
template <typename G, typename W, int kT, int kVecs> __global__ __launch_bounds__(kThreads) void sum_kernel(EmbeddingGrad a, Sorted s, int64_t first_block) {
    constexpr int kE = 16 / sizeof(G), kAhead = 8, kPer = kThreads / kT;
    const int tid = threadIdx.x % kT;
    const int64_t number = (first_block + blockIdx.x) * kPer + (kT == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x / 64) : 0);
    if (number >= s.stretches) return;
    const int64_t begin = number * s.stretch, end = min(begin + s.stretch, a.N), column = (int64_t)blockIdx.y * kT * kVecs * kE;
    const int C = (int)min(a.C - column, (int64_t)kT * kVecs * kE);   // columns from there on
    const G *g = static_cast<const G *>(a.gout) + column;
    float *partial = s.partial + (number * 2) * a.C + column;
    const uint32_t none = (uint32_t)a.V;
    const uint32_t came = begin > 0 ? s.keys[begin - 1] : none, goes = end < a.N ? s.keys[end] : none;
    float sum[kVecs][kE];
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
#pragma unroll
        for (int e = 0; e < kE; ++e) sum[i][e] = 0.f;
    uint32_t run = s.keys[begin];
    bool from_before = run == came;
    const auto flush = [&](bool to_next) {
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            const int at = (i * kT + tid) * kE;
            if (from_before || to_next) {
                Piece<float, kE> o;
                pack(sum[i], o);
                o.template store<false>(partial + (from_before ? 0 : a.C) + at, C - at);
            } else {
                store_row<W, kE>(a, run, column + at, C - at, sum[i]);
            }
#pragma unroll
            for (int e = 0; e < kE; ++e) sum[i][e] = 0.f;
        }
    };
    for (int64_t j = begin; j < end && run != none; j += kAhead) {
        Piece<G, kE> b[kAhead][kVecs];
        uint32_t key[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            key[k] = j + k < end ? s.keys[j + k] : none;
            const int64_t place = key[k] != none ? s.places[j + k] : 0;
#pragma unroll
            for (int i = 0; i < kVecs; ++i) {
                const int at = (i * kT + tid) * kE;
                b[k][i].template load<false>(g + place * a.C + at, key[k] != none ? C - at : 0);
            }
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            if (j + k >= end) break;
            if (key[k] != run) {
                flush(false);
                from_before = false;
                run = key[k];
            }
            if (run == none) break;
#pragma unroll
            for (int i = 0; i < kVecs; ++i) {
                float v[kE];
                unpack(b[k][i], v);
#pragma unroll
                for (int e = 0; e < kE; ++e) sum[i][e] += v[e];
            }
        }
    }
    if (run != none) flush(run == goes);
}

// The runs that reach over an end of a stretch, by the stretch that they begin in.
template <typename W> __global__ __launch_bounds__(kThreads) void join_kernel(EmbeddingGrad a, Sorted s, int64_t first_block) {
    constexpr int kE = 4, kAhead = 32;
    const int64_t number = first_block + blockIdx.x, begin = number * s.stretch, end = begin + s.stretch;
    if (end >= a.N) return;
    const uint32_t run = s.keys[end];
    if (run == (uint32_t)a.V || s.keys[end - 1] != run || (begin > 0 && s.keys[begin - 1] == run)) return;
    // the last stretch that begins with this run
    const int lane = threadIdx.x & 63;
    int64_t last = number + 1;
    for (;;) {
        const int64_t at = last + 1 + lane;
        const uint64_t same = __ballot(at < s.stretches && s.keys[min(at, s.stretches - 1) * s.stretch] == run);
        const int more = ~same == 0 ? 64 : __builtin_ctzll(~same);
        last += more;
        if (more < 64) break;
    }
    const int64_t column = ((int64_t)blockIdx.y * kThreads + threadIdx.x) * kE;
    const int n = (int)min(a.C - column, (int64_t)kE);
    if (n <= 0) return;
    Piece<float, kE> b[kAhead];
    float sum[kE];
    b[0].template load<false>(s.partial + (2 * number + 1) * a.C + column, n);
    unpack(b[0], sum);
    for (int64_t t = number + 1; t <= last; t += kAhead) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k) b[k].template load<false>(s.partial + 2 * min(t + k, last) * a.C + column, t + k <= last ? n : 0);
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            float v[kE];
            unpack(b[k], v);   // (zero behind the last)
#pragma unroll
            for (int e = 0; e < kE; ++e) sum[e] += v[e];
        }
    }
    store_row<W, kE>(a, run, column, n, sum);
}

template <typename F> hipError_t by_types(int table, int out, F &&f) {
    if (table == kBF16) f(bf16_t{}, bf16_t{});
    else if (table == kF16) f(f16_t{}, f16_t{});
    else if (out == kF32) f(float{}, float{});
    else if (out == kBF16) f(float{}, bf16_t{});
    else f(float{}, f16_t{});
    return hipGetLastError();
}

int key_bits(int64_t V) {   // of the numbers 0 .. V
    int bits = 0;
    while (V >> bits) ++bits;
    return bits;
}
bool is_small(int64_t N, int64_t V) { return N <= kSmall && key_bits(V) <= kSmallKeyBits; }

// Places of a stretch, a multiple of the rows that are loaded at once.  Few: more run side by side (1665 rows of 777 fp16 16 us with 16 to a stretch, 11 with 8); many: fewer
// parts are left for the tokens that occur often.
int64_t stretch_of(int64_t N) { return N <= 4096 ? 8 : N <= 16384 ? 16 : (N / 1024 + 7) / 8 * 8; }

int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

}  // namespace

hipError_t embedding(hipStream_t st, int dtype, int out_dtype, const EmbeddingArgs &a) {
    return by_types(dtype, out_dtype, [&](auto w, auto o) {
        const int64_t blocks = (a.N + kThreads / 64 - 1) / (kThreads / 64);
        for (int64_t first = 0; first < blocks; first += kMostBlocks)
            hipLaunchKernelGGL((embedding_kernel<decltype(w), decltype(o)>), dim3((unsigned)std::min(blocks - first, kMostBlocks)), dim3(kThreads), 0, st, a, first);
    });
}

size_t embedding_backward_workspace_bytes(int64_t N, int64_t V, int64_t C) {
    const int64_t stretches = (N + stretch_of(N) - 1) / stretch_of(N), list = round_up(4 * N, 16), tiles = (N + kTile - 1) / kTile;
    const int64_t sorting = is_small(N, V) ? 2 * list : 4 * list + round_up(4 * kBins * (tiles + 1), 16);
    return (size_t)(sorting + stretches * 2 * C * (int64_t)sizeof(float));
}

hipError_t embedding_backward(hipStream_t st, int dtype, int out_dtype, const EmbeddingGrad &a, void *workspace) {
    const int64_t list = round_up(4 * a.N, 16) / 4, table_bytes = a.V * a.C * (dtype == kF32 ? 4 : 2);
    const int bits = key_bits(a.V);
    uint32_t *keys = static_cast<uint32_t *>(workspace), *places = keys + list, *end = places + list;
    // (a workgroup of the sorting launch sets 64 KiB or more to zero; 2048 of them keep every unit writing)
    const int64_t zeroing = std::max<int64_t>(1, std::min<int64_t>(2048, table_bytes / 65536));
    if (is_small(a.N, a.V)) {
        hipLaunchKernelGGL(sort_small_kernel, dim3((unsigned)(1 + zeroing)), dim3(kSmallThreads), 0, st, a, bits, table_bytes, keys, places);
    } else {
        const int tiles = (int)((a.N + kTile - 1) / kTile);
        uint32_t *other_keys = end, *other_places = end + list, *counts = other_places + list, *totals = counts + (int64_t)kBins * tiles;
        end = counts + round_up(4 * kBins * ((int64_t)tiles + 1), 16) / 4;
        const uint32_t *from_keys = nullptr, *from_places = nullptr;
        for (int shift = 0; shift < bits; shift += kDigit) {
            hipLaunchKernelGGL(sort_count_kernel, dim3((unsigned)(tiles + (shift == 0 ? zeroing : 0))), dim3(kThreads), 0, st, a, from_keys, shift, tiles, counts, table_bytes);
            hipLaunchKernelGGL(sort_sum_kernel, dim3(kBins), dim3(kThreads), 0, st, tiles, counts, totals);
            hipLaunchKernelGGL(sort_place_kernel, dim3((unsigned)tiles), dim3(kThreads), 0, st, a, from_keys, from_places, shift, tiles, counts, totals, keys, places);
            from_keys = keys, from_places = places;
            std::swap(keys, other_keys);
            std::swap(places, other_places);
        }
        keys = const_cast<uint32_t *>(from_keys), places = const_cast<uint32_t *>(from_places);
    }
    Sorted s{keys, places, reinterpret_cast<float *>(end), (int)stretch_of(a.N), 0};
    s.stretches = (a.N + s.stretch - 1) / s.stretch;
    return by_types(dtype, out_dtype, [&](auto w, auto g) {
        using W = decltype(w);
        using G = decltype(g);
        constexpr int kE = 16 / sizeof(G);
        const auto launch = [&](auto threads, auto vecs) {
            constexpr int kT = decltype(threads)::value, kVecs = decltype(vecs)::value;
            const int64_t blocks = (s.stretches + kThreads / kT - 1) / (kThreads / kT), columns = (a.C + kT * kVecs * kE - 1) / (kT * kVecs * kE);
            for (int64_t first = 0; first < blocks; first += kMostBlocks)
                hipLaunchKernelGGL((sum_kernel<G, W, kT, kVecs>), dim3((unsigned)std::min(blocks - first, kMostBlocks), (unsigned)columns), dim3(kThreads), 0, st, a, s, first);
        };
        if (a.C <= 64 * kE) launch(std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
        else if (a.C <= 64 * 2 * kE) launch(std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
        else if (a.C <= 256 * kE) launch(std::integral_constant<int, 256>{}, std::integral_constant<int, 1>{});
        else launch(std::integral_constant<int, 256>{}, std::integral_constant<int, 2>{});
        for (int64_t first = 0; first < s.stretches; first += kMostBlocks)
            hipLaunchKernelGGL((join_kernel<W>), dim3((unsigned)std::min(s.stretches - first, kMostBlocks), (unsigned)((a.C + kThreads * 4 - 1) / (kThreads * 4))), dim3(kThreads), 0,
                               st, a, s, first);
    });
}

}  // namespace wkv6
