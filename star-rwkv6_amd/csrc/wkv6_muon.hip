// Weight updates brought near to the nearest matrix with orthonormal rows or columns, by Newton-Schulz products, and the optimizer's step with them.
//
//   X = U / (|U| + eps)              (|U|: the 2-norm of all elements; transposed if U has more rows than columns, so that X is m x n with m <= n)
//   steps times:  A = X X^T,   B = a I + b A + c A A,   X = B X
//   the step: buf = mu buf + (1 - mu) g,   U = (1 - mu) g + mu buf, or buf,   p = p (1 - lr wd) - rate X
//
// Precision.  The polynomial takes a singular value s to about a s while it is small, so five steps multiply what is lost in the small ones by up to a^5 = 485: with the
// matrices in bf16 throughout the result is off by 1 to 16 % of its size, with fp16 by 0.1 to 2 %.  Here every matrix is a pair of fp16 numbers hi + lo,
// 22 bits, and a product the three matrix instructions hi hi + hi lo + lo hi, which accumulate in fp32: 0.7 to 1.2 times the error of fp32 throughout, at
// 5 times the rate of the fp32 matrix instructions.  Values are held times 1024: those of X, A and B stay below some 4, so the pairs' range of
// 64 is not left by coefficients of any use, and lo keeps its bits down to 2^-13 of 1 (below, the pair is exact to 2^-35).
//
// A pair's row of K numbers: for every 32 of them 64 bytes of hi, then 64 of lo; zeros behind the last.  So what the matrix instructions take of a row
// in one stage is one line of 128 bytes.  A and A A are products of rows by rows, C_ij = sum_k P_ik Q_jk, and symmetric: only the tiles on and above the diagonal are
// computed, and each is written to both of its places.  Of B X the columns of X are multiplied with rows of B; LDS hands them out across its rows.
// B has a I in it, so that B X is the whole step.
//
// What bounds it: 12 matrices of 2048 x 2048 and 4 of 2048 x 7168 together, 1140 to 1260 TFLOP/s of fp16 products in B X (1.06 ms) and 1030 in A and A A (0.65 and 0.41 ms), where a library's
// product of 8192^3 fp16 runs at 1445: the chip's power lowers its clock to 1.6 to 1.8 GHz while the matrix units are busy 53 to 60 % of the time, so that
// fewer waits give fewer cycles a second, and what costs energy (LDS and cache traffic: tiles of 256) counts.  One matrix of 2048 x 2048: 36 to 49 us a product, of which the matrix
// units need 20; its tiles of 128 read 285 to 537 MB out of the caches at 8 to 11 TB/s, and half of the units have no tile of A.  Dividing the stages
// evenly among 256 workgroups instead, parts exchanged through memory: the same time for it, twice as long for many matrices.  Small ones: 17 launches of 10 to 14 us.
#include "wkv6_common.h"
#include "wkv6_kernels.h"
#include "wkv6_mfma.h"
#include "wkv6_pieces.h"

#include <math.h>

#include <algorithm>

namespace wkv6 {
namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef float f16x __attribute__((ext_vector_type(16)));

constexpr float kHeld = 1024.f;     // what values are multiplied by in a pair
constexpr int kThreads = 256;
constexpr int kGroup = 56;          // matrices of one launch: they travel in its arguments, which hold 4 KB
constexpr int kChunk = 16384;       // elements of a matrix that a workgroup squares and adds up
constexpr int kLine = 128;          // bytes of 32 numbers of a pair

struct Item {
    const void *grad;
    float *momentum;      // null: U is the gradient
    void *out;            // the weights, or the orthogonalized matrix
    float *master;
    int64_t at;           // of this matrix in the workspace, in bytes
    int m, n;             // m <= n
    float rate;           // of the step, over lr
    int tall;             // it has n rows and m columns
};
struct Group {
    Item t[kGroup];
    int first[kGroup + 1];   // unit of work (chunk, tile) at which a matrix begins
    int count;
};
struct Step {
    float momentum, kept;    // kept = 1 - momentum
    int nesterov, update;    // update: the last product is applied to weights
    float weight_decay, lr;
    double eps;
    const float *lr_device;  // one value in lr's place, or null
    float a, b, c;
    char *workspace;
};
static_assert(sizeof(Group) + sizeof(Step) + 64 <= 4096, "a launch's arguments");

__host__ __device__ inline int64_t pitch_of(int k) { return (int64_t)((k + 31) / 32) * kLine; }
__host__ __device__ inline int tiles(int k, int tile) { return (k + tile - 1) / tile; }

// Kinds of matrices, which go through in launches of their own.  kThinMatrix: m <= 64, see thin_kernel.  kLongMatrix: A has so few tiles, of so long a k, that workgroups share them.
constexpr int kThin = 64, kLongTile = 64;
enum { kGeneral = 0, kThinMatrix = 1, kLongMatrix = 2, kKinds = 3 };
__host__ __device__ inline int kind_of(int m, int n) { return m <= kThin ? kThinMatrix : m <= 512 && n >= 8192 && n >= 16 * m ? kLongMatrix : kGeneral; }
__host__ __device__ inline int half_of(int across) { return across * (across + 1) / 2; }   // tiles on and above the diagonal
// Workgroups that share a tile of a long matrix's A: 512 of them to all of its tiles, with 16 stages or more each.
__host__ __device__ inline int shares_of(int m, int n) { return max(1, min((n + 31) / 32 / 16, 512 / half_of(tiles(m, kLongTile)))); }
// Parts of a thin matrix's A at most: all workgroups of a launch read all of them, so not as many as there are blocks of 64 columns where those are many.
__host__ __device__ inline int thin_parts_of(int n) { return min(tiles(n, kThin), n <= 64 * 1024 / 4 ? 16 : 64); }

// What a matrix has in the workspace: X twice (one is read while the other is written), with zeros in rows up to a multiple of 32, A, B, the parts of a long matrix's A, sums of
// squares.  Of a thin matrix: the parts of A for two launches, 4 KB for each 32 x 32 of a part, and X's transpose.
struct Layout {
    int64_t x, x_other, a, b, parts, sums, end;
};
__host__ __device__ inline Layout layout_of(int m, int n) {
    Layout l;
    const int down = (m + 31) / 32, kind = kind_of(m, n);
    l.x = 0;
    l.x_other = l.x + (kind == kThinMatrix ? (int64_t)down * down * 2 * thin_parts_of(n) * 4096 : down * 32 * pitch_of(n));
    l.a = l.x_other + (kind == kThinMatrix ? n * pitch_of(m) : down * 32 * pitch_of(n));
    l.b = l.a + m * pitch_of(m);
    l.parts = l.b + m * pitch_of(m);
    l.sums = l.parts + (kind == kLongMatrix ? (int64_t)shares_of(m, n) * half_of(tiles(m, kLongTile)) * (kLongTile * kLongTile * 4) : 0);
    l.end = l.sums + ((int64_t)m * n + kChunk - 1) / kChunk * 8;
    l.end = (l.end + 255) / 256 * 256;
    return l;
}

// (by all lanes at once: each step of a search would wait for its own load of an argument)
__device__ __forceinline__ int item_of(const Group &g, int unit) {
    static_assert(kGroup <= 64, "one lane to a matrix");
    const int lane = threadIdx.x & 63;
    return __popcll(__ballot(lane < g.count && g.first[min(lane, kGroup - 1)] <= unit)) - 1;
}

__device__ __forceinline__ double block_sum(double v, double *part) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[0];
    for (int i = 1; i < kThreads / 64; ++i) v += part[i];
    return v;
}

// kHeld / (|U| + eps), which leaves fp32 at either end where |U| and what is multiplied do not: a power of two, and the rest.
struct Scale {
    float power, rest;
    __device__ __forceinline__ Scale(double squares, double eps) {
        const double norm = sqrt(squares), s = kHeld / (norm + eps);
        power = s > 0x1p64 ? 0x1p100f : s < 0x1p-64 ? 0x1p-100f : 1.f;
        rest = norm == 0. && eps > 0. ? 0.f : (float)(s / power);   // (of zeros and a small eps s may be more than any factor)
    }
    __device__ __forceinline__ float operator()(float v) const { return v * power * rest; }
};

// The momentum's update, and sums of squares of U by chunk.
template <typename G> __global__ __launch_bounds__(kThreads) void momentum_kernel(Group g, Step s) {
    constexpr int kE = 4;
    __shared__ double part[kThreads / 64];
    const int k = item_of(g, blockIdx.x);
    const Item &t = g.t[k];
    const int64_t numel = (int64_t)t.m * t.n;
    const int chunk = blockIdx.x - g.first[k];
    double sum = 0.;
#pragma unroll 4
    for (int i = 0; i < kChunk / kThreads / kE; ++i) {
        const int64_t at = (int64_t)chunk * kChunk + (i * kThreads + (int)threadIdx.x) * kE;
        const int n = (int)max((int64_t)0, min((int64_t)kE, numel - at));
        Piece<G, kE> p;
        p.template load<false>(static_cast<const G *>(t.grad) + at, n);
        float v[kE];
        unpack(p, v);
        if (t.momentum) {
            Piece<float, kE> q;
            q.template load<false>(t.momentum + at, n);
            float b[kE];
            unpack(q, b);
#pragma unroll
            for (int e = 0; e < kE; ++e) {
                b[e] = b[e] * s.momentum + v[e] * s.kept;
                v[e] = s.nesterov ? v[e] * s.kept + b[e] * s.momentum : b[e];
            }
            pack(b, q);
            q.template store<false>(t.momentum + at, n);
        }
#pragma unroll
        for (int e = 0; e < kE; ++e) sum = __builtin_fma((double)v[e], (double)v[e], sum);
    }
    sum = block_sum(sum, part);
    if (threadIdx.x == 0) reinterpret_cast<double *>(s.workspace + t.at + layout_of(t.m, t.n).sums)[chunk] = sum;
}

__device__ __forceinline__ void split(float v, f16_t &hi, f16_t &lo) {
    hi = to_f16(v);
    lo = to_f16(v - (float)hi);
}

// Eight values (times kHeld) into a pair's row.
__device__ __forceinline__ void store_pair8(char *row, int k, const float (&v)[8]) {
    h8 hi, lo;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        f16_t x, y;
        split(v[e], x, y);
        hi[e] = x, lo[e] = y;
    }
    char *p = row + (int64_t)(k / 32) * kLine + k % 32 * 2;
    *reinterpret_cast<h8 *>(p) = hi;
    *reinterpret_cast<h8 *>(p + 64) = lo;
}

constexpr int kSpread = 64;   // rows and columns of U that a workgroup takes

// U over its norm as a pair: X, or of a matrix with more rows than columns its transpose.
template <typename G> __global__ __launch_bounds__(kThreads) void spread_kernel(Group g, Step s) {
    __shared__ double part[kThreads / 64];
    __shared__ float tile[kSpread][kSpread + 1];
    const int k = item_of(g, blockIdx.x);
    const Item &t = g.t[k];
    const Layout l = layout_of(t.m, t.n);
    const int rows = t.tall ? t.n : t.m, columns = t.tall ? t.m : t.n;
    char *base = s.workspace + t.at;
    const double *sums = reinterpret_cast<const double *>(base + l.sums);
    const int chunks = (int)(((int64_t)t.m * t.n + kChunk - 1) / kChunk);
    double sum = 0.;
    for (int i = threadIdx.x; i < chunks; i += kThreads) sum += sums[i];
    const Scale scale(block_sum(sum, part), s.eps);
    const int across = (columns + kSpread - 1) / kSpread, number = blockIdx.x - g.first[k], r0 = number / across * kSpread, c0 = number % across * kSpread;
    // pieces of 8 of a row; rows of X as they are, columns through LDS.  Behind X's last row there are zeros, here and in the other X.
    constexpr int kE = 8, kPieces = kSpread * kSpread / kE / kThreads;
    const int x0 = t.tall ? c0 : r0, y0 = t.tall ? r0 : c0;
    const int64_t pitch = pitch_of(t.n);
    const auto store = [&](int r, int q, const float (&v)[kE]) {
        if (x0 + r >= (t.m + 31) / 32 * 32 || y0 + q >= (t.n + 31) / 32 * 32) return;
        store_pair8(base + l.x + (x0 + r) * pitch, y0 + q, v);
        if (x0 + r >= t.m) store_pair8(base + l.x_other + (x0 + r) * pitch, y0 + q, v);
    };
    Piece<G, kE> grad[kPieces];
    Piece<float, kE> momentum[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const int which = i * kThreads + threadIdx.x, r = r0 + which / 8, c = c0 + which % 8 * kE, n = r < rows ? columns - c : 0;
        grad[i].template load<false>(static_cast<const G *>(t.grad) + (int64_t)r * columns + c, n);
        if (t.momentum) momentum[i].template load<false>(t.momentum + (int64_t)r * columns + c, n);
    }
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const int which = i * kThreads + threadIdx.x;
        float v[kE], m[kE];
        unpack(grad[i], v);   // (zero where there is nothing)
        if (t.momentum) {
            unpack(momentum[i], m);
#pragma unroll
            for (int e = 0; e < kE; ++e) v[e] = s.nesterov ? v[e] * s.kept + m[e] * s.momentum : m[e];
        }
#pragma unroll
        for (int e = 0; e < kE; ++e) v[e] = scale(v[e]);
        if (!t.tall) store(which / 8, which % 8 * kE, v);
        else
#pragma unroll
            for (int e = 0; e < kE; ++e) tile[which / 8][which % 8 * kE + e] = v[e];
    }
    if (!t.tall) return;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const int which = i * kThreads + threadIdx.x, q = which % 8 * kE, r = which / 8;
        float v[kE];
#pragma unroll
        for (int e = 0; e < kE; ++e) v[e] = tile[q + e][r];
        store(r, q, v);
    }
}

// A = X X^T; B = a I + b A + c A A; X = B X; the same into the result; of long matrices a workgroup's part of A, and A from the parts
enum { kGram = 0, kPoly = 1, kApply = 2, kLast = 3, kGramPart = 4, kGramJoin = 5 };
constexpr bool is_symmetric(int mode) { return mode != kApply && mode != kLast; }

// Product tiles of T x T.  WM x WN waves share a tile's rows and columns, KS of such sets its stages of 32 k, of which LDS holds NB (to a set) at a time.
template <int T, int WM, int WN, int KS, int NB> struct TileShape {
    static constexpr int tile = T, wm = WM, wn = WN, ks = KS, buffers = NB, threads = 64 * WM * WN * KS;
    static constexpr int set_bytes = 2 * T * kLine, stage_bytes = KS * set_bytes;
};

// Between what the lanes of a wave write to LDS and what others of them read there, and before it is written anew: the hardware takes a wave's LDS accesses in
// their order, the compiler would be free to exchange those that are at different addresses for each lane.
__device__ __forceinline__ void between_lanes() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ __forceinline__ f16x product(h8 a, h8 b, f16x c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

template <typename S, int kMode, typename O> __global__ __launch_bounds__(S::threads) void product_kernel(Group g, Step s, int turn, int total, int run) {
    constexpr int T = S::tile, kSet = S::wm * S::wn, kMT = T / S::wm / 32, kNT = T / S::wn / 32, kOctets = 2 * T / 8 / kSet;
    __shared__ __align__(1024) char lds[S::buffers * S::stage_bytes];
    // Workgroups go to the eight caches in turn: `run` neighbouring tiles, which read the same rows, to one, the next ones to the next, so that each gets as
    // many of the long ones.
    const int turn_of = blockIdx.x / 8, unit = (turn_of / run * 8 + (int)blockIdx.x % 8) * run + turn_of % run;
    if (unit >= total) return;
    const int item = item_of(g, unit);
    const Item &t = g.t[item];
    const Layout l = layout_of(t.m, t.n);
    char *base = s.workspace + t.at;
    int number = unit - g.first[item], ti, tj;
    constexpr bool kShare = kMode == kGramPart;
    const int half = half_of((t.m + T - 1) / T), share = kShare ? number / half : 0, tile_number = kShare ? number % half : number;
    number = tile_number;
    // rows of P and Q, and the length of either
    int I, J, K;
    const char *P, *Q;
    if (is_symmetric(kMode)) {
        I = J = t.m, K = kMode == kPoly ? t.m : t.n;
        P = Q = base + (kMode == kPoly ? l.a : turn ? l.x_other : l.x);
        // blocks of 4 x 4 tiles, row by row of blocks: what follows each other shares rows of either side
        const int N = (t.m + T - 1) / T;
        int row = 0, rows, diagonal, beyond;
        for (;; row += 4) {
            rows = min(4, N - row), diagonal = rows * (rows + 1) / 2, beyond = N - row - rows;
            const int all = diagonal + rows * beyond;
            if (number < all) break;
            number -= all;
        }
        if (number < diagonal) {
            int wide = rows;
            ti = row;
            while (number >= wide) number -= wide--, ++ti;
            tj = ti + number;
        } else {
            number -= diagonal;
            const int block = number / (4 * rows), inside = number % (4 * rows), width = min(4, beyond - block * 4);
            ti = row + inside / width, tj = row + rows + block * 4 + inside % width;
        }
    } else {
        I = t.n, J = K = t.m;
        P = base + (turn ? l.x_other : l.x), Q = base + l.b;
        // (eight columns of tiles at a time, for the same reason)
        const int down = (t.m + T - 1) / T, side = number / (8 * down), inside = number % (8 * down), width = min(8, (t.n + T - 1) / T - side * 8);
        ti = side * 8 + inside % width, tj = inside / width;
    }
    constexpr bool kColumns = !is_symmetric(kMode);   // P's rows are X's columns: its stages are 32 rows of X
    const int64_t pitch = pitch_of(K), x_pitch = pitch_of(t.n);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), set = wave / kSet, in_set = wave % kSet;
    const int lines = (int)(pitch / kLine), shares = kShare ? shares_of(t.m, t.n) : 1;
    const int begin = kShare ? (int)((int64_t)lines * share / shares) : 0, end = kShare ? (int)((int64_t)lines * (share + 1) / shares) : lines;
    const int stages = kMode == kGramJoin ? 0 : end - begin, rounds = (stages + S::ks - 1) / S::ks;

    // This wave's part of a stage: lines 8 at a time, each with its eight pieces of 16 bytes in an order of its own, so that what the lanes of one read want lies in
    // different ones of the 64 banks.  Of a line of row r, piece p is at p ^ (r / 2 & 7): 16 lanes read as many rows.  Of T columns of row k of X (T / 32 lines), line
    // l is at l ^ (k & 1), and piece p at p ^ 4 (k / 2 & 1): 32 lanes read 64 bytes of each of four rows.
    constexpr int kWide = T / 32;
    uint32_t from[kOctets];
#pragma unroll
    for (int q = 0; q < kOctets; ++q) {
        const int octet = in_set * kOctets + q, r = octet * 8 + (lane >> 3);
        if (kColumns && octet * 8 < T) {
            const int k = r / kWide, line = (r % kWide) ^ (k & 1);
            from[q] = (uint32_t)(k * x_pitch) + (uint32_t)(min(ti * kWide + line, (I + 31) / 32 - 1) * kLine + ((lane & 7) ^ ((k >> 1 & 1) * 4)) * 16);
            continue;
        }
        const int row = r < T ? min(ti * T + r, I - 1) : min(tj * T + r - T, J - 1);
        from[q] = (uint32_t)(row * pitch) + (uint32_t)(((lane & 7) ^ ((r >> 1) & 7)) * 16);
    }
    const uint32_t to = lds_address(lds) + set * S::set_bytes + in_set * kOctets * 1024;
    const auto load = [&](int round, int q) {
        const int stage = begin + min(round * S::ks + set, stages - 1);   // (what the last round may be short of is loaded all the same, and not used)
        const bool rows_of_p = (in_set * kOctets + q) * 8 < T;
        load_rows8_to_lds((rows_of_p ? P : Q) + stage * (kColumns && rows_of_p ? 32 * x_pitch : (int64_t)kLine), from[q], to + round % S::buffers * S::stage_bytes + q * 1024);
    };
    const auto load_stage = [&](int round) {
#pragma unroll
        for (int q = 0; q < kOctets; ++q) load(round, q);
    };
    f16x acc[kMT][kNT];
#pragma unroll
    for (int a = 0; a < kMT; ++a)
#pragma unroll
        for (int b = 0; b < kNT; ++b) acc[a][b] = (f16x)(0.f);
    const int row_i = (in_set / S::wn) * (T / S::wm), row_j = (in_set % S::wn) * (T / S::wn);
    // A stage is two halves of 16 k.  While a half's products run, the rows of the next are read and, in the second half, the stage after the next ones is
    // loaded; between the two halves of a stage all waves have read all of it, and what was loaded before is there.  Reads and loads stand between the
    // products, in this order: put before them, they hold the wave up for as long as the products take (a tile of 128 x 128 alone on its compute
    // unit: 0.88 us a stage).
    struct Half {
        h8 ph[kMT], qh[kNT], ql[kNT], pl[kMT];
    };
    constexpr int kReads = 2 * (kMT + kNT), kProducts = 3 * kMT * kNT;
    // (reads evenly among the products, loads in the first two thirds: later, or reads earlier, 2 % more)
    constexpr int kMost = kProducts * 2 / 3;
    const auto read_p = [&](const char *stage, int half, int a, bool lo) {
        if constexpr (kColumns) {
            // (the transposing read hands lane l of 16 lanes the l-th element of each of four rows: 8 k of 16 columns in two)
            s16x4 x[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int k = half * 16 + (lane >> 5) * 8 + e * 4 + (lane >> 2 & 3), piece = (lane >> 4 & 1) * 2 + (lane >> 1 & 1) + (lo ? 4 : 0);
                const char *p = stage + (k * kWide + ((row_i / 32 + a) ^ (k & 1))) * kLine + (piece ^ ((k >> 1 & 1) * 4)) * 16 + (lane & 1) * 8;
                x[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3))) *)p);
            }
            const u32x2 y = __builtin_bit_cast(u32x2, x[0]), z = __builtin_bit_cast(u32x2, x[1]);
            return __builtin_bit_cast(h8, (u32x4){y[0], y[1], z[0], z[1]});
        } else {
            return *reinterpret_cast<const h8 *>(stage + (row_i + a * 32 + (lane & 31)) * kLine + (((half * 2 + (lane >> 5)) ^ ((lane >> 1) & 7)) * 16 ^ (lo ? 64 : 0)));
        }
    };
    const auto read = [&](Half &h, int round, int half, int which) {
        const char *stage = lds + round % S::buffers * S::stage_bytes + set * S::set_bytes;
        const char *q = stage + (T + row_j + (lane & 31)) * kLine;
        const int hi_at = ((half * 2 + (lane >> 5)) ^ ((lane >> 1) & 7)) * 16, lo_at = hi_at ^ 64;
        if (which < kMT) h.ph[which] = read_p(stage, half, which, false);
        else if (which < kMT + kNT) h.qh[which - kMT] = *reinterpret_cast<const h8 *>(q + (which - kMT) * 32 * kLine + hi_at);
        else if (which < kMT + 2 * kNT) h.ql[which - kMT - kNT] = *reinterpret_cast<const h8 *>(q + (which - kMT - kNT) * 32 * kLine + lo_at);
        else h.pl[which - kMT - 2 * kNT] = read_p(stage, half, which - kMT - 2 * kNT, true);
    };
    const auto multiply = [&](const Half &h, int which) {
        const int a = which % (kMT * kNT) / kNT, b = which % kNT;
        if (which < kMT * kNT) acc[a][b] = product(h.ph[a], h.qh[b], acc[a][b]);
        else if (which < 2 * kMT * kNT) acc[a][b] = product(h.ph[a], h.ql[b], acc[a][b]);
        else acc[a][b] = product(h.pl[a], h.qh[b], acc[a][b]);
    };
    const auto wait_for_all = [&](bool more) {   // more: the loads of buffers - 2 stages may stay under way
        if (more) wait_loads<(S::buffers - 2) * kOctets>();
        else wait_loads<0>();
        __syncthreads();
    };
    if constexpr (kMode != kGramJoin) {
    Half first, second;
#pragma unroll
    for (int k = 0; k < S::buffers - 1; ++k)
        if (k < rounds) load_stage(k);
    wait_for_all(S::buffers - 1 <= rounds);
    if (S::buffers - 1 < rounds) load_stage(S::buffers - 1);
#pragma unroll
    for (int k = 0; k < kReads; ++k) read(first, 0, 0, k);
    int round = 0;
    for (; round + S::buffers < rounds; ++round) {
#pragma unroll
        for (int o = 0; o < kProducts; ++o) {
#pragma unroll
            for (int k = 0; k < kReads; ++k)
                if (k * kProducts / kReads == o) read(second, round, 1, k);
            multiply(first, o);
            __builtin_amdgcn_sched_barrier(0);
        }
        wait_for_all(true);
#pragma unroll
        for (int o = 0; o < kProducts; ++o) {
#pragma unroll
            for (int k = 0; k < kReads; ++k)
                if (k * kProducts / kReads == o) read(first, round + 1, 0, k);
#pragma unroll
            for (int k = 0; k < kOctets; ++k)
                if (k * kMost / kOctets == o) load(round + S::buffers, k);
            multiply(second, o);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    for (; round < rounds; ++round) {   // nothing more to load
        const bool mine = S::ks == 1 || round * S::ks + set < stages;
        if (mine) {
#pragma unroll
            for (int k = 0; k < kReads; ++k) read(second, round, 1, k);
#pragma unroll
            for (int o = 0; o < kProducts; ++o) multiply(first, o);
        }
        if (round + 1 < rounds) {
            wait_for_all(false);
#pragma unroll
            for (int k = 0; k < kReads; ++k) read(first, round + 1, 0, k);
        }
        if (mine) {
#pragma unroll
            for (int o = 0; o < kProducts; ++o) multiply(second, o);
        }
    }
    }
    if constexpr (S::ks > 1) {
        // the sets' sums, to the first
        static_assert(S::buffers * S::stage_bytes >= (S::ks - 1) * T * T * 4, "room for the sums");
        float *sums = reinterpret_cast<float *>(lds);
        __syncthreads();
        if (set > 0) {
#pragma unroll
            for (int a = 0; a < kMT; ++a)
#pragma unroll
                for (int b = 0; b < kNT; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r) sums[((((set - 1) * kSet + in_set) * kMT + a) * kNT + b) * 1024 + r * 64 + lane] = acc[a][b][r];
        }
        __syncthreads();
        if (set > 0) return;
#pragma unroll
        for (int other = 0; other < S::ks - 1; ++other)
#pragma unroll
            for (int a = 0; a < kMT; ++a)
#pragma unroll
                for (int b = 0; b < kNT; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[a][b][r] += sums[(((other * kSet + in_set) * kMT + a) * kNT + b) * 1024 + r * 64 + lane];
    }

    // (a part as the lanes hold it: 64 of a register next to each other)
    float *part = kMode == kGramPart || kMode == kGramJoin ? reinterpret_cast<float *>(base + l.parts) + (int64_t)tile_number * (T * T) + in_set * (kMT * kNT * 1024) + lane : nullptr;
    if constexpr (kMode == kGramPart) {
#pragma unroll
        for (int a = 0; a < kMT; ++a)
#pragma unroll
            for (int b = 0; b < kNT; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) part[(int64_t)share * half * (T * T) + (a * kNT + b) * 1024 + r * 64] = acc[a][b][r];
        return;
    }
    if constexpr (kMode == kGramJoin) {
        const int all = shares_of(t.m, t.n);
#pragma unroll 4
        for (int k = 0; k < all; ++k)
#pragma unroll
            for (int a = 0; a < kMT; ++a)
#pragma unroll
                for (int b = 0; b < kNT; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[a][b][r] += part[(int64_t)k * half * (T * T) + (a * kNT + b) * 1024 + r * 64];
    }

    // Lane l has column l % 32 of a 32 x 32 tile, and rows 8 k + 4 (l / 32) + (0 .. 3).  A tile goes out through 4 KB of LDS of the wave's own, so that stores
    // are of 16 bytes to a lane and 64 or 128 to a line.
    const float lr = kMode != kLast ? 0.f : s.lr_device ? *s.lr_device : s.lr, decay = 1.f - lr * s.weight_decay, rate = lr * t.rate;
    const int64_t out_pitch = pitch_of(J), across_pitch = pitch_of(I);
    char *out = base + (kMode == kGram || kMode == kGramJoin ? l.a : kMode == kPoly ? l.b : turn ? l.x : l.x_other), *across = out;
    __syncthreads();   // (all waves have read their stages)
    char *stage = lds + in_set * 4096;
#pragma unroll
    for (int a = 0; a < kMT; ++a)
#pragma unroll
        for (int b = 0; b < kNT; ++b) {
            const int i0 = ti * T + row_i + a * 32, j0 = tj * T + row_j + b * 32;
            if (i0 >= I || j0 >= J) continue;
            if constexpr (kMode == kLast) {
                // rows of the result: X's columns i, or its rows j
                float *rows = reinterpret_cast<float *>(stage);
                constexpr int kE = 4;
                if (t.tall) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) rows[(r / 4 * 8 + (lane >> 5) * 4 + r % 4) * 32 + (lane & 31)] = acc[a][b][r] * (1.f / (kHeld * kHeld));
                } else {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        f32x4 x;
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] = acc[a][b][q * 4 + e] * (1.f / (kHeld * kHeld));
                        *reinterpret_cast<f32x4 *>(rows + (lane & 31) * 32 + (((q * 2 + (lane >> 5)) ^ (lane & 7)) * 4)) = x;   // (in an order that spreads them over the banks)
                    }
                }
                between_lanes();
                const int r0 = t.tall ? i0 : j0, c0 = t.tall ? j0 : i0, R = t.tall ? I : J, C = t.tall ? J : I;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int r = q * 8 + (lane >> 3), n = r0 + r < R ? min(C - c0 - (lane & 7) * kE, kE) : 0;
                    const int64_t at = (int64_t)(r0 + r) * C + c0 + (lane & 7) * kE;
                    const f32x4 x = *reinterpret_cast<const f32x4 *>(rows + r * 32 + (t.tall ? (lane & 7) : (lane & 7) ^ (r & 7)) * kE);
                    float v[kE] = {x[0], x[1], x[2], x[3]};
                    Piece<O, kE> w;
                    if (s.update) {
                        Piece<float, kE> master;
                        float old[kE];
                        if (t.master) {
                            master.template load<false>(t.master + at, n);
                            unpack(master, old);
                        } else {
                            w.template load<false>(static_cast<const O *>(t.out) + at, n);
                            unpack(w, old);
                        }
#pragma unroll
                        for (int e = 0; e < kE; ++e) v[e] = old[e] * decay - rate * v[e];
                        if (t.master) {
                            pack(v, master);
                            master.template store<false>(t.master + at, n);
                        }
                    }
                    pack(v, w);
                    w.template store<false>(static_cast<O *>(t.out) + at, n);
                }
            } else {
                // rows of `across`, j, with their pieces in the order that stages have too
                const int j = j0 + (lane & 31), turned = (lane >> 1) & 7;
                char *row = stage + (lane & 31) * kLine;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int i = i0 + q * 8 + (lane >> 5) * 4;
                    float v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = acc[a][b][q * 4 + e];
                    if constexpr (kMode == kPoly) {
                        // (A is symmetric: four of a row instead of a column's)
                        const char *gram = base + l.a + min(j, J - 1) * across_pitch + (int64_t)(i0 / 32) * kLine + (i - i0) * 2;
                        const h4 hi = *reinterpret_cast<const h4 *>(gram), lo = *reinterpret_cast<const h4 *>(gram + 64);
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] = v[e] * (s.c / kHeld) + s.b * ((float)hi[e] + (float)lo[e]) + (i + e == j ? s.a * kHeld : 0.f);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] *= 1.f / kHeld;
                    }
                    h4 hi, lo;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        f16_t x, y;
                        split(i + e < I && j < J ? v[e] : 0.f, x, y);
                        hi[e] = x, lo[e] = y;
                    }
                    *reinterpret_cast<h4 *>(row + (q ^ turned) * 16 + (lane >> 5) * 8) = hi;
                    *reinterpret_cast<h4 *>(row + ((q + 4) ^ turned) * 16 + (lane >> 5) * 8) = lo;
                }
                between_lanes();
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int r = q * 8 + (lane >> 3), piece = lane & 7;
                    const u32x4 x = *reinterpret_cast<const u32x4 *>(stage + r * kLine + ((piece ^ (r >> 1)) & 7) * 16);
                    if (j0 + r < J) *reinterpret_cast<u32x4 *>(across + (j0 + r) * across_pitch + (int64_t)(i0 / 32) * kLine + piece * 16) = x;
                }
                if (kMode != kApply && ti != tj) {
                    // rows of `out`, i: the transposing read hands lane l of 16 lanes the l-th element of each of four rows j
                    const int group = lane >> 4, l16 = lane & 15;
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const int i = i0 + half * 16 + l16;
#pragma unroll
                        for (int part = 0; part < 2; ++part) {   // hi, lo
                            s16x4 x[2];
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                const int r = group * 8 + k * 4 + (l16 >> 2), piece = part * 4 + half * 2 + (l16 >> 1 & 1);
                                const char *p = stage + r * kLine + ((piece ^ (r >> 1)) & 7) * 16 + (l16 & 1) * 8;
                                x[k] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3))) *)p);
                            }
                            const u32x2 y = __builtin_bit_cast(u32x2, x[0]), z = __builtin_bit_cast(u32x2, x[1]);
                            if (i < I) *reinterpret_cast<u32x4 *>(out + i * out_pitch + (int64_t)(j0 / 32) * kLine + part * 64 + group * 16) = (u32x4){y[0], y[1], z[0], z[1]};
                        }
                    }
                }
            }
            between_lanes();   // (the next tile goes out through the same 4 KB)
        }
}

// ---- matrices of at most 64 rows (or columns) ----
//
// A and B are one tile, and what a step costs is launches and latency.  So a step is one launch: a workgroup adds up the parts of A that the launch before left,
// forms B (each for itself), multiplies its columns of X by it 64 at a time, and leaves its part of the new A.  10 matrices of 32 x 2048: 17 launches of
// the general form 150 us of kernels.
constexpr int kThinRegion = 2 * kThin * kLine;   // 64 rows of 64 k

// LDS operands: 64 rows of kThin k as lines of 32 k, pieces in the order that stages have.
__device__ __forceinline__ char *thin_piece(char *region, int row, int block, int piece) {
    return region + (block * kThin + row) * kLine + ((piece ^ (row >> 1)) & 7) * 16;
}
__device__ __forceinline__ h8 thin_read(char *region, int row, int k, bool lo) {   // k: a multiple of 8
    return *reinterpret_cast<const h8 *>(thin_piece(region, row, k / 32, k % 32 / 8 + (lo ? 4 : 0)));
}
// 32 x 32 of P Q^T from row_i of P and row_j of Q on, over `blocks` times 32 k
__device__ __forceinline__ void thin_product(char *p, char *q, int row_i, int row_j, int blocks, int lane, f16x &acc) {
    for (int block = 0; block < blocks; ++block)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int k = block * 32 + half * 16 + (lane >> 5) * 8;
            const h8 ph = thin_read(p, row_i + (lane & 31), k, false), pl = thin_read(p, row_i + (lane & 31), k, true);
            const h8 qh = thin_read(q, row_j + (lane & 31), k, false), ql = thin_read(q, row_j + (lane & 31), k, true);
            acc = product(ph, qh, acc);
            acc = product(ph, ql, acc);
            acc = product(pl, qh, acc);
        }
}
// A 32 x 32 tile (lane l has column l % 32, rows 8 k + 4 (l / 32) + (0 .. 3); values times kHeld) as rows of its columns.
__device__ __forceinline__ void thin_put(char *region, int row_i, int row_j, int lane, const float (&v)[16]) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        h4 hi, lo;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f16_t x, y;
            split(v[q * 4 + e], x, y);
            hi[e] = x, lo[e] = y;
        }
        *reinterpret_cast<h4 *>(thin_piece(region, row_j + (lane & 31), row_i / 32, q) + (lane >> 5) * 8) = hi;
        *reinterpret_cast<h4 *>(thin_piece(region, row_j + (lane & 31), row_i / 32, q + 4) + (lane >> 5) * 8) = lo;
    }
}

enum { kThinFirst = 0, kThinStep = 1, kThinLast = 2 };   // X0 and its part of A; a step; the last step, into the result

// turn: which of two sets of parts of A is written (the other is read).
template <int kPhase, typename O> __global__ __launch_bounds__(kThreads) void thin_kernel(Group g, Step s, int turn) {
    __shared__ __align__(1024) char ra[kThinRegion], rb[kThinRegion], rx[kThinRegion], rr[kThinRegion];
    __shared__ float tile[kPhase == kThinFirst ? kThin : 1][kThin + 1];
    __shared__ double part[kThreads / 64];
    const int item = item_of(g, blockIdx.x);
    const Item &t = g.t[item];
    const Layout l = layout_of(t.m, t.n);
    char *base = s.workspace + t.at, *xt = base + l.x_other;
    const int m = t.m, n = t.n, number = blockIdx.x - g.first[item], parts = g.first[item + 1] - g.first[item];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int bi = wave / 2 * 32, bj = wave % 2 * 32, down = (m + 31) / 32;   // this wave's 32 x 32 of a tile; 32s of m
    const int64_t pitch = pitch_of(m);
    f32x4 *sums = reinterpret_cast<f32x4 *>(base + l.x);
    const int part_size = down * down * 256, most_parts = thin_parts_of(n);   // f32x4s: 4 to a lane of each 32 x 32
    const int my_part = (bi / 32 * down + bj / 32) * 256 + lane;
    const bool of_a = bi < m && bj < m;

    double norm2 = 0.;
    if constexpr (kPhase == kThinFirst) {
        const double *squares = reinterpret_cast<const double *>(base + l.sums);
        const int chunks = (int)(((int64_t)m * n + kChunk - 1) / kChunk);
        double sum = 0.;
        for (int i = threadIdx.x; i < chunks; i += kThreads) sum += squares[i];
        norm2 = block_sum(sum, part);
    } else {
        float a[16];
        if (of_a) {
            f32x4 v[4];
            const f32x4 *from = sums + (int64_t)(turn ^ 1) * most_parts * part_size + my_part;
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] = from[q * 64];
#pragma unroll 5
            for (int p = 1; p < parts; ++p)
#pragma unroll
                for (int q = 0; q < 4; ++q) v[q] += from[(int64_t)p * part_size + q * 64];
#pragma unroll
            for (int r = 0; r < 16; ++r) a[r] = v[r / 4][r % 4] * (1.f / kHeld);
            thin_put(ra, bi, bj, lane, a);   // (symmetric)
        }
        __syncthreads();
        if (of_a) {
            f16x acc = (f16x)(0.f);
            thin_product(ra, ra, bi, bj, down, lane, acc);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int i = bi + r / 4 * 8 + (lane >> 5) * 4 + r % 4, j = bj + (lane & 31);
                a[r] = i < m && j < m ? acc[r] * (s.c / kHeld) + s.b * a[r] + (i == j ? s.a * kHeld : 0.f) : 0.f;
            }
            thin_put(rb, bi, bj, lane, a);
        }
    }

    const Scale scale(norm2, s.eps);
    f16x gram = (f16x)(0.f);
    const int across = (n + kThin - 1) / kThin;
    const float lr = kPhase != kThinLast ? 0.f : s.lr_device ? *s.lr_device : s.lr, decay = 1.f - lr * s.weight_decay, rate = lr * t.rate;
    for (int block = number; block < across; block += parts) {
        const int j0 = block * kThin;
        __syncthreads();   // (the last block's rows have been read)
        if constexpr (kPhase == kThinFirst) {
            // U's rows are X's, or its columns
            const int rows = t.tall ? n : m, columns = t.tall ? m : n, r0 = t.tall ? j0 : 0, c0 = t.tall ? 0 : j0;
#pragma unroll 4
            for (int k = 0; k < kThin / 4; ++k) {
                const int r = r0 + k * 4 + wave, c = c0 + lane;
                float v = 0.f;
                if (r < rows && c < columns) {
                    const int64_t at = (int64_t)r * columns + c;
                    v = load1(static_cast<const O *>(t.grad) + at);
                    if (t.momentum) {
                        const float b = t.momentum[at];
                        v = s.nesterov ? v * s.kept + b * s.momentum : b;
                    }
                }
                tile[k * 4 + wave][lane] = scale(v);
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < kThin * 8 / kThreads; ++k) {
                const int which = k * kThreads + threadIdx.x, q = which % 8 * 8, r = which / 8;
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = t.tall ? tile[r][q + e] : tile[q + e][r];   // column j0 + r of X
                if (j0 + r < n && q < down * 32) store_pair8(xt + (j0 + r) * pitch, q, v);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = t.tall ? tile[q + e][r] : tile[r][q + e];   // row r of X
                h8 hi, lo;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    f16_t x, y;
                    split(v[e], x, y);
                    hi[e] = x, lo[e] = y;
                }
                *reinterpret_cast<h8 *>(thin_piece(rr, r, q / 32, q % 32 / 8)) = hi;
                *reinterpret_cast<h8 *>(thin_piece(rr, r, q / 32, q % 32 / 8 + 4)) = lo;
            }
        } else {
            for (int k = threadIdx.x; k < kThin * down * 8; k += kThreads) {
                const int piece = k & 7, q = k / 8 % down, r = k / 8 / down;
                *reinterpret_cast<u32x4 *>(thin_piece(rx, r, q, piece)) = *reinterpret_cast<const u32x4 *>(xt + min(j0 + r, n - 1) * pitch + q * kLine + piece * 16);
            }
            __syncthreads();
            f16x acc = (f16x)(0.f);
            if (bi < m) thin_product(rb, rx, bi, bj, down, lane, acc);
            float v[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int i = bi + r / 4 * 8 + (lane >> 5) * 4 + r % 4;
                v[r] = i < m && j0 + bj + (lane & 31) < n ? acc[r] * (1.f / kHeld) : 0.f;
            }
            if constexpr (kPhase == kThinLast) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int i = bi + r / 4 * 8 + (lane >> 5) * 4 + r % 4, j = j0 + bj + (lane & 31);
                    if (i >= m || j >= n) continue;
                    const int64_t at = t.tall ? (int64_t)j * m + i : (int64_t)i * n + j;
                    O *out = static_cast<O *>(t.out) + at;
                    float x = v[r] * (1.f / kHeld);
                    if (s.update) {
                        x = (t.master ? t.master[at] : load1(out)) * decay - rate * x;
                        if (t.master) t.master[at] = x;
                    }
                    store1(out, x);
                }
            } else {
                __syncthreads();   // (rx has been read, its rows are the new ones from here on)
                if (bi < down * 32) {
                    thin_put(rx, bi, bj, lane, v);
                    between_lanes();
                    // the same as rows of X: the transposing read hands lane l of 16 lanes the l-th element of each of four rows
                    const int group = lane >> 4, l16 = lane & 15;
#pragma unroll
                    for (int half = 0; half < 2; ++half)
#pragma unroll
                        for (int lo = 0; lo < 2; ++lo) {
                            s16x4 x[2];
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                const char *p = thin_piece(rx, bj + group * 8 + k * 4 + (l16 >> 2), bi / 32, lo * 4 + half * 2 + (l16 >> 1 & 1)) + (l16 & 1) * 8;
                                x[k] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3))) *)p);
                            }
                            const u32x2 y = __builtin_bit_cast(u32x2, x[0]), z = __builtin_bit_cast(u32x2, x[1]);
                            *reinterpret_cast<u32x4 *>(thin_piece(rr, bi + half * 16 + l16, bj / 32, group + lo * 4)) = (u32x4){y[0], y[1], z[0], z[1]};
                        }
                }
                __syncthreads();
                for (int k = threadIdx.x; k < kThin * down * 8; k += kThreads) {
                    const int piece = k & 7, q = k / 8 % down, r = k / 8 / down;
                    if (j0 + r < n) *reinterpret_cast<u32x4 *>(xt + (j0 + r) * pitch + q * kLine + piece * 16) = *reinterpret_cast<const u32x4 *>(thin_piece(rx, r, q, piece));
                }
            }
        }
        if constexpr (kPhase != kThinLast) {
            if (kPhase == kThinFirst) __syncthreads();
            if (of_a) thin_product(rr, rr, bi, bj, 2, lane, gram);
        }
    }
    if (kPhase != kThinLast && of_a) {
        f32x4 *to = sums + ((int64_t)turn * most_parts + number) * part_size + my_part;
#pragma unroll
        for (int q = 0; q < 4; ++q) to[q * 64] = (f32x4){gram[q * 4], gram[q * 4 + 1], gram[q * 4 + 2], gram[q * 4 + 3]};
    }
}

template <typename F> hipError_t by_type(int dtype, F &&f) {
    if (dtype == kBF16) f(bf16_t{});
    else if (dtype == kF16) f(f16_t{});
    else f(float{});
    return hipGetLastError();
}

template <typename O> void launch_thin(hipStream_t st, Group &g, Step s, int steps, const double *coefficients) {
    // (workgroups to a matrix: each of them reads all of their parts; as many as it may have parts while there are few matrices)
    int total = 0;
    for (int i = 0; i < g.count; ++i) {
        g.first[i] = total;
        total += std::min(thin_parts_of(g.t[i].n), std::max(4, 512 / g.count));
    }
    g.first[g.count] = total;
    hipLaunchKernelGGL((thin_kernel<kThinFirst, O>), dim3(total), dim3(kThreads), 0, st, g, s, 0);
    for (int step = 0; step < steps; ++step) {
        s.a = (float)coefficients[3 * step], s.b = (float)coefficients[3 * step + 1], s.c = (float)coefficients[3 * step + 2];
        if (step + 1 < steps) hipLaunchKernelGGL((thin_kernel<kThinStep, O>), dim3(total), dim3(kThreads), 0, st, g, s, step & 1 ^ 1);
        else hipLaunchKernelGGL((thin_kernel<kThinLast, O>), dim3(total), dim3(kThreads), 0, st, g, s, step & 1 ^ 1);
    }
}

// One launch of products over all matrices of a group.
template <typename S, int kMode, typename O> void launch_tiles(hipStream_t st, Group &g, const Step &s, int turn) {
    int total = 0;
    for (int i = 0; i < g.count; ++i) {
        g.first[i] = total;
        const int down = tiles(g.t[i].m, S::tile);
        total += is_symmetric(kMode) ? half_of(down) * (kMode == kGramPart ? shares_of(g.t[i].m, g.t[i].n) : 1) : down * tiles(g.t[i].n, S::tile);
    }
    g.first[g.count] = total;
    const int run = std::min(32, (total + 7) / 8);
    hipLaunchKernelGGL((product_kernel<S, kMode, O>), dim3((total + 8 * run - 1) / (8 * run) * 8 * run), dim3(S::threads), 0, st, g, s, turn, total, run);
}

int64_t tiles_of(const Group &g, int tile, bool symmetric) {
    int64_t all = 0;
    for (int i = 0; i < g.count; ++i) {
        const int64_t down = tiles(g.t[i].m, tile);
        all += symmetric ? down * (down + 1) / 2 : down * tiles(g.t[i].n, tile);
    }
    return all;
}

// The largest tiles of which there are enough.  Per operation a tile of 256 moves half of what one of 128 does, which counts where the chip's power sets the clock; of
// 128, two workgroups of two buffers fit a compute unit, and where there is no second, one of eight waves and four buffers is faster; fewer leave units idle, and tiles of
// 64 have the same two forms.  By 256 / 128 twice / 128 alone / 64 twice / 64 alone, a whole call in us, what is taken in brackets:
//   8 of 2048 x 2048  4644 [4161] 4481 6062 6805     16 of 1024 x 1024  1294 [1303] 1447 1610 1854     1 of 512 x 2048    905 403 327 226 [180]
//   4 of 1024 x 1024   952 461 [423] 538 568          8 of 512 x 512      596 273 244 [212] 251         1 of 1024 x 1024   918 409 332 235 [188]
// and 256 for B X of 16 of 2048 x 2048 and more (1190 for 1250 of 12 with 4 of 2048 x 7168, whose A and A A, 768 tiles, take 833 and 529 for 682 and 434).
template <int kMode, typename O> void launch_products(hipStream_t st, Group &g, const Step &s, int turn) {
    constexpr bool symmetric = is_symmetric(kMode);
    const int64_t of_128 = tiles_of(g, 128, symmetric);
    if (tiles_of(g, 256, symmetric) >= 1024) launch_tiles<TileShape<256, 2, 4, 1, 2>, kMode, O>(st, g, s, turn);
    else if (of_128 > 256) launch_tiles<TileShape<128, 2, 2, 1, 2>, kMode, O>(st, g, s, turn);
    else if (of_128 >= 128) launch_tiles<TileShape<128, 2, 4, 1, 4>, kMode, O>(st, g, s, turn);
    else if (tiles_of(g, 64, symmetric) <= 256) launch_tiles<TileShape<64, 2, 2, 2, 4>, kMode, O>(st, g, s, turn);
    else launch_tiles<TileShape<64, 2, 2, 2, 2>, kMode, O>(st, g, s, turn);
}

template <typename O> void launch_steps(hipStream_t st, Group &by_n, Step s, int steps, const double *coefficients) {
    // (the longest products first: what is begun last is done soon)
    Group by_m = by_n;
    std::sort(by_n.t, by_n.t + by_n.count, [](const Item &x, const Item &y) { return x.n != y.n ? x.n > y.n : x.at < y.at; });
    std::sort(by_m.t, by_m.t + by_m.count, [](const Item &x, const Item &y) { return x.m != y.m ? x.m > y.m : x.at < y.at; });
    for (int step = 0; step < steps; ++step) {
        s.a = (float)coefficients[3 * step], s.b = (float)coefficients[3 * step + 1], s.c = (float)coefficients[3 * step + 2];
        if (kind_of(by_n.t[0].m, by_n.t[0].n) == kLongMatrix) {   // (a group is of one kind)
            launch_tiles<TileShape<kLongTile, 2, 2, 2, 4>, kGramPart, float>(st, by_n, s, step & 1);
            launch_tiles<TileShape<kLongTile, 2, 2, 1, 2>, kGramJoin, float>(st, by_n, s, step & 1);
        } else {
            launch_products<kGram, float>(st, by_n, s, step & 1);
        }
        launch_products<kPoly, float>(st, by_m, s, 0);
        if (step + 1 < steps) launch_products<kApply, float>(st, by_m, s, step & 1);
        else launch_products<kLast, O>(st, by_m, s, step & 1);
    }
}

}  // namespace

size_t muon_matrix_bytes(int64_t rows, int64_t columns) {
    return (size_t)layout_of((int)std::min(rows, columns), (int)std::max(rows, columns)).end;
}

hipError_t muon(hipStream_t st, int dtype, int64_t count, const MuonMatrix *matrices, const MuonStep &a, void *workspace, size_t workspace_bytes) {
    const Step s{(float)a.momentum, (float)(1. - a.momentum), a.nesterov, a.update, (float)a.weight_decay, (float)a.lr, a.eps, a.lr_device, 0.f, 0.f, 0.f,
                 static_cast<char *>(workspace)};
    // groups of each kind, as they fit into a launch's arguments and the workspace
    int64_t next[kKinds] = {};
    for (int kind = 0; kind < kKinds;) {
        Group g{};
        size_t used = 0;
        int64_t &at = next[kind];
        for (; at < count && g.count < kGroup; ++at) {
            const MuonMatrix &t = matrices[at];
            if (t.rows == 0 || t.columns == 0 || kind_of((int)std::min(t.rows, t.columns), (int)std::max(t.rows, t.columns)) != kind) continue;
            const size_t bytes = muon_matrix_bytes(t.rows, t.columns);
            if (g.count > 0 && used + bytes > workspace_bytes) break;
            g.t[g.count++] = Item{t.grad, t.momentum, t.out, t.master, (int64_t)used, (int)std::min(t.rows, t.columns), (int)std::max(t.rows, t.columns), (float)t.rate,
                                  t.rows > t.columns};
            used += bytes;
        }
        if (g.count == 0) {
            ++kind;
            continue;
        }
        const hipError_t e = by_type(dtype, [&](auto type) {
            using O = decltype(type);
            int total = 0;
            for (int i = 0; i < g.count; ++i) g.first[i] = total, total += (int)(((int64_t)g.t[i].m * g.t[i].n + kChunk - 1) / kChunk);
            g.first[g.count] = total;
            hipLaunchKernelGGL((momentum_kernel<O>), dim3(total), dim3(kThreads), 0, st, g, s);
            if (kind == kThinMatrix) {
                launch_thin<O>(st, g, s, a.steps, a.coefficients);
                return;
            }
            total = 0;
            for (int i = 0; i < g.count; ++i) g.first[i] = total, total += tiles(g.t[i].m, kSpread) * tiles(g.t[i].n, kSpread);
            g.first[g.count] = total;
            hipLaunchKernelGGL((spread_kernel<O>), dim3(total), dim3(kThreads), 0, st, g, s);
            launch_steps<O>(st, g, s, a.steps, a.coefficients);
        });
        if (e != hipSuccess) return e;
    }
    return hipGetLastError();
}

}  // namespace wkv6
