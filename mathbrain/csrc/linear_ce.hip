// Softmax cross entropy of a linear layer's outputs, without keeping them, with its gradients, on gfx950.
//
//   s_nv = h_n . w_v,   loss_n = log sum_v exp(s_nv) - s_n,t(n)
//   U_nv = exp(s_nv) / sum_v' exp(s_nv') - [v = t(n)],   dh_n = g_n sum_v U_nv w_v,   dw_v = sum_n U_nv (g_n h_n)
//
// with the loss's gradient g_n of each row.  Rows with the ignored target have loss 0 and g_n = 0.
//
// Bound by the matrix instructions (gemm16.h).  Forward: workgroups take tiles of vocabulary x rows; a lane holds
// the tile's vocabulary entries of a row in registers, so the tile's maximum and sum of exponentials need one
// exchange; they go to memory, two floats for a tile's row, and a second kernel joins them in a fixed order.
// Backward, for pieces of the vocabulary: the tile again, U as 16-bit planes to memory, then the two products with it.
// Recomputing the scores takes the time of one product; keeping them would take N V values.
//
// For bf16 tensors U (times 2^15), w and g h (each matrix times one power of two) are single fp16 planes: U and g h are rounded
// to 11 bits (elementwise tensor operations in bf16 would round them to 8), w is exact down to 2^-31 of the matrix's largest
// value (plane_scale).  U's step is never below 2^-39: a probability has the 8 bits of a bf16 result down to 2^-32, and
// one below 2^-40 counts as none, so dw of a word that improbable in every row is zero.
//
// For fp32 tensors they are two fp16 planes, 24 bits, with a power of two for every row of hidden and of the weights, and for
// every row and word of a tile of U (scaled_u): what is held is as exact as fp32 down to 2^-16 of the largest value of its own row
// (or of its word's or row's terms in the sum), whatever other rows and words hold.
//
// A row's sum of exponentials is kept as maximum and logarithm (of base 2), two floats, so that neither the loss nor a
// probability rounds their sum.
#include "gemm16.h"

#include <algorithm>
#include <climits>
#include <cstdint>

namespace mb {
namespace {

using namespace g16;

constexpr int kThreads = 256;       // of the kernels around the products
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kUScale = 32768.f;
constexpr int kMaxBlocks = 2048;     // of the kernels that look for the largest value
constexpr int kRowRuns = 512;       // of the kernel that finds the rows' places
constexpr int kRowsPerBlock = 16;   // of the joining kernel
constexpr int kLeastExp = -126;     // of a row of fp32 values

// e^x.  Scores are natural ones, and the difference is taken before the factor: of equal scores it is 0, however large they are.
__device__ inline float exp_of(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

struct Targets {
    const void* target;
    int bytes;
    int64_t ignore, V;
    // the row's target, -1 where it is ignored, -2 where it is outside the vocabulary
    __device__ int at(int64_t n) const {
        const int64_t t = bytes == 8 ? ((const int64_t*)target)[n] : (int64_t)((const int32_t*)target)[n];
        return t == ignore ? -1 : t < 0 || t >= V ? -2 : (int)t;
    }
};
// The rows that the scores are taken for: with many rows those that count alone, next to each other (`rows` their
// numbers, `pos` each row's place or -1, `m` how many); otherwise all, in their places.
struct Rows {
    const int *rows, *pos, *m;
    int N;
    __device__ int count() const { return m ? __builtin_amdgcn_readfirstlane(*m) : N; }
    __device__ int at(int c) const { return rows ? rows[c] : c; }
    __device__ int of(int64_t n) const { return pos ? pos[n] : (int)n; }
};
// The gradient of each row's loss.
struct RowGrad {
    Targets t;
    const float* dloss;      // [N] (reduction 0) or one
    const float* count;      // rows that count (reduction 1)
    int reduction;
    __device__ float at(int64_t n) const {
        if (t.at(n) == -1) return 0.f;
        return reduction == 0 ? dloss[n] : reduction == 1 ? dloss[0] / count[0] : dloss[0];
    }
};

__device__ inline float block_max(float v) {
    __shared__ float s[kThreads / 64];
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    return fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
}

template <typename T>
__device__ inline void load8(const T* p, bool vec, int left, float* v) {
    if (vec && left >= 8) {
        typedef T vec8 __attribute__((ext_vector_type(8), aligned(16)));
        const vec8 q = *reinterpret_cast<const vec8*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)q[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < left ? (float)p[i] : 0.f;
    }
}

// Places for the rows that count.  A workgroup takes a run of rows, and first counts what counts before it: its targets are
// read by the workgroups behind it, too, out of L2, and nobody waits for another.
__global__ void __launch_bounds__(kThreads) ce_rows_kernel(const Targets t, int N, int each, int* rows, int* pos, int* m) {
    __shared__ int s[64];
    const int n0 = blockIdx.x * each, n1 = min(N, n0 + each);
    int before = 0, total;
#pragma unroll 16
    for (int n = threadIdx.x; n < n0; n += kThreads) before += t.at(n) != -1;
    block_exclusive_scan(before, s, total);
    int base = total;
    for (int n = n0; n < n1; n += kThreads) {
        const int i = n + (int)threadIdx.x;
        const bool counts = i < n1 && t.at(i) != -1;
        const int c = base + block_exclusive_scan(counts, s, total);
        if (i < n1) pos[i] = counts ? c : -1;
        if (counts) rows[c] = i;
        base += total;
    }
    if (n1 == N && threadIdx.x == 0) *m = base;
}

// A user's matrix [rows, D], rows ld apart, with what the scaling and the copies of it want to know.
struct Matrix {
    const void* p;
    int64_t ld;
    int rows, D, vec;
    int graded;                  // 1: times each row's g; 1 or 2: an ignored row counts for nothing, whatever it holds
    float* largest;              // the largest magnitudes of the workgroups' parts; copies without: not scaled
    int blocks, copy_blocks;
    float* scale;
    int* exps;                   // of the rows' copies
    void* out;                   // planes [rows_pad, Dp]
    int rows_pad, Dp, gathered;  // gathered: rows in their places of Rows
};
// Up to three matrices a launch, each with workgroups of its own.
constexpr int kMatrices = 3;
struct Set {
    Matrix x[kMatrices];
    int n, first[kMatrices];     // their first workgroups
    RowGrad g;
    Rows r;
    __device__ const Matrix& mine(int& block) const {
        int i = 0;
        while (i + 1 < n && (int)blockIdx.x >= first[i + 1]) ++i;
        block = (int)blockIdx.x - first[i];
        return x[i];
    }
};

// The largest finite magnitude of each workgroup's part of x (graded: of g_n x_n).
template <typename T>
__global__ void __launch_bounds__(kThreads) ce_largest_kernel(const Set a) {
    int block;
    const Matrix& x = a.mine(block);
    const int pieces = (x.D + 7) / 8;
    float most = 0.f;
#pragma unroll 4
    for (int64_t i = (int64_t)block * kThreads + threadIdx.x; i < (int64_t)x.rows * pieces; i += (int64_t)x.blocks * kThreads) {
        const int64_t n = i / pieces;
        const int d = (int)(i - n * pieces) * 8;
        const float gn = !x.graded ? 1.f : x.graded == 1 ? fabsf(a.g.at(n)) : a.g.t.at(n) == -1 ? 0.f : 1.f;
        if (gn == 0.f) continue;
        float v[8];
        load8((const T*)x.p + n * x.ld + d, x.vec, x.D - d, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float m = fabsf(v[e]) * gn;
            most = fmaxf(most, m < INFINITY ? m : 0.f);
        }
    }
    most = block_max(most);
    if (threadIdx.x == 0) x.largest[block] = most;
}

__device__ inline float scale_from(const float* part, int n) {
    float m = 0.f;
    for (int i = threadIdx.x; i < n; i += kThreads) m = fmaxf(m, part[i]);
    return plane_scale(__builtin_bit_cast(uint32_t, block_max(m)));
}

// x (graded: g_n x_n) as a plane [rows_pad, Dp] of O, zeros around it, scaled by its largest value, which goes to *scale.
template <typename T, typename O>
__global__ void __launch_bounds__(kThreads) ce_planes_kernel(const Set a) {
    int block;
    const Matrix& x = a.mine(block);
    float s = 1.f;
    if (x.largest) {
        s = scale_from(x.largest, x.blocks);
        if (block == 0 && threadIdx.x == 0) *x.scale = s;
    }
    const int pieces = x.Dp / 8, count = x.gathered ? a.r.count() : x.rows;
    O* out = (O*)x.out;
    typedef O vec8 __attribute__((ext_vector_type(8), aligned(16)));
    for (int64_t i = (int64_t)block * kThreads + threadIdx.x; i < (int64_t)x.rows_pad * pieces; i += (int64_t)x.copy_blocks * kThreads) {
        const int64_t n = i / pieces;
        const int d = (int)(i - n * pieces) * 8;
        float v[8] = {};
        if (n < count) {
            const int64_t row = x.gathered ? a.r.at((int)n) : n;
            const float gn = !x.graded ? 1.f : x.graded == 1 ? a.g.at(row) : a.g.t.at(row) == -1 ? 0.f : 1.f;
            load8((const T*)x.p + row * x.ld + d, x.vec, x.D - d, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = gn == 0.f ? 0.f : v[e] * gn * s;
        }
        vec8 y;
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = (O)v[e];
        *reinterpret_cast<vec8*>(out + n * x.Dp + d) = y;
    }
}

// fp32 rows as two fp16 planes [rows_pad, Dp], zeros around them and in place of ignored rows; each row by its own power of
// two, 2^(14 - exps[n]), which brings its largest finite value to 2^14 .. 2^15.  A wave a row; the second read comes out of the caches.
__global__ void __launch_bounds__(kThreads) ce_row_planes_kernel(const Set a) {
    int block;
    const Matrix& x = a.mine(block);
    const int lane = threadIdx.x & 63, count = x.gathered ? a.r.count() : x.rows;
    _Float16* out = (_Float16*)x.out;
    for (int64_t n = (int64_t)block * (kThreads / 64) + wave_id(); n < x.rows_pad; n += (int64_t)x.copy_blocks * (kThreads / 64)) {
        bool there = n < count;
        int64_t row = 0;
        if (there) {
            row = x.gathered ? a.r.at((int)n) : n;
            there = !x.graded || a.g.t.at(row) != -1;
        }
        const float* from = (const float*)x.p + row * x.ld;
        float most = 0.f, v[8];
        if (there)
#pragma unroll 4
            for (int d = lane * 8; d < x.D; d += 512) {
                load8(from + d, x.vec, x.D - d, v);
#pragma unroll
                for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(v[e]) < INFINITY ? fabsf(v[e]) : 0.f);
            }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
        const int exp = std::max(kLeastExp, (int)(__builtin_bit_cast(uint32_t, most) >> 23) - 127);
        if (lane == 0) x.exps[n] = exp;
#pragma unroll 4
        for (int d = lane * 8; d < x.Dp; d += 512) {
            if (there) load8(from + d, x.vec, x.D - d, v);
            f16x8 hi, lo;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                _Float16 h, l;
                split(there ? __builtin_amdgcn_ldexpf(v[e], 14 - exp) : 0.f, h, l);
                hi[e] = h, lo[e] = l;
            }
            *reinterpret_cast<f16x8*>(out + n * x.Dp + d) = hi;
            *reinterpret_cast<f16x8*>(out + ((int64_t)x.rows_pad + n) * x.Dp + d) = lo;
        }
    }
}

// Tiles to workgroups: each of the eight XCDs, to which workgroups go in turn, takes a run of the tiles, in which
// eight tiles of rows walk the vocabulary together: what is at work at once on an XCD fits its L2.
constexpr int kXcds = 8, kTogether = 8;
__device__ inline bool tile_of(int tiles_p, int tiles_q, int& p, int& q) {
    const int64_t tiles = (int64_t)tiles_p * tiles_q, each = (tiles + kXcds - 1) / kXcds;
    const int64_t id = (int64_t)(blockIdx.x % kXcds) * each + blockIdx.x / kXcds;
    if (blockIdx.x / kXcds >= each || id >= tiles) return false;
    const int64_t run = (int64_t)tiles_p * kTogether;
    const int group = (int)(id / run), rest = (int)(id - group * run);
    const int wide = min(kTogether, tiles_q - group * kTogether);
    p = rest / wide;
    q = group * kTogether + rest % wide;
    return true;
}
inline unsigned tile_grid(int64_t tiles) { return (unsigned)pad(tiles, kXcds); }

struct ScoreArgs {
    Side w, h;                    // kRows: [V, Dp], [N, Dp]
    const int *exp_w, *exp_h;     // fp32: the rows' exponents
    RowGrad g;
    Rows r;
    int V, N, Dp, tiles_p;
    float2* part;                 // forward: [tiles_p, N] maximum and sum
    float* target_score;          // forward: [N]
    const float* lse;             // backward: [2, N]
    _Float16* u;                  // backward: [PL][rows, width], the piece's entries from v0 on; fp32: for dh
    _Float16* u_w;                // fp32: the same for dw
    int *exps_h, *exps_w;         // fp32: [tiles of the vocabulary, Np] and [tiles of rows, width]
    int Np;
    int v0, v1;
    int64_t plane, width;         // elements to the second plane, and to the next row
};

// fp32 operands are planes scaled row by row: the scores have the exponents of both.
template <typename P>
constexpr bool kScaled = std::is_same<typename P::T, _Float16>::value;
struct alignas(16) Int4 {
    int v[4];
};
// The exponents of this lane's words (the array has whole tiles; what lies behind the vocabulary is not used).
template <typename P>
struct WordExps {
    Int4 v[P::FP][4];
    __device__ WordExps(const ScoreArgs& a, int p0) {
#pragma unroll
        for (int i = 0; i < P::FP; ++i)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                if constexpr (kScaled<P>) v[i][r / 4] = *reinterpret_cast<const Int4*>(a.exp_w + p0 + P::row(i, r));
    }
    __device__ int at(int i, int r) const { return kScaled<P> ? v[i][r / 4].v[r % 4] : 0; }
};
template <typename P>
__device__ inline int row_exp(const ScoreArgs& a, int place, int count) { return kScaled<P> && place < count ? a.exp_h[place] : 0; }
template <typename P>
__device__ inline float score_of(float sum, int exps) { return kScaled<P> ? __builtin_amdgcn_ldexpf(sum, exps - 28) : sum; }

// Matrix instructions bound it: 28672 rows, 50257 words of 512 in bf16 1.54 - 1.60 ms, 922 - 960 TFLOP/s; 16 rows 13.8 us, the weights' 51 MB at
// 3.7 TB/s.
template <typename P>
__global__ void __launch_bounds__(P::kThreads, P::kWaves) ce_stats_kernel(const ScoreArgs a) {
    extern __shared__ char smem[];
    int tp, tq;
    const int count = a.r.count();
    if (!tile_of(a.tiles_p, (count + P::TQ - 1) / P::TQ, tp, tq)) return;
    const int p0 = tp * P::TP, q0 = tq * P::TQ;
    P prod;
    prod.run(a.w, Side{a.h.p, a.h.plane, a.h.ld, count}, p0, q0, 0, a.Dp, smem);
    float2* both = (float2*)smem;   // [2][TQ]
    float m[P::FQ], sum[P::FQ];
    const bool tail = p0 + P::TP > a.V;
    const WordExps<P> exps(a, p0);
#pragma unroll
    for (int j = 0; j < P::FQ; ++j) {
        const int n = q0 + P::col(j), exp = row_exp<P>(a, n, count);
        const int target = n < count ? a.g.t.at(a.r.at(n)) : -1;
        m[j] = -INFINITY;
#pragma unroll
        for (int i = 0; i < P::FP; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                float s = score_of<P>(prod.acc[i][j][r], exp + exps.at(i, r));
                if (tail && p0 + P::row(i, r) >= a.V) s = -INFINITY;
                prod.acc[i][j][r] = s;
                m[j] = fmaxf(m[j], s);
            }
        m[j] = fmaxf(m[j], __shfl_xor(m[j], 32, 64));
        const float base = m[j] == -INFINITY ? 0.f : m[j];
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < P::FP; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) t += exp_of(prod.acc[i][j][r] - base);
        sum[j] = t + __shfl_xor(t, 32, 64);
        // the target's score, from the lane that holds it
        const int at = target - p0 - P::wave_p();
        if (__any(at >= 0 && at < P::WP)) {
#pragma unroll
            for (int i = 0; i < P::FP; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (target >= 0 && p0 + P::row(i, r) == target) a.target_score[n] = prod.acc[i][j][r];
        }
    }
    __syncthreads();
    const int half = wave_id() % P::kWavesP;
#pragma unroll
    for (int j = 0; j < P::FQ; ++j)
        if ((threadIdx.x & 63) < 32) both[half * P::TQ + P::col(j)] = make_float2(m[j], sum[j]);
    __syncthreads();
    for (int c = threadIdx.x; c < P::TQ; c += P::kThreads)
        if (q0 + c < count) {
            float top = both[c].x, t = 0.f;
#pragma unroll
            for (int w = 1; w < P::kWavesP; ++w) top = fmaxf(top, both[w * P::TQ + c].x);
            const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int w = 0; w < P::kWavesP; ++w) t += both[w * P::TQ + c].y * exp_of(both[w * P::TQ + c].x - base);
            a.part[(int64_t)tp * a.N + q0 + c] = make_float2(top, t);
        }
}

struct JoinArgs {
    const float2* part;
    const float* target_score;
    Targets t;
    Rows r;
    int N, parts, reduction;
    float *loss, *lse, *count;
    double* sums;     // [2, blocks]: losses and counted rows (reduction 1 and 2)
};

__global__ void __launch_bounds__(kThreads) ce_join_kernel(const JoinArgs a) {
    constexpr int kSlices = kThreads / kRowsPerBlock;
    __shared__ float2 s[kSlices][kRowsPerBlock + 1];
    __shared__ double both[2][kRowsPerBlock];
    const int c = threadIdx.x % kRowsPerBlock, slice = threadIdx.x / kRowsPerBlock;
    const int n = blockIdx.x * kRowsPerBlock + c;
    float m = -INFINITY, sum = 0.f;
    auto take = [&](float2 x) {
        const float top = fmaxf(m, x.x), base = top == -INFINITY ? 0.f : top;
        sum = sum * exp_of(m - base) + x.y * exp_of(x.x - base);
        m = top;
    };
    const int place = n < a.N ? a.r.of(n) : -1;
    if (place >= 0)
#pragma unroll 8
        for (int i = slice; i < a.parts; i += kSlices) take(a.part[(int64_t)i * a.N + place]);
    s[slice][c] = make_float2(m, sum);
    __syncthreads();
    if (slice == 0) {
        for (int i = 1; i < kSlices; ++i) take(s[i][c]);
        float loss = 0.f;
        bool counts = false;
        if (n < a.N) {
            const int target = a.t.at(n);
            counts = target != -1;
            const float l = __builtin_log2f(sum);
            if (counts) loss = target < 0 ? NAN : (m - a.target_score[place]) + kLn2 * l;
            a.lse[n] = target < 0 && counts ? NAN : m;     // a target outside the vocabulary: NaN, in the gradients too
            a.lse[a.N + n] = l;
            if (a.reduction == 0) a.loss[n] = loss;
        }
        both[0][c] = (double)loss;
        both[1][c] = counts ? 1.0 : 0.0;
    }
    __syncthreads();
    if (a.reduction && threadIdx.x < 2) {
        double v = 0.0;
        for (int i = 0; i < kRowsPerBlock; ++i) v += both[threadIdx.x][i];
        a.sums[(int64_t)threadIdx.x * gridDim.x + blockIdx.x] = v;
    }
}

__global__ void __launch_bounds__(kThreads) ce_total_kernel(const double* sums, int n, int reduction, float* loss, float* count) {
    __shared__ double s[2][kThreads];
    double a = 0.0, b = 0.0;
    for (int i = threadIdx.x; i < n; i += kThreads) a += sums[i], b += sums[n + i];
    s[0][threadIdx.x] = a, s[1][threadIdx.x] = b;
    __syncthreads();
    for (int half = kThreads / 2; half >= 1; half >>= 1) {
        if (threadIdx.x < half) {
            s[0][threadIdx.x] += s[0][threadIdx.x + half];
            s[1][threadIdx.x] += s[1][threadIdx.x + half];
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        *loss = (float)(reduction == 1 ? s[0][0] / s[1][0] : s[0][0]);
        *count = (float)s[1][0];
    }
}

// U in fp32, as two fp16 planes, twice: the words' sum (dh) wants every row's largest term near the top of the planes' range, the rows' sum
// (dw) every word's.  So a tile's values have a power of two for each row in the one copy and for each word in the other, with which go the
// exponents of what they are multiplied with: the planes of w and hidden have largest values of 2^14 .. 2^15 in every row.
//
//   y = U 2^(exp_w(v) + 15 - E(n)),      sum_v U w_v   = 2^(E(n) - 29) sum_v y w'_v
//   y = U g 2^(exp_h(n) + 15 - E(v)),    sum_n U g h_n = 2^(E(v) - 29) sum_n y h'_n       (U with its factor of 2^15)
// A word that is improbable in every row keeps its 24 bits so, and rows (or words) beside one of another size theirs.  One copy with one
// power of two would be less to write: 2865 rows, 20011 words of 384 218 us against 283, both gradients' products 337 against 373 (run_scaled),
// but a probability of 4e-11 (2^-34.5, of steps of 2^-39) is left with 5 bits there, and one of 1e-13 with none.

// 2^exponent(x) is above |x| (of zeros and denormals: 2^-126).
__device__ inline int exponent(float x) { return (int)(__builtin_bit_cast(uint32_t, x) >> 23 & 255) - 126; }

template <typename P>
constexpr int kULds = kScaled<P> ? (P::kLds > 2 * P::kOutPlane + 4096 ? P::kLds : 2 * P::kOutPlane + 4096) : P::kLds;
template <typename P>
__device__ inline void planes_out(P& prod, const ScoreArgs& a, _Float16* u, int p0, int q0, int p_end, int end, char* smem) {
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) P::store(smem, h, u + h * a.plane - a.v0, a.width, p0, q0, p_end, end);
    __syncthreads();
}
template <typename P>
__device__ inline void held_split(char* smem, int i, int j, int r, const float* y) {
    f16x4 hi, lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        _Float16 x, z;
        split(y[e], x, z);
        hi[e] = x, lo[e] = z;
    }
    P::held(smem, 0, i, j, r) = hi;
    P::held(smem, 1, i, j, r) = lo;
}

// prod.acc holds U.  LDS is free.
template <typename P>
__device__ inline void scaled_u(const ScoreArgs& a, P& prod, const WordExps<P>& w, const float (&gm)[P::FQ], const int (&ge)[P::FQ], int tp, int tq, int p0, int q0, int end,
                                int p_end, char* smem) {
    constexpr int kWavesQ = P::TQ / P::WQ, kMine = P::FP * 16;
    static_assert(2 * P::kOutPlane + 4 * (P::kWavesP * P::TQ + kWavesQ * P::TP) <= kULds<P> && kMine == 32, "");
    int* row_exps = (int*)(smem + 2 * P::kOutPlane);            // [waves along the vocabulary][TQ]
    int* word_most = row_exps + P::kWavesP * P::TQ;             // [waves along the rows][TP]
    const int lane = threadIdx.x & 63, half = lane >> 5, wave_p = wave_id() % P::kWavesP, wave_q = wave_id() / P::kWavesP;
#pragma unroll
    for (int j = 0; j < P::FQ; ++j) {
        int most = INT_MIN;
#pragma unroll
        for (int i = 0; i < P::FP; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) most = max(most, exponent(prod.acc[i][j][r]) + (p0 + P::row(i, r) < a.v1 ? w.at(i, r) : kLeastExp));
        most = max(most, __shfl_xor(most, 32, 64));
        if (half == 0) row_exps[wave_p * P::TQ + P::col(j)] = most;
    }
    // the words' largest over the rows (|gm| is at most 1): each step leaves half of the values to half of the lanes
    int t[kMine];
#pragma unroll
    for (int n = 0; n < kMine; ++n) {
        t[n] = exponent(prod.acc[n / 16][0][n % 16]) + ge[0];
#pragma unroll
        for (int j = 1; j < P::FQ; ++j) t[n] = max(t[n], exponent(prod.acc[n / 16][j][n % 16]) + ge[j]);
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
        const bool upper = lane & o;
#pragma unroll
        for (int n = 0; n < o; ++n) {
            const int give = upper ? t[n] : t[n + o], keep = upper ? t[n + o] : t[n];
            t[n] = max(keep, __shfl_xor(give, o, 64));
        }
    }
    const int mine = lane & 31;     // the value that this lane is left with
    word_most[wave_q * P::TP + P::wave_p() + 32 * (mine / 16) + 8 * (mine % 16 / 4) + 4 * half + mine % 4] = t[0];
    __syncthreads();
    for (int c = threadIdx.x; c < P::TQ; c += P::kThreads) {
        int most = row_exps[c];
#pragma unroll
        for (int i = 1; i < P::kWavesP; ++i) most = max(most, row_exps[i * P::TQ + c]);
        row_exps[c] = most;
        if (q0 + c < a.Np) a.exps_h[(int64_t)tp * a.Np + q0 + c] = most;
    }
    for (int c = threadIdx.x; c < P::TP; c += P::kThreads) {
        int most = word_most[c];
#pragma unroll
        for (int i = 1; i < kWavesQ; ++i) most = max(most, word_most[i * P::TP + c]);
        word_most[c] = most;
        if (p0 + c < p_end) a.exps_w[tq * a.width + p0 - a.v0 + c] = most;
    }
    __syncthreads();
    if (a.u) {     // dh is wanted
#pragma unroll
        for (int j = 0; j < P::FQ; ++j) {
            const int exp = 15 - row_exps[P::col(j)];
#pragma unroll
            for (int i = 0; i < P::FP; ++i)
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    float y[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[e] = __builtin_amdgcn_ldexpf(prod.acc[i][j][r + e], w.at(i, r + e) + exp);
                    held_split<P>(smem, i, j, r, y);
                }
        }
        planes_out(prod, a, a.u, p0, q0, p_end, end, smem);
    }
    if (!a.u_w) return;
#pragma unroll
    for (int i = 0; i < P::FP; ++i)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const Int4 exps = *(const Int4*)(word_most + P::row(i, r));
#pragma unroll
            for (int j = 0; j < P::FQ; ++j) {
                float y[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = __builtin_amdgcn_ldexpf(prod.acc[i][j][r + e] * gm[j], ge[j] + 15 - exps.v[e]);
                held_split<P>(smem, i, j, r, y);
            }
        }
    planes_out(prod, a, a.u_w, p0, q0, p_end, end, smem);
}

// U of a piece of the vocabulary, zeros behind its end and behind the last row.  28672 rows, 50257 words of 512 in bf16: 358 us a piece
// of 9216 words on average, 687 TFLOP/s; 309 us without its 528 MB of stores.  Stores past the caches: 0.4 - 0.9 % less for the whole
// call there and at 4096 rows of 1024, 1 % more at 1186.
template <typename P>
__global__ void __launch_bounds__(P::kThreads, P::kWaves) ce_u_kernel(const ScoreArgs a) {
    extern __shared__ char smem[];
    int tp, tq;
    const int count = a.r.count();
    if (!tile_of(a.tiles_p, (count + P::TQ - 1) / P::TQ, tp, tq)) return;
    const int p0 = a.v0 + tp * P::TP, q0 = tq * P::TQ;
    P prod;
    prod.run(a.w, Side{a.h.p, a.h.plane, a.h.ld, count}, p0, q0, 0, a.Dp, smem);
    const int end = (count + kPad - 1) / kPad * kPad, p_end = a.v0 + (int)a.width;
    const WordExps<P> exps(a, p0);
    float gm[P::FQ];     // fp32: g_n (times its row of hidden's scale) is gm 2^ge
    int ge[P::FQ];
    static_assert(P::kOutPlane <= P::kLds, "");
    __syncthreads();
#pragma unroll
    for (int j = 0; j < P::FQ; ++j) {
        const int place = q0 + P::col(j), n = place < count ? a.r.at(place) : -1, exp = row_exp<P>(a, place, count);
        const int target = n >= 0 ? a.g.t.at(n) : -1;
        const bool counts = target != -1;
        const float m = counts ? a.lse[n] : 0.f, l = counts ? a.lse[a.N + n] : 0.f;
        if constexpr (kScaled<P>) {
            const float g = counts ? a.g.at(n) : 0.f;
            gm[j] = __builtin_amdgcn_frexp_mantf(g), ge[j] = g != 0.f ? __builtin_amdgcn_frexp_expf(g) + exp : 4 * kLeastExp;
        }
#pragma unroll
        for (int i = 0; i < P::FP; ++i)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int v = p0 + P::row(i, r);
                f16x4 y;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float u = __builtin_amdgcn_exp2f((score_of<P>(prod.acc[i][j][r + e], exp + exps.at(i, r + e)) - m) * kLog2e - l);
                    u = v + e == target ? u - 1.f : u;
                    u = counts && v + e < a.v1 ? u * kUScale : 0.f;     // (of a product a select, of the exponential itself a branch)
                    if constexpr (kScaled<P>) prod.acc[i][j][r + e] = u;
                    else y[e] = (_Float16)u;
                }
                if constexpr (!kScaled<P>) P::held(smem, 0, i, j, r) = y;
            }
    }
    if constexpr (kScaled<P>) {
        scaled_u<P>(a, prod, exps, gm, ge, tp, tq, p0, q0, end, p_end, smem);
    } else {
        __syncthreads();
        P::store(smem, 0, a.u - a.v0, a.width, p0, q0, p_end, end);
    }
}

struct PartArgs {
    Side p, q;
    Rows r;                             // of one of the two
    int k_rows;                         // whether k is the rows; otherwise the result's rows are
    int tiles_p, tiles_q, splits, k1;   // k from 0 to k1 (or the last row that counts), shared out to the splits in whole steps
    float* out;                         // [splits][q.n, ld]
    int64_t ld;
    int add;                            // onto what is there
    void* result;                       // set: the result itself, [q.n, p.n] of the tensors' type
    const float* scale;                 // its scale (fp32: none)
    const int* exps;                    // fp32: [blocks of k, exps_ld] the exponents of q's columns
    int64_t exps_ld;
    __host__ __device__ int blocks() const { return tiles_p * tiles_q * splits; }
};

// Sums over k of operands whose second one has a power of two for each column q in every BLOCK of k: the sum so far changes to the next
// block's.  A block that is 2^60 below the column's largest counts as one that is just that: the sum stays below 2^(30 + 24 + 60).
// The exponents wait in LDS behind the tiles, kExpBlocks of k at a time.
constexpr int kExpBlocks = 64, kExpRange = 60;
template <typename P>
constexpr int kExpBytes = kExpBlocks * P::TQ * 2;
template <typename P, int BLOCK>
__device__ inline void run_scaled(P& prod, const PartArgs& a, const Side& q, int p0, int q0, int k0, int k1, char* smem) {
    int16_t* exps = (int16_t*)(smem + P::kLds);
    int first = k0 / BLOCK, most = INT16_MIN;
    const int last = (k1 - 1) / BLOCK;
    static_assert(P::kThreads >= P::TQ, "");
    auto bring = [&] {
        const int blocks = min(kExpBlocks, last + 1 - first);
        for (int n = threadIdx.x; n < blocks * P::TQ; n += P::kThreads) {
            const int c = n % P::TQ;
            exps[n] = q0 + c < q.n ? (int16_t)a.exps[(first + n / P::TQ) * a.exps_ld + q0 + c] : (int16_t)0;
        }
        __syncthreads();
        if (threadIdx.x < P::TQ) {
            for (int n = 0; n < blocks; ++n) most = max(most, (int)exps[n * P::TQ + threadIdx.x]);
            for (int n = 0; n < blocks; ++n) {
                int16_t& x = exps[n * P::TQ + threadIdx.x];
                x = (int16_t)max((int)x, most - kExpRange);
            }
        }
    };
    int now[P::FQ];
    auto exponents = [&](int block, int (&x)[P::FQ]) {
#pragma unroll
        for (int j = 0; j < P::FQ; ++j) x[j] = exps[(block - first) * P::TQ + P::col(j)];
    };
    bring();
    __syncthreads();
    exponents(first, now);
    prod.run(a.p, q, p0, q0, k0, k1, smem, [&](int k, uint32_t) {
        if (k % BLOCK || k == k0) return;
        const int block = k / BLOCK;
        if (block == first + kExpBlocks) {
            __syncthreads();
            first = block;
            bring();
            __syncthreads();
        }
        int next[P::FQ];
        exponents(block, next);
#pragma unroll
        for (int j = 0; j < P::FQ; ++j) {
            const float f = __builtin_amdgcn_ldexpf(1.f, now[j] - next[j]);
#pragma unroll
            for (int i = 0; i < P::FP; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) prod.acc[i][j][r] *= f;
            now[j] = next[j];
        }
    });
#pragma unroll
    for (int j = 0; j < P::FQ; ++j)
#pragma unroll
        for (int i = 0; i < P::FP; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) prod.acc[i][j][r] = __builtin_amdgcn_ldexpf(prod.acc[i][j][r], now[j] - 29 - 15);     // kUScale
}

template <typename T, typename P, int BLOCK>
__device__ inline void part_of(const PartArgs& a, int block, char* smem) {
    const int tiles = a.tiles_p * a.tiles_q;
    const int split = block / tiles, tile = block - split * tiles;
    const int p0 = tile % a.tiles_p * P::TP, q0 = tile / a.tiles_p * P::TQ;
    const int count = a.r.count(), end = a.k_rows ? a.q.n : count;
    if (q0 >= end) return;
    const int steps = (a.k_rows ? (count + kPad - 1) / kPad * kPad : a.k1) / P::kStep;
    const int k0 = (int)((int64_t)steps * split / a.splits) * P::kStep, k1 = (int)((int64_t)steps * (split + 1) / a.splits) * P::kStep;
    P prod;
    const Side q_side = {a.q.p, a.q.plane, a.q.ld, end};
    if (k1 <= k0) prod.clear();
    else if constexpr (sizeof(T) == 4) run_scaled<P, BLOCK>(prod, a, q_side, p0, q0, k0, k1, smem);
    else prod.run(a.p, q_side, p0, q0, k0, k1, smem);
    // out by way of LDS, kAtOnce blocks of every wave at a time: a thread four values of a row, a wave whole rows
    constexpr int kAtOnce = P::kOut32 <= P::kLds ? P::FQ : 1;
    static_assert(P::kOut32 / P::FQ * kAtOnce <= P::kLds, "");
    constexpr int kRowsOut = P::TQ / P::FQ * kAtOnce, kPieces = P::TP / 4;
    const float f = a.scale ? 1.f / *a.scale / kUScale : 1.f;
    const bool four = a.p.n % 4 == 0 && ((uintptr_t)a.result & 15) == 0;
    typedef T four_t __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int j0 = 0; j0 < P::FQ; j0 += kAtOnce) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j)
#pragma unroll
            for (int i = 0; i < P::FP; ++i)
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const f32x16& v = prod.acc[i][j0 + j];
                    P::held32(smem, i, j, r, kAtOnce) = f32x4v{v[r], v[r + 1], v[r + 2], v[r + 3]};
                }
        __syncthreads();
#pragma unroll 4
        for (int n = threadIdx.x; n < kRowsOut * kPieces; n += P::kThreads) {
            const int row = n / kPieces, p = p0 + n % kPieces * 4, q = q0 + P::out32_col(row, j0, kAtOnce);
            if (q >= end) continue;
            f32x4v v = P::out32x4(smem, row, p - p0);
            if (a.result) {
                T* to = (T*)a.result + (int64_t)q * a.p.n + p;
                const four_t y = {(T)(v[0] * f), (T)(v[1] * f), (T)(v[2] * f), (T)(v[3] * f)};
                if (four && p < a.p.n) {
                    *reinterpret_cast<four_t*>(to) = y;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (p + e < a.p.n) to[e] = y[e];
                }
            } else if (p < a.ld) {
                float* to = a.out + ((int64_t)split * a.q.n + q) * a.ld + p;
                if (a.add) v += *reinterpret_cast<const f32x4v*>(to);
                *reinterpret_cast<f32x4v*>(to) = v;
            }
        }
    }
}

// Both gradients' products with a piece of U in one launch, either without tiles where it is not wanted: the one's
// workgroups fill what the other's leave of the card's last round.  The longer ones come first.
template <typename T, typename H, typename W, int BLOCK_H, int BLOCK_W>
__global__ void __launch_bounds__(H::kThreads, H::kWaves) ce_part_kernel(const PartArgs h, const PartArgs w) {
    static_assert(H::kThreads == W::kThreads && H::kWaves == W::kWaves, "");
    extern __shared__ char smem[];
    const bool h_first = (int64_t)h.k1 * w.splits >= (int64_t)w.k1 * h.splits;
    const int n = h_first ? h.blocks() : w.blocks(), block = blockIdx.x;
    if ((block < n) == h_first) part_of<T, H, BLOCK_H>(h, h_first ? block : block - n, smem);
    else part_of<T, W, BLOCK_W>(w, h_first ? block - n : block, smem);
}

// out[n, d] = factor (g_n) sum_s part[s][n, d], in the parts' order; graded rows come from their places.
struct SumArgs {
    const float* part;
    int splits, rows, D, ld, graded, blocks;
    const float* scale;
    void* out;
};

template <typename T>
__global__ void __launch_bounds__(kThreads) ce_sum_kernel(const SumArgs x, const SumArgs y, const RowGrad g, const Rows r) {
    const bool first = (int)blockIdx.x < x.blocks;
    const SumArgs& a = first ? x : y;
    const int block = first ? blockIdx.x : blockIdx.x - x.blocks;
    const float f = a.scale ? 1.f / *a.scale / kUScale : 1.f;
    const int pieces = a.ld / 4;
    T* out = (T*)a.out;
    for (int64_t i = (int64_t)block * kThreads + threadIdx.x; i < (int64_t)a.rows * pieces; i += (int64_t)a.blocks * kThreads) {
        const int64_t n = i / pieces;
        const int d = (int)(i - n * pieces) * 4;
        const int64_t from = a.graded ? r.of(n) : n;
        f32x4v v = {0.f, 0.f, 0.f, 0.f};
        const float gn = a.graded ? g.at(n) : 1.f;
        if (from >= 0 && gn != 0.f) {
            v = *reinterpret_cast<const f32x4v*>(a.part + from * a.ld + d);
            for (int s = 1; s < a.splits; ++s) v += *reinterpret_cast<const f32x4v*>(a.part + ((int64_t)s * a.rows + from) * a.ld + d);
        }
        typedef T four_t __attribute__((ext_vector_type(4)));
        const four_t y = {(T)(v[0] * f * gn), (T)(v[1] * f * gn), (T)(v[2] * f * gn), (T)(v[3] * f * gn)};
        if (a.D % 4 == 0 && ((uintptr_t)out & 15) == 0) {
            if (d < a.D) *reinterpret_cast<four_t*>(out + n * a.D + d) = y;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (d + e < a.D) out[n * a.D + d + e] = y[e];
        }
    }
}

// ---- few rows ----------------------------------------------------------------------------
//
// The time is the weights' read (and dw's write) then, so fp32 products from registers do: a wave takes a few words at a time, 16
// bytes of each a lane and chunk, and reads hidden (fp32 in LDS) once for them.  The backward has the scores' words still in its
// registers for dh, whose sums it keeps over all its words, and writes dw at once: w is read once a direction, without the copies
// that the matrix instructions want.  One row on 128789 words of 256 in fp32: 22.6 us forward, 44.5 us backward, the weights' 132 MB at
// 5.8 and (with dw) 5.9 TB/s, partly out of the last-level cache; 5 rows on 100000 of 1024 in bf16 126.6 us backward, 3.2 TB/s (vector instructions).  A score's sum over the lanes leaves it with the lane whose number begins with it.
constexpr int kFewThreads = 512;
constexpr int kFewLanes = 64;
struct FewArgs {
    const void *hidden, *weight;
    int64_t h_ld, w_ld;
    RowGrad g;
    int n0, rows, N, V, D, vec, out_vec;   // the launch's rows, of all N
    int n1, rows1;                // further rows, which count for dw alone
    float2* part;                 // forward: [workgroups, N] maximum and sum
    float* target_score;          // forward: [N]
    const float* lse;             // backward: [2, N]
    float* part_h;                // backward: [workgroups, rows, D4], or NULL
    int D4;
    void* dweight;                // backward: [V, D], or NULL
};

// R: rows; C: channels of a lane.  R C is at most 128, the sums of dh in registers.
template <typename T, int R, int C>
struct Few {
    static constexpr int kVec = 16 / sizeof(T), kChunks = C / kVec, kQuads = kVec / 4;
    static constexpr int kWords = C * sizeof(T) > 64 || R * C > 64 ? 2 : 4;   // at a time, what registers hold beside the sums
    static constexpr int M = kWords * R;
    static constexpr int kLds = R * C * kFewLanes * 4;
    static_assert(R * C <= 128 && M <= kFewLanes && C % kVec == 0, "");
    typedef T vec_t __attribute__((ext_vector_type(kVec), aligned(16)));

    static __device__ int lane() { return threadIdx.x & 63; }
    static __device__ int channel(int c) { return (c * kFewLanes + lane()) * kVec; }
    static __device__ int at(int r, int c, int q) { return (((r * kChunks + c) * kQuads + q) * kFewLanes + lane()) * 4; }
    // which of the wave's scores this lane has
    static constexpr int kEach = kFewLanes / M;
    static __device__ int word() { return lane() / kEach / R; }
    static __device__ int row() { return lane() / kEach % R; }

    // hidden in LDS, zeros in place of ignored rows and behind the end
    static __device__ void stage(const FewArgs& a, int n0, int rows, float* h) {
        for (int i = threadIdx.x; i < R * C * kFewLanes; i += kFewThreads) {
            const int r = i / (C * kFewLanes), c = i / (kVec * kFewLanes) % kChunks, q = i / (4 * kFewLanes) % kQuads;
            const int d = (c * kFewLanes + i / 4 % kFewLanes) * kVec + 4 * q + i % 4;
            h[i] = r < rows && d < a.D && a.g.t.at(n0 + r) != -1 ? (float)((const T*)a.hidden)[(n0 + r) * a.h_ld + d] : 0.f;
        }
        __syncthreads();
    }
    static __device__ void load(const FewArgs& a, int v0, vec_t (&w)[kWords][kChunks]) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            const T* from = (const T*)a.weight + (int64_t)min(v0 + i, a.V - 1) * a.w_ld;
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                const int d = channel(c);
                if (a.vec) {
                    w[i][c] = d < a.D ? *reinterpret_cast<const vec_t*>(from + d) : vec_t{};
                } else {
#pragma unroll
                    for (int e = 0; e < kVec; ++e) w[i][c][e] = d + e < a.D ? from[d + e] : (T)0.f;
                }
            }
        }
    }
    // this lane's score
    static __device__ float score(const float* h, const vec_t (&w)[kWords][kChunks]) {
        float s[M] = {};
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int q = 0; q < kQuads; ++q) {
                __builtin_amdgcn_sched_barrier(0);     // hidden's reads stay where they are: all of them at once would not fit
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const f32x4v x = *reinterpret_cast<const f32x4v*>(h + at(r, c, q));
#pragma unroll
                    for (int i = 0; i < kWords; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[i * R + r] = __builtin_fmaf((float)w[i][c][4 * q + e], x[e], s[i * R + r]);
                }
            }
#pragma unroll
        for (int k = 0; k < 6; ++k) {
            const int o = 32 >> k, left = M >> (k + 1);
            if (left == 0) {
                s[0] += __shfl_xor(s[0], o, 64);
            } else {
                const bool upper = lane() & o;
#pragma unroll
                for (int i = 0; i < left; ++i) {
                    const float give = upper ? s[i] : s[i + left], keep = upper ? s[i + left] : s[i];
                    s[i] = keep + __shfl_xor(give, o, 64);
                }
            }
        }
        return s[0];
    }
    // what this lane's row has to do with U, and all lanes' g U of the words
    struct Row {
        int target;
        float g, m, l;
        __device__ Row(const FewArgs& a, int n0, int rows) {
            const int n = n0 + row();
            target = row() < rows ? a.g.t.at(n) : -1;
            const bool counts = target != -1;
            g = counts ? a.g.at(n) : 0.f, m = counts ? a.lse[n] : 0.f, l = counts ? a.lse[a.N + n] : 0.f;
        }
    };
    static __device__ void gradients(const FewArgs& a, const Row& o, const float* h, const vec_t (&w)[kWords][kChunks], int v0, float (&u)[kWords][R]) {
        const int v = v0 + word();
        float mine = __builtin_amdgcn_exp2f((score(h, w) - o.m) * kLog2e - o.l);
        mine = v == o.target ? mine - 1.f : mine;
        mine = v < a.V && o.g != 0.f ? mine * o.g : 0.f;
#pragma unroll
        for (int i = 0; i < M; ++i)
            u[i / R][i % R] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, mine), i * kEach));
    }
};

template <typename T, int R, int C>
__global__ void __launch_bounds__(kFewThreads, 2) ce_few_stats_kernel(const FewArgs a) {
    typedef Few<T, R, C> F;
    extern __shared__ char smem[];
    float* h = (float*)smem;
    F::stage(a, a.n0, a.rows, h);
    constexpr int kWaves = kFewThreads / 64;
    const int wave = wave_id(), n = a.n0 + F::row(), target = F::row() < a.rows ? a.g.t.at(n) : -1;
    float m = -INFINITY, sum = 0.f;
    for (int64_t v0 = ((int64_t)blockIdx.x * kWaves + wave) * F::kWords; v0 < a.V; v0 += (int64_t)gridDim.x * kWaves * F::kWords) {
        typename F::vec_t w[F::kWords][F::kChunks];
        F::load(a, (int)v0, w);
        const float s = F::score(h, w);
        const int v = (int)v0 + F::word();
        if (v >= a.V) continue;
        if (v == target) a.target_score[n] = s;
        const float top = fmaxf(m, s), base = top == -INFINITY ? 0.f : top;
        sum = sum * exp_of(m - base) + exp_of(s - base);
        m = top;
    }
    __shared__ float2 both[kWaves][F::M];
    if (F::lane() % F::kEach == 0) both[wave][F::lane() / F::kEach] = make_float2(m, sum);
    __syncthreads();
    if ((int)threadIdx.x < a.rows) {
        float top = -INFINITY, t = 0.f;
        for (int i = 0; i < kWaves * F::kWords; ++i) top = fmaxf(top, both[i / F::kWords][i % F::kWords * R + threadIdx.x].x);
        const float base = top == -INFINITY ? 0.f : top;
        for (int i = 0; i < kWaves * F::kWords; ++i) {
            const float2 x = both[i / F::kWords][i % F::kWords * R + threadIdx.x];
            t += x.y * exp_of(x.x - base);
        }
        a.part[(int64_t)blockIdx.x * a.N + a.n0 + threadIdx.x] = make_float2(top, t);
    }
}

// BOTH: dw of further rows too, whose dh another launch sums: nothing of dw is read again.
template <typename T, int R, int C, bool BOTH>
__global__ void __launch_bounds__(kFewThreads, 2) ce_few_grads_kernel(const FewArgs a) {
    typedef Few<T, R, C> F;
    extern __shared__ char smem[];
    float *h = (float*)smem, *h1 = h + F::kLds / 4;
    F::stage(a, a.n0, a.rows, h);
    if (BOTH) F::stage(a, a.n1, a.rows1, h1);
    constexpr int kWaves = kFewThreads / 64;
    const int wave = wave_id();
    const typename F::Row row(a, a.n0, a.rows), row1(a, a.n1, BOTH ? a.rows1 : 0);
    float dh[R][C] = {};
    for (int64_t v0 = ((int64_t)blockIdx.x * kWaves + wave) * F::kWords; v0 < a.V; v0 += (int64_t)gridDim.x * kWaves * F::kWords) {
        typename F::vec_t w[F::kWords][F::kChunks];
        F::load(a, (int)v0, w);
        float u[F::kWords][R], u1[F::kWords][R];
        F::gradients(a, row, h, w, (int)v0, u);
        if (BOTH) F::gradients(a, row1, h1, w, (int)v0, u1);
#pragma unroll
        for (int c = 0; c < F::kChunks; ++c) {
            typename F::vec_t out[F::kWords];
#pragma unroll
            for (int q = 0; q < F::kQuads; ++q) {
                __builtin_amdgcn_sched_barrier(0);
                f32x4v y[F::kWords] = {};
#pragma unroll
                for (int n = 0; n < R; ++n) {
                    const f32x4v x = *reinterpret_cast<const f32x4v*>(h + F::at(n, c, q));
#pragma unroll
                    for (int i = 0; i < F::kWords; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            y[i][e] = __builtin_fmaf(u[i][n], x[e], y[i][e]);
                            float& sum = dh[n][c * F::kVec + 4 * q + e];
                            sum = __builtin_fmaf(u[i][n], (float)w[i][c][4 * q + e], sum);
                        }
                }
                if (BOTH) {
#pragma unroll
                    for (int n = 0; n < R; ++n) {
                        const f32x4v x = *reinterpret_cast<const f32x4v*>(h1 + F::at(n, c, q));
#pragma unroll
                        for (int i = 0; i < F::kWords; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e) y[i][e] = __builtin_fmaf(u1[i][n], x[e], y[i][e]);
                    }
                }
#pragma unroll
                for (int i = 0; i < F::kWords; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) out[i][4 * q + e] = (T)y[i][e];
            }
            const int d = F::channel(c);
            if (!a.dweight || d >= a.D) continue;
#pragma unroll
            for (int i = 0; i < F::kWords; ++i) {
                if (v0 + i >= a.V) continue;
                T* to = (T*)a.dweight + (v0 + i) * a.D + d;
                if (a.out_vec) {
                    *reinterpret_cast<typename F::vec_t*>(to) = out[i];
                } else {
#pragma unroll
                    for (int e = 0; e < F::kVec; ++e)
                        if (d + e < a.D) to[e] = out[i][e];
                }
            }
        }
    }
    if (!a.part_h) return;
    // the waves' sums of dh in their order, in hidden's place
    for (int i = 0; i < kWaves; ++i) {
        __syncthreads();
        if (wave != i) continue;
#pragma unroll
        for (int n = 0; n < R; ++n)
#pragma unroll
            for (int c = 0; c < F::kChunks; ++c)
#pragma unroll
                for (int q = 0; q < F::kQuads; ++q) {
                    f32x4v& sum = *reinterpret_cast<f32x4v*>(h + F::at(n, c, q));
                    const float* x = dh[n] + c * F::kVec + 4 * q;
                    const f32x4v y = {x[0], x[1], x[2], x[3]};
                    sum = i ? sum + y : y;
                }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.rows * C * kFewLanes / 4; i += kFewThreads) {
        const int n = i / (C * kFewLanes / 4), c = i / (F::kQuads * kFewLanes) % F::kChunks, q = i / kFewLanes % F::kQuads;
        const int d = (c * kFewLanes + i % kFewLanes) * F::kVec + 4 * q;
        if (d < a.D4)
            *reinterpret_cast<f32x4v*>(a.part_h + ((int64_t)blockIdx.x * a.rows + n) * a.D4 + d) = *reinterpret_cast<const f32x4v*>(h + 4 * i);
    }
}

// dh from the workgroups' parts: 16 pieces of a row a workgroup, each by 16 threads in a fixed order.  A row without a gradient has
// sums of 0 w, which are not zeros where a weight is infinite.
template <typename T>
__global__ void __launch_bounds__(kThreads) ce_few_sum_kernel(const float* part, int parts, const RowGrad g, int n0, int N, int D, int D4, T* out) {
    constexpr int kCols = 16, kSlices = kThreads / kCols;
    __shared__ f32x4v s[kSlices][kCols];
    const int col = threadIdx.x % kCols, slice = threadIdx.x / kCols, pieces = D4 / 4;
    const int i = blockIdx.x * kCols + col;
    f32x4v v = {};
    if (i < N * pieces)
#pragma unroll 8
        for (int n = slice; n < parts; n += kSlices) v += *reinterpret_cast<const f32x4v*>(part + ((int64_t)n * N * pieces + i) * 4);
    s[slice][col] = v;
    __syncthreads();
    if (slice || i >= N * pieces) return;
    for (int n = 1; n < kSlices; ++n) v += s[n][col];
    const int d = i % pieces * 4;
    if (g.at(n0 + i / pieces) == 0.f) v = f32x4v{0.f, 0.f, 0.f, 0.f};
    T* to = out + (int64_t)(i / pieces) * D + d;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (d + e < D) to[e] = (T)v[e];
}

// ---- host side ---------------------------------------------------------------------------

// Cuts a workspace; with a null base only the size is wanted.
struct Carve {
    char* base;
    int64_t used = 0;
    template <typename T>
    T* take(int64_t n) {
        T* p = base ? (T*)(base + used) : nullptr;
        used += pad(n * (int64_t)sizeof(T), 256);
        return p;
    }
};

// Bytes of a copy of U in a piece (of 256 words at least): few launches and few passes over dh's sums against what stays in the
// caches and the memory that is wanted.  56 x 512 rows, 50257 words: 256 MiB 7.14 ms, 512 6.88, 1024 6.93, 2048 7.05.
constexpr int64_t kPieceBytes = (int64_t)512 << 20;
// From so many rows on the ones that count are put next to each other first: a launch more and a copy of the rows, 15.5 + 15.2 us a
// direction (both directions: 6.8 ms) at 56 x 512; where 0.3 of 4093 rows are ignored (20011 words of 384, fp32) 929 -> 782 us.
constexpr int64_t kGatherRows = 1024;
constexpr int64_t kWordTile = 256;      // words of the largest of the scores' tiles

// The products of each type: the scores (vocabulary x rows), dh (D x rows) and dw (D x vocabulary).
struct Bf16 {
    typedef __bf16 T;
    static constexpr int kPlanes = 1;
    typedef Product<__bf16, 1, 192, 128, kRows, kRows, 2, 2, 64> Score;
    typedef Score U;
    typedef Product<_Float16, 1, 256, 128, kCols, kRows> GradH;
    typedef Product<_Float16, 1, 256, 128, kCols, kCols> GradW;
};
struct F32 {
    typedef float T;
    static constexpr int kPlanes = 2;
    typedef Product<_Float16, 2, 256, 128, kRows, kRows, 4, 2> Score;
    typedef Product<_Float16, 2, 128, 128, kRows, kRows> U;
    typedef Product<_Float16, 2, 128, 128, kCols, kRows> GradH;
    typedef Product<_Float16, 2, 128, 128, kCols, kCols> GradW;
};

// Up to 64 rows: the scores' tiles take 64 rows and more of the vocabulary, whose reads are the time then (12 rows on 100 000
// words of 1024, bf16: maxima and sums 67 -> 52 us, U 56 -> 42).
constexpr int64_t kFewRows = 64;
struct FewBf16 : Bf16 {
    typedef Product<__bf16, 1, 256, 64, kRows, kRows, 2, 2, 64> Score;
    typedef Score U;
};
struct FewF32 : F32 {
    typedef Product<_Float16, 2, 128, 64, kRows, kRows, 2, 2, 32> Score;
    typedef Score U;
};

struct Plan {
    int64_t N, V, D, Dp, Np, Vp, width;
    bool direct_h, direct_w, gather;
    int planes, tiles_p, tiles_q;           // of the scores
    int width_tiles;                         // of a piece's
    int s_h, s_w;                            // splits of the two gradients' products
};

template <typename P>
int64_t tiles_of(int64_t np, int64_t nq) { return ((np + P::TP - 1) / P::TP) * ((nq + P::TQ - 1) / P::TQ); }

// Splits of the two gradients' k: those (of 1 to 32 each, runs of 256 k at least) with the shortest launch.  A workgroup takes its
// steps of k and about kOverhead more to begin and end, and its part of the sums is written and read again; the longer ones go
// first, in rounds of kSlots, and the shorter ones fill what the last of these leaves.  56 x 512 rows, a piece of 9216 words of
// 512: 448 workgroups of 144 steps and 576 of 112 in two full rounds; the six pieces' launches take 500 us on average, 983 TFLOP/s.
constexpr int kOverhead = 12, kSlots = 512;
void choose_splits(int64_t tiles_h, int64_t k_h, int64_t tiles_w, int64_t k_w, int& s_h, int& s_w) {
    double best = 1e300;
    s_h = s_w = 1;
    for (int x = 1; x <= 32 && (x == 1 || k_h / x >= 256); ++x)
        for (int y = 1; y <= 32 && (y == 1 || k_w / y >= 256); ++y) {
            const double h = (double)k_h / x / kPad + kOverhead, w = (double)k_w / y / kPad + kOverhead;
            const double t1 = std::max(h, w), t2 = std::min(h, w);
            const int64_t n1 = h >= w ? tiles_h * x : tiles_w * y, n2 = tiles_h * x + tiles_w * y - n1;
            const int64_t late = n1 % kSlots;                                           // slots with a long one in the last round,
            const int64_t beside = late ? (int64_t)(t1 / t2) * (kSlots - late) : 0;     // short ones in the others meanwhile
            const int64_t left = n2 - std::min(n2, beside);
            const double span = (double)(n1 / kSlots + (late > 0)) * t1 + (double)((left + kSlots - 1) / kSlots) * t2;
            const double cost = span + 0.02 * kOverhead * (double)(n1 + n2) / kSlots;
            if (cost < best * 0.999) best = cost, s_h = x, s_w = y;
        }
}

// Whether the scores' product takes a user's matrix without a copy.
template <typename C>
bool as_it_is(int64_t D, const void* x, int64_t ld) {
    return C::kPlanes == 1 && D % C::Score::kStep == 0 && ((uintptr_t)x & 15) == 0 && ld % 8 == 0;
}

template <typename C>
Plan plan_of(const mb_linear_ce* a) {
    Plan p = {};
    p.N = a->N, p.V = a->V, p.D = a->D;
    p.Dp = pad(p.D, kPad), p.Np = pad(p.N, kPad), p.Vp = pad(p.V, kPad);
    p.planes = C::kPlanes;
    p.gather = p.N >= kGatherRows;
    p.direct_h = !p.gather && as_it_is<C>(p.D, a->hidden, a->hidden_ld), p.direct_w = as_it_is<C>(p.D, a->weight, a->weight_ld);
    p.tiles_p = (int)((p.V + C::Score::TP - 1) / C::Score::TP), p.tiles_q = (int)((p.N + C::Score::TQ - 1) / C::Score::TQ);
    p.width = std::min<int64_t>(pad(p.V, 256), std::max<int64_t>(256, kPieceBytes / (p.Np * 2 * p.planes) / 256 * 256));
    p.width_tiles = (int)((p.width + C::U::TP - 1) / C::U::TP);
    choose_splits(tiles_of<typename C::GradH>(p.D, p.N), std::min(p.width, p.Vp), tiles_of<typename C::GradW>(p.D, std::min(p.width, p.V)), p.Np, p.s_h,
                  p.s_w);
    static_assert(C::GradH::kThreads == 256, "kSlots: two a CU");
    return p;
}

struct Buffers {
    int *rows, *pos, *m;
    float *largest_w, *largest_g, *scales;   // bf16: scales of w and g h
    int *exp_w, *exp_h, *exps_h, *exps_w;    // fp32: the rows' exponents, and those of U's copies
    void *h, *w;                 // copies for the scores (planes, or padded bf16)
    float2* part;
    float* target_score;
    double* sums;
    _Float16 *w16, *h16, *u, *u_w;   // backward
    float *part_h, *part_w;
    int64_t bytes;
};

Buffers buffers_of(const Plan& p, bool backward, void* base) {
    Carve c = {(char*)base};
    Buffers b = {};
    const bool f32 = p.planes == 2;
    if (f32) b.exp_h = c.take<int>(p.Np), b.exp_w = c.take<int>(pad(p.V, kWordTile));
    else b.largest_w = c.take<float>(kMaxBlocks), b.largest_g = c.take<float>(kMaxBlocks), b.scales = c.take<float>(2);
    if (p.gather) b.rows = c.take<int>(p.N), b.pos = c.take<int>(p.N), b.m = c.take<int>(1);
    if (!p.direct_h) b.h = c.take<_Float16>(p.planes * p.Np * p.Dp);
    if (!p.direct_w) b.w = c.take<_Float16>(p.planes * p.Vp * p.Dp);
    if (!backward) {
        b.part = c.take<float2>((int64_t)p.tiles_p * p.N);
        b.target_score = c.take<float>(p.N);
        b.sums = c.take<double>(2 * ((p.N + kRowsPerBlock - 1) / kRowsPerBlock));
    } else {
        b.w16 = f32 ? (_Float16*)b.w : c.take<_Float16>(p.Vp * p.Dp);
        b.h16 = f32 ? (_Float16*)b.h : c.take<_Float16>(p.Np * p.Dp);
        b.u = c.take<_Float16>(p.planes * p.Np * p.width);
        if (f32) {
            b.u_w = c.take<_Float16>(p.planes * p.Np * p.width);
            b.exps_h = c.take<int>(p.width_tiles * p.Np), b.exps_w = c.take<int>(p.tiles_q * p.width);
        }
        b.part_h = c.take<float>(p.s_h * p.N * p.Dp);
        if (p.s_w > 1) b.part_w = c.take<float>(p.s_w * p.width * p.Dp);
    }
    b.bytes = c.used;
    return b;
}

unsigned blocks_for(int64_t items) { return (unsigned)std::max<int64_t>(1, std::min<int64_t>((items + kThreads - 1) / kThreads, 4096)); }

Matrix matrix(const void* p, int64_t ld, int64_t rows, int64_t D, int size, float* largest, float* scale, void* out, int64_t rows_pad, int64_t Dp) {
    Matrix x = {};
    x.p = p, x.ld = ld, x.rows = (int)rows, x.D = (int)D, x.vec = ((uintptr_t)p & 15) == 0 && ld * size % 16 == 0;
    x.largest = largest, x.scale = scale, x.out = out, x.rows_pad = (int)rows_pad, x.Dp = (int)Dp;
    x.blocks = (int)std::min<int64_t>(blocks_for(rows * ((D + 7) / 8)), kMaxBlocks);
    return x;
}
// Copies of the set's matrices as one plane; scaled ones after a launch that looks for their largest values.
template <typename T, typename O>
void copies(Set a, hipStream_t st) {
    if (a.n == 0) return;
    int total = 0;
    if (a.x[0].largest) {
        for (int i = 0; i < a.n; ++i) a.first[i] = total, total += a.x[i].blocks;
        hipLaunchKernelGGL((ce_largest_kernel<T>), dim3(total), dim3(kThreads), 0, st, a);
    }
    total = 0;
    for (int i = 0; i < a.n; ++i) {
        a.x[i].copy_blocks = (int)blocks_for((int64_t)a.x[i].rows_pad * a.x[i].Dp / 8);
        a.first[i] = total, total += a.x[i].copy_blocks;
    }
    hipLaunchKernelGGL((ce_planes_kernel<T, O>), dim3(total), dim3(kThreads), 0, st, a);
}
// fp32 matrices as two planes.
void row_planes(Set a, hipStream_t st) {
    int total = 0;
    for (int i = 0; i < a.n; ++i) {
        a.x[i].copy_blocks = (int)blocks_for((int64_t)a.x[i].rows_pad * 64);
        a.first[i] = total, total += a.x[i].copy_blocks;
    }
    hipLaunchKernelGGL(ce_row_planes_kernel, dim3(total), dim3(kThreads), 0, st, a);
}

// The rows' places and the operands of the scores: the user's own, or copies of them; and what the gradients want copied: g h
// for dw, and for dh w in fp16 (fp32: the scores' planes serve both).
template <typename C>
void operands(const mb_linear_ce* a, const Plan& p, const Buffers& b, ScoreArgs& s, const RowGrad& g, bool wants_h, bool wants_w, hipStream_t st) {
    typedef typename C::T T;
    s.g = g;
    s.r = {b.rows, b.pos, b.m, (int)p.N};
    if (p.gather) {
        const int each = (int)pad((p.N + kRowRuns - 1) / kRowRuns, kThreads);
        hipLaunchKernelGGL(ce_rows_kernel, dim3((unsigned)((p.N + each - 1) / each)), dim3(kThreads), 0, st, g.t, (int)p.N, each, b.rows, b.pos, b.m);
    }
    Set scores = {}, grads = {};
    scores.g = grads.g = g, scores.r = grads.r = s.r;
    auto hidden = [&](float* largest, float* scale, void* out, int graded) {
        Matrix x = matrix(a->hidden, a->hidden_ld, p.N, p.D, sizeof(T), largest, scale, out, p.Np, p.Dp);
        x.gathered = p.gather, x.graded = graded;
        return x;
    };
    auto weight = [&](float* largest, float* scale, void* out) {
        return matrix(a->weight, a->weight_ld, p.V, p.D, sizeof(T), largest, scale, out, p.Vp, p.Dp);
    };
    if constexpr (sizeof(T) == 4) {
        scores.x[0] = hidden(nullptr, nullptr, b.h, 1), scores.x[1] = weight(nullptr, nullptr, b.w), scores.n = 2;
        scores.x[0].exps = b.exp_h, scores.x[1].exps = b.exp_w;
        row_planes(scores, st);
        s.exp_h = b.exp_h, s.exp_w = b.exp_w;
    } else {
        if (!p.direct_h) scores.x[scores.n++] = hidden(nullptr, nullptr, b.h, 0);
        if (!p.direct_w) scores.x[scores.n++] = weight(nullptr, nullptr, b.w);
        if (wants_w) grads.x[grads.n++] = hidden(b.largest_g, b.scales + 1, b.h16, 1);
        if (wants_h) grads.x[grads.n++] = weight(b.largest_w, b.scales, b.w16);
        copies<T, __bf16>(scores, st);
        copies<T, _Float16>(grads, st);
    }
    s.h = {p.direct_h ? a->hidden : b.h, p.Np * p.Dp * 2, p.direct_h ? a->hidden_ld : p.Dp, (int)p.N};
    s.w = {p.direct_w ? a->weight : b.w, p.Vp * p.Dp * 2, p.direct_w ? a->weight_ld : p.Dp, (int)p.V};
    s.V = (int)p.V, s.N = (int)p.N, s.Dp = (int)(p.direct_h && p.direct_w ? p.D : p.Dp), s.tiles_p = p.tiles_p;
}

template <typename K, typename A>
int launch(const char* what, K kernel, int threads, int lds, Told& told, unsigned grid, hipStream_t st, const A& args) {
    if (const int rc = allow_lds(what, (const void*)kernel, lds, told)) return rc;
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(threads), lds, st, args);
    return MB_OK;
}

template <typename P>
int stats(const ScoreArgs& s, int tiles_q, hipStream_t st) {
    static Told told;
    return launch("mb_linear_ce_fwd", ce_stats_kernel<P>, P::kThreads, P::kLds, told, tile_grid((int64_t)s.tiles_p * tiles_q), st, s);
}
template <typename P>
int piece_of_u(const ScoreArgs& s, int tiles_q, hipStream_t st) {
    static Told told;
    return launch("mb_linear_ce_bwd", ce_u_kernel<P>, P::kThreads, kULds<P>, told, tile_grid((int64_t)s.tiles_p * tiles_q), st, s);
}
template <typename P>
void tiles_for(PartArgs& a) {
    a.tiles_p = (int)((a.p.n + P::TP - 1) / P::TP), a.tiles_q = (int)((a.q.n + P::TQ - 1) / P::TQ);
}
template <typename C>
int parts(const PartArgs& h, const PartArgs& w, hipStream_t st) {
    typedef typename C::T T;
    typedef typename C::GradH H;
    typedef typename C::GradW W;
    static Told told;
    constexpr int lds = std::max(H::kLds + (sizeof(T) == 4 ? kExpBytes<H> : 0), W::kLds + (sizeof(T) == 4 ? kExpBytes<W> : 0));
    static_assert(lds <= H::kRoom, "two workgroups a CU");
    constexpr auto kernel = ce_part_kernel<T, H, W, C::U::TP, C::U::TQ>;
    if (const int rc = allow_lds("mb_linear_ce_bwd", (const void*)kernel, lds, told)) return rc;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(h.blocks() + w.blocks())), dim3(H::kThreads), lds, st, h, w);
    return MB_OK;
}

int check(const char* what, const mb_linear_ce* a) {
    MB_REQUIRE(a, "%s: null args", what);
    MB_REQUIRE(a->N >= 1 && a->N <= (1 << 28), "%s: N=%lld (1 to 2^28)", what, (long long)a->N);
    MB_REQUIRE(a->V >= 1 && a->V <= (1 << 24), "%s: V=%lld (1 to 2^24)", what, (long long)a->V);
    MB_REQUIRE(a->D >= 1 && a->D <= (1 << 16), "%s: D=%lld (1 to 2^16)", what, (long long)a->D);
    MB_REQUIRE(a->dtype == MB_DTYPE_F32 || a->dtype == MB_DTYPE_BF16, "%s: dtype=%lld", what, (long long)a->dtype);
    MB_REQUIRE(a->reduction >= 0 && a->reduction <= 2, "%s: reduction=%lld", what, (long long)a->reduction);
    MB_REQUIRE(a->target_bytes == 4 || a->target_bytes == 8, "%s: target_bytes=%lld (4 or 8)", what, (long long)a->target_bytes);
    MB_REQUIRE(a->hidden && a->weight && a->target && a->lse && a->count, "%s: null pointer argument", what);
    for (const int64_t ld : {a->hidden_ld, a->weight_ld})
        MB_REQUIRE(ld >= a->D && ld <= (1 << 22), "%s: rows are %lld elements apart (D to 2^22)", what, (long long)ld);
    return MB_OK;
}

// Workgroups of a launch, whose threads are counted in 32 bits.
int fits(const char* what, const mb_linear_ce* a, const Plan& p, int64_t tiles_d) {
    const int64_t most = 0x7fffff;
    if ((int64_t)p.tiles_p * p.tiles_q > most || tiles_d * (p.tiles_q * p.s_h + (p.width / 128 + 1) * p.s_w) > most)
        return fail(MB_ERR_UNSUPPORTED, "%s: %lld rows of %lld on %lld words are too many for a launch", what, (long long)a->N, (long long)a->D,
                    (long long)a->V);
    return MB_OK;
}

int enough(const char* what, const mb_linear_ce* a, int64_t need) {
    MB_REQUIRE(((uintptr_t)a->workspace & 255) == 0, "%s: the workspace has to begin at a multiple of 256 bytes", what);
    if (!a->workspace || a->workspace_bytes < need)
        return fail(MB_ERR_WORKSPACE, "%s: workspace of %lld bytes, %lld are needed", what, (long long)a->workspace_bytes, (long long)need);
    return MB_OK;
}

// What the call writes must not be anything that it reads, nor twice the same.
int apart(const char* what, const mb_linear_ce* a, bool backward) {
    const int64_t size = a->dtype == MB_DTYPE_F32 ? 4 : 2, rows = a->reduction == 0 ? a->N : 1;
    const Span read[] = {span(a->hidden, ((a->N - 1) * a->hidden_ld + a->D) * size), span(a->weight, ((a->V - 1) * a->weight_ld + a->D) * size),
                         span(a->target, a->N * a->target_bytes), span(backward ? a->lse : nullptr, 8 * a->N), span(backward ? a->count : nullptr, 4),
                         span(backward ? a->dloss : nullptr, 4 * rows)};
    const Span written[] = {span(a->workspace, a->workspace_bytes), span(backward ? a->dhidden : nullptr, a->N * a->D * size),
                            span(backward ? a->dweight : nullptr, a->V * a->D * size), span(backward ? nullptr : a->loss, 4 * rows),
                            span(backward ? nullptr : a->lse, 8 * a->N), span(backward ? nullptr : a->count, 4)};
    for (const Span& x : written) {
        for (const Span& y : read) MB_REQUIRE(!touch(x, y), "%s: memory that is written is shared with an input", what);
        for (const Span& y : written) MB_REQUIRE(&x == &y || !touch(x, y), "%s: two tensors that are written share memory", what);
    }
    return MB_OK;
}

// ---- few rows, the host's part ----

constexpr int kVectorRows = 8;                       // of a launch
constexpr int kFewStats = 512, kFewGrads = 256;      // workgroups, at most

// Channels of a lane, and rows, of the kernels for these sizes; 0 where there are none.
int few_channels(int64_t D, int size) {
    for (int c = 16 / size; c <= 32; c *= 2)
        if (c * kFewLanes >= D) return c;
    return 0;
}
// Rows of a launch, at most (0: none).
int launch_rows(int64_t D, int size) {
    const int c = few_channels(D, size);
    return c ? std::min(kVectorRows, 128 / c) : 0;
}
int few_rows(int64_t N) { return N <= 1 ? 1 : N <= 2 ? 2 : N <= 4 ? 4 : 8; }
// A launch's rows; fp32 takes two launches a direction for twice as many, bf16 none (its matrix instructions' kernels read the weights
// less often: 9 rows on 50257 of 512 120 us).  Both directions (us, matrix instructions' kernels and these): fp32, 1 row on 128789 words
// of 256 385 and 81, 8 on 50257 of 1024 398 and 157, 2 on 30000 of 2048 499 and 173, 8 on 50257 of 2048 1027 and 624, 16 on 50257 of
// 1024 400 and 286, 16 on 50257 of 512 219 and 167; bf16, 5 on 100000 of 1024 323 and 187, 4 on 50257 of 2048 359 and 213, 8 on 128000
// of 256 158 and 138, 2 on 50257 of 101 141 and 136 (the host).  A bf16 forward that reads the weights as they are stays with the matrix instructions: 5 on 100000 of
// 1024 41 and 50, 8 on 128000 of 256 25 and 39; with copies it does not, 2 on 50257 of 101 32 and 25.  But where a backward follows
// the forward takes the backward's kernels: scores that are summed in another order are off by 2^-24 of themselves, which is
// what a probability is off by then, and is not small for large ones.
bool vector_rows(const mb_linear_ce* a, bool backward) {
    const bool f32 = a->dtype == MB_DTYPE_F32;
    if (!backward && !a->dloss && !f32 && as_it_is<FewBf16>(a->D, a->weight, a->weight_ld)) return false;
    return a->N <= (f32 ? 2 : 1) * launch_rows(a->D, f32 ? 4 : 2);
}

struct FewBuffers {
    float2* part;
    float *target_score, *part_h;
    double* sums;
    int64_t bytes;
};
FewBuffers few_buffers(const mb_linear_ce* a, bool backward, void* base) {
    Carve c = {(char*)base};
    FewBuffers b = {};
    if (backward) {
        b.part_h = c.take<float>((int64_t)kFewGrads * a->N * pad(a->D, 4));
    } else {
        b.part = c.take<float2>((int64_t)kFewStats * a->N), b.target_score = c.take<float>(a->N), b.sums = c.take<double>(2);
    }
    b.bytes = c.used;
    return b;
}

template <typename T, int R, int C>
int few_launch(const char* what, const FewArgs& f, bool backward, int blocks, hipStream_t st) {
    typedef Few<T, R, C> F;
    static_assert(2 * F::kLds <= 65536, "no more than a kernel has without being told");
    if constexpr (sizeof(T) == 4 && R == std::min(kVectorRows, 128 / C)) {
        if (backward && f.rows1) {
            hipLaunchKernelGGL((ce_few_grads_kernel<T, R, C, true>), dim3(blocks), dim3(kFewThreads), 2 * F::kLds, st, f);
            return check_launch(what);
        }
    }
    if (backward) hipLaunchKernelGGL((ce_few_grads_kernel<T, R, C, false>), dim3(blocks), dim3(kFewThreads), F::kLds, st, f);
    else hipLaunchKernelGGL((ce_few_stats_kernel<T, R, C>), dim3(blocks), dim3(kFewThreads), F::kLds, st, f);
    return check_launch(what);
}
template <typename T, int C>
int few_by_rows(const char* what, const FewArgs& f, bool backward, int blocks, hipStream_t st) {
    const int rows = few_rows(f.rows);
    if (rows == 1) return few_launch<T, 1, C>(what, f, backward, blocks, st);
    if (rows == 2) return few_launch<T, 2, C>(what, f, backward, blocks, st);
    if (rows == 4) return few_launch<T, 4, C>(what, f, backward, blocks, st);
    if constexpr (8 * C <= 128) return few_launch<T, 8, C>(what, f, backward, blocks, st);
    return fail(MB_ERR_UNSUPPORTED, "%s: %d rows of %d", what, f.rows, f.D);
}
template <typename T>
int few(const char* what, const mb_linear_ce* a, bool backward, hipStream_t st) {
    const FewBuffers b = few_buffers(a, backward, a->workspace);
    if (const int rc = enough(what, a, b.bytes)) return rc;
    if (const int rc = apart(what, a, backward)) return rc;
    if (backward && !a->dhidden && !a->dweight) return MB_OK;
    constexpr int vec = 16 / sizeof(T);
    FewArgs f = {};
    f.hidden = a->hidden, f.weight = a->weight, f.h_ld = a->hidden_ld, f.w_ld = a->weight_ld;
    f.g = {{a->target, (int)a->target_bytes, a->ignore_index, a->V}, backward ? a->dloss : nullptr, a->count, (int)a->reduction};
    f.N = (int)a->N, f.V = (int)a->V, f.D = (int)a->D, f.D4 = (int)pad(a->D, 4);
    f.vec = ((uintptr_t)a->weight & 15) == 0 && a->weight_ld % vec == 0 && a->D % vec == 0;
    f.part = b.part, f.target_score = b.target_score;
    if (backward) {
        f.lse = a->lse, f.part_h = a->dhidden ? b.part_h : nullptr, f.dweight = a->dweight;
        f.out_vec = ((uintptr_t)a->dweight & 15) == 0 && a->D % vec == 0;
    }
    // of every launch of the call, whose parts are joined together: one that finds no words has a sum of nothing
    const int blocks = (int)std::min<int64_t>(backward ? kFewGrads : kFewStats, (a->V + kFewThreads / 32 - 1) / (kFewThreads / 32));
    for (f.n0 = 0; f.n0 < f.N; f.n0 += f.rows) {
        int rc = MB_OK;
        f.rows = std::min(f.N - f.n0, launch_rows(a->D, sizeof(T)));
        if (backward && f.n0) {      // dw has all rows from the first launch
            f.dweight = nullptr, f.rows1 = 0;
            if (!a->dhidden) break;
        } else if (a->dweight) {
            f.n1 = f.rows, f.rows1 = f.N - f.rows;
        }
        switch (few_channels(a->D, sizeof(T))) {
            case 4: if constexpr (vec == 4) rc = few_by_rows<T, 4>(what, f, backward, blocks, st); break;
            case 8: rc = few_by_rows<T, 8>(what, f, backward, blocks, st); break;
            case 16: rc = few_by_rows<T, 16>(what, f, backward, blocks, st); break;
            default: rc = few_by_rows<T, 32>(what, f, backward, blocks, st);
        }
        if (rc) return rc;
        if (backward && a->dhidden)
            hipLaunchKernelGGL((ce_few_sum_kernel<T>), dim3((unsigned)((f.rows * f.D4 / 4 + 15) / 16)), dim3(kThreads), 0, st, (const float*)b.part_h,
                               blocks, f.g, f.n0, f.rows, f.D, f.D4, (T*)a->dhidden + (int64_t)f.n0 * a->D);
    }
    if (backward) return check_launch(what);
    static_assert(2 * kVectorRows <= kRowsPerBlock, "one workgroup joins");
    const JoinArgs j = {b.part, b.target_score, f.g.t, {nullptr, nullptr, nullptr, f.N}, f.N, blocks, (int)a->reduction, a->loss, a->lse, a->count, b.sums};
    hipLaunchKernelGGL(ce_join_kernel, dim3(1), dim3(kThreads), 0, st, j);
    if (a->reduction) hipLaunchKernelGGL(ce_total_kernel, dim3(1), dim3(kThreads), 0, st, (const double*)b.sums, 1, (int)a->reduction, a->loss, a->count);
    return check_launch(what);
}

template <typename C>
int forward(const mb_linear_ce* a, hipStream_t st) {
    const Plan p = plan_of<C>(a);
    const Buffers b = buffers_of(p, false, a->workspace);
    if (const int rc = fits("mb_linear_ce_fwd", a, p, 0)) return rc;
    if (const int rc = enough("mb_linear_ce_fwd", a, b.bytes)) return rc;
    if (const int rc = apart("mb_linear_ce_fwd", a, false)) return rc;
    ScoreArgs s = {};
    const RowGrad g = {{a->target, (int)a->target_bytes, a->ignore_index, a->V}, nullptr, nullptr, 0};
    operands<C>(a, p, b, s, g, false, false, st);
    s.part = b.part, s.target_score = b.target_score;
    if (const int rc = stats<typename C::Score>(s, p.tiles_q, st)) return rc;
    const int blocks = (int)((p.N + kRowsPerBlock - 1) / kRowsPerBlock);
    const JoinArgs j = {b.part, b.target_score, g.t, s.r, (int)p.N, p.tiles_p, (int)a->reduction, a->loss, a->lse, a->count, b.sums};
    hipLaunchKernelGGL(ce_join_kernel, dim3(blocks), dim3(kThreads), 0, st, j);
    if (a->reduction)
        hipLaunchKernelGGL(ce_total_kernel, dim3(1), dim3(kThreads), 0, st, b.sums, blocks, (int)a->reduction, a->loss, a->count);
    return check_launch("mb_linear_ce_fwd");
}

template <typename C>
int backward(const mb_linear_ce* a, hipStream_t st) {
    typedef typename C::T T;
    const Plan p = plan_of<C>(a);
    const Buffers b = buffers_of(p, true, a->workspace);
    if (const int rc = fits("mb_linear_ce_bwd", a, p, (p.D + C::GradH::TP - 1) / C::GradH::TP)) return rc;
    if (const int rc = enough("mb_linear_ce_bwd", a, b.bytes)) return rc;
    if (const int rc = apart("mb_linear_ce_bwd", a, true)) return rc;
    const bool wants_h = a->dhidden, wants_w = a->dweight;
    if (!wants_h && !wants_w) return MB_OK;
    ScoreArgs s = {};
    const RowGrad g = {{a->target, (int)a->target_bytes, a->ignore_index, a->V}, a->dloss, a->count, (int)a->reduction};
    operands<C>(a, p, b, s, g, wants_h, wants_w, st);
    constexpr bool f32 = sizeof(T) == 4;
    s.lse = a->lse, s.u = f32 && !wants_h ? nullptr : b.u, s.u_w = wants_w ? b.u_w : nullptr, s.exps_h = b.exps_h, s.exps_w = b.exps_w, s.Np = (int)p.Np, s.width = p.width, s.plane = p.Np * p.width;
    const float *scale_h = f32 ? nullptr : b.scales, *scale_w = f32 ? nullptr : b.scales + 1;
    for (int64_t v0 = 0; v0 < p.V; v0 += p.width) {
        const int64_t v1 = std::min(p.V, v0 + p.width), kv = pad(v1 - v0, kPad);
        s.v0 = (int)v0, s.v1 = (int)v1;
        s.tiles_p = (int)((v1 - v0 + C::U::TP - 1) / C::U::TP);
        if (const int rc = piece_of_u<typename C::U>(s, p.tiles_q, st)) return rc;
        PartArgs ph = {}, pw = {};
        SumArgs sh = {}, sw = {};
        ph.r = pw.r = s.r, pw.k_rows = 1;
        if (wants_h) {
            ph.p = {b.w16 + v0 * p.Dp, p.Vp * p.Dp * 2, p.Dp, (int)p.D};
            ph.q = {b.u, s.plane * 2, p.width, (int)p.N};
            ph.exps = b.exps_h, ph.exps_ld = p.Np;
            ph.splits = (int)std::min<int64_t>(p.s_h, kv / kPad), ph.k1 = (int)kv, ph.out = b.part_h, ph.ld = p.Dp, ph.add = v0 > 0;
            tiles_for<typename C::GradH>(ph);
            if (v1 == p.V)
                sh = {b.part_h, p.s_h, (int)p.N, (int)p.D, (int)p.Dp, 1, (int)blocks_for(p.N * p.Dp / 4), scale_h, a->dhidden};
        }
        if (wants_w) {
            pw.p = {b.h16, p.Np * p.Dp * 2, p.Dp, (int)p.D};
            pw.q = {f32 ? b.u_w : b.u, s.plane * 2, p.width, (int)(v1 - v0)};
            pw.exps = b.exps_w, pw.exps_ld = p.width;
            pw.splits = p.s_w, pw.k1 = (int)p.Np, pw.out = b.part_w, pw.ld = p.Dp;
            tiles_for<typename C::GradW>(pw);
            if (p.s_w == 1) pw.scale = scale_w, pw.result = (T*)a->dweight + v0 * p.D;
            else sw = {b.part_w, p.s_w, (int)(v1 - v0), (int)p.D, (int)p.Dp, 0, (int)blocks_for((v1 - v0) * p.Dp / 4), scale_w,
                  (T*)a->dweight + v0 * p.D};
        }
        if (const int rc = parts<C>(ph, pw, st)) return rc;
        if (sh.blocks + sw.blocks)
            hipLaunchKernelGGL((ce_sum_kernel<T>), dim3(sh.blocks + sw.blocks), dim3(kThreads), 0, st, sh, sw, g, s.r);
    }
    return check_launch("mb_linear_ce_bwd");
}

}  // namespace
}  // namespace mb

using namespace mb;

extern "C" int64_t mb_linear_ce_workspace(const mb_linear_ce* a, int backward) {
    if (check("mb_linear_ce_workspace", a)) return -1;
    if (vector_rows(a, backward != 0)) return few_buffers(a, backward != 0, nullptr).bytes;
    const bool few = a->N <= kFewRows;
    const Plan p = a->dtype == MB_DTYPE_F32 ? few ? plan_of<FewF32>(a) : plan_of<F32>(a) : few ? plan_of<FewBf16>(a) : plan_of<Bf16>(a);
    return buffers_of(p, backward != 0, nullptr).bytes;
}

extern "C" int mb_linear_ce_fwd(const mb_linear_ce* a, void* stream) {
    if (const int rc = check("mb_linear_ce_fwd", a)) return rc;
    MB_REQUIRE(a->loss, "mb_linear_ce_fwd: null pointer argument");
    hipStream_t st = (hipStream_t)stream;
    if (vector_rows(a, false)) return a->dtype == MB_DTYPE_F32 ? few<float>("mb_linear_ce_fwd", a, false, st) : few<__bf16>("mb_linear_ce_fwd", a, false, st);
    if (a->N <= kFewRows) return a->dtype == MB_DTYPE_F32 ? forward<FewF32>(a, st) : forward<FewBf16>(a, st);
    return a->dtype == MB_DTYPE_F32 ? forward<F32>(a, st) : forward<Bf16>(a, st);
}

extern "C" int mb_linear_ce_bwd(const mb_linear_ce* a, void* stream) {
    if (const int rc = check("mb_linear_ce_bwd", a)) return rc;
    MB_REQUIRE(a->dloss, "mb_linear_ce_bwd: null pointer argument");
    hipStream_t st = (hipStream_t)stream;
    if (vector_rows(a, true)) return a->dtype == MB_DTYPE_F32 ? few<float>("mb_linear_ce_bwd", a, true, st) : few<__bf16>("mb_linear_ce_bwd", a, true, st);
    if (a->N <= kFewRows) return a->dtype == MB_DTYPE_F32 ? backward<FewF32>(a, st) : backward<FewBf16>(a, st);
    return a->dtype == MB_DTYPE_F32 ? backward<F32>(a, st) : backward<Bf16>(a, st);
}
