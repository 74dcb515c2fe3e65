// Orthogonalised matrices by Newton-Schulz products, and the optimiser's step that applies them, on gfx950.
//
//   X = G / (|G|_F + eps), transposed where it has more rows than columns;  `steps` times:
//   A = X X^T,  B = b A + c A^2,  X <- a X + B X
//   step:  M <- mu M + g,  G = g + mu M (or M),  P <- P (1 - lr decay) - lr rate X
//
// Bound by the matrix instructions (gemm16.h), for small matrices by the number of launches: all matrices of a
// call go through every launch together.  The iterations multiply what is lost in small directions by a few hundred
// (a a a a a), so X, A and B are held as two fp16 planes (24 bits), whatever the type of G.  Their scales are powers
// of two from bounds on the iterates (the largest singular value of X is at most 1 at first, and the polynomial's
// largest value on the interval after each step): nothing is measured in between.  A and B are symmetric: of the
// tiles above and below the diagonal one is computed and written twice.
//
// What the launches work on is written to the workspace once, by a launch that has it in its arguments.
#include "gemm16.h"

#include <algorithm>
#include <new>
#include <vector>

namespace mb {
namespace {

using namespace g16;

constexpr int kThreads = 256;
constexpr int kChunk = 8192;     // elements of a workgroup in the norms' launch
constexpr int kSquare = 64;      // of the planes' launch

// The products by tiles of TILE x TILE: A and B (X and A with themselves), and X (B with X).
template <int TILE>
struct By;
template <>
struct By<128> {
    typedef Product<_Float16, 2, 128, 128, kRows, kRows, 2, 4, 64> Gram;
    typedef Product<_Float16, 2, 128, 128, kCols, kRows> Apply;
};
template <>
struct By<64> {
    typedef Product<_Float16, 2, 64, 64, kRows, kRows, 2, 2, 64> Gram;
    typedef Product<_Float16, 2, 64, 64, kCols, kRows, 2, 2, 64> Apply;
};

struct Mat {
    const void* src;             // the matrix, or the gradient of a step
    void *dst, *momentum;
    float* u;                    // a step's G
    _Float16 *x[2], *a, *b;      // [2][mp, np], [2][mp, mp]
    double* part;                // [chunks]
    int rows, cols, m, n, mp, np, chunks;
    uint8_t src_bf16, dst_bf16, momentum_bf16, tall;
    float rate;
};
enum { kFirstChunk, kFirstSquare, kFirstPair, kFirstPair64, kFirstTile, kFirstTile64, kFirsts };

constexpr int kMatsOfLaunch = 24;
struct TableArgs {
    Mat m[kMatsOfLaunch];
    int first[kFirsts][kMatsOfLaunch];
    Mat* to;
    int* to_first;               // [kFirsts][count]
    int at, n, count;
};
static_assert(sizeof(TableArgs) <= 4096, "kernel arguments");

__global__ void muon_table_kernel(const TableArgs a) {
    const int i = threadIdx.x;
    if (i >= a.n) return;
    a.to[a.at + i] = a.m[i];
    for (int f = 0; f < kFirsts; ++f) a.to_first[f * a.count + a.at + i] = a.first[f][i];
}

// Each of the eight XCDs, to which workgroups go in turn, takes a run of a launch's tiles, of about the same cost each:
// what a matrix's tiles share is fetched into one or two L2s instead of all eight.
constexpr int kXcds = 8;
struct Runs {
    int from[kXcds + 1];
};

struct Args {
    const Mat* mats;
    const int* first;            // [kFirsts][count]
    int count;
    int from, to;                // X's buffers
    float a, b, c;
    float x_scale, a_scale, b_scale;
    double eps;
    float lr, mu, keep;          // keep = 1 - lr decay
    int nesterov, is_step, last;
    Runs runs;                   // of this launch
    float* parts;                // A's tiles, k split
    int splits, tiles;
};

// The workgroup's tile, or -1.
__device__ inline int tile_of(const Runs& r) {
    const int xcd = blockIdx.x % kXcds, id = r.from[xcd] + (int)(blockIdx.x / kXcds);
    return id < r.from[xcd + 1] ? id : -1;
}

// The matrix that holds item `id` of a launch, and the item's number in it.
__device__ inline Mat find(const Args& a, int which, int& id) {
    const int* first = a.first + which * a.count;
    const int lane = threadIdx.x & 63;
    int at = 0;
    for (int base = 0; base < a.count; base += 64) {
        const int i = base + lane;
        at += __popcll(__ballot(i < a.count && first[i] <= id));
    }
    at = __builtin_amdgcn_readfirstlane(at - 1);
    id -= __builtin_amdgcn_readfirstlane(first[at]);
    return a.mats[at];
}

__device__ inline float load1(const void* p, int64_t i, bool bf16) { return bf16 ? (float)((const __bf16*)p)[i] : ((const float*)p)[i]; }
__device__ inline void store1(void* p, int64_t i, bool bf16, float v) {
    if (bf16) ((__bf16*)p)[i] = (__bf16)v;
    else ((float*)p)[i] = v;
}

__device__ inline f32x4v load4(const void* p, int64_t i, bool bf16) {
    if (!bf16) return *reinterpret_cast<const f32x4v*>((const float*)p + i);
    typedef __bf16 bf16x4v __attribute__((ext_vector_type(4)));
    const bf16x4v q = *reinterpret_cast<const bf16x4v*>((const __bf16*)p + i);
    return f32x4v{(float)q[0], (float)q[1], (float)q[2], (float)q[3]};
}
__device__ inline void store4(void* p, int64_t i, bool bf16, f32x4v v) {
    if (!bf16) {
        *reinterpret_cast<f32x4v*>((float*)p + i) = v;
    } else {
        typedef __bf16 bf16x4v __attribute__((ext_vector_type(4)));
        *reinterpret_cast<bf16x4v*>((__bf16*)p + i) = bf16x4v{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
    }
}
// Whether four elements at a multiple of four are aligned as load4 wants them.
__device__ inline bool fours(const void* p, bool bf16) { return ((uintptr_t)p & (bf16 ? 7 : 15)) == 0; }

__device__ inline double block_sum(double v) {
    __shared__ double s[16];
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = s[0];
    for (int i = 1; i < (int)blockDim.x / 64; ++i) v += s[i];
    __syncthreads();
    return v;
}

// Sums of squares in 64 bits; a step's momentum and G first.  HBM-bound at a distance: 48 matrices of the six-layer model in fp32 54.8 us.
__global__ void __launch_bounds__(kThreads) muon_norm_kernel(const Args a) {
    int chunk = blockIdx.x;
    const Mat m = find(a, kFirstChunk, chunk);
    const int64_t total = (int64_t)m.rows * m.cols, e0 = (int64_t)chunk * kChunk, e1 = std::min(total, e0 + kChunk);
    double sum = 0.0;
    const bool four = fours(m.src, m.src_bf16) && (!a.is_step || fours(m.momentum, m.momentum_bf16));
    const int64_t e4 = four ? e0 + (e1 - e0) / 4 * 4 : e0;
#pragma unroll 4
    for (int64_t e = e0 + 4 * threadIdx.x; e < e4; e += 4 * kThreads) {
        f32x4v g = load4(m.src, e, m.src_bf16);
        if (a.is_step) {
            const f32x4v mom = a.mu * load4(m.momentum, e, m.momentum_bf16) + g;
            store4(m.momentum, e, m.momentum_bf16, mom);
            g = a.nesterov ? g + a.mu * mom : mom;
            *reinterpret_cast<f32x4v*>(m.u + e) = g;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) sum = __builtin_fma((double)g[i], (double)g[i], sum);
    }
    for (int64_t e = e4 + threadIdx.x; e < e1; e += kThreads) {
        float g = load1(m.src, e, m.src_bf16);
        if (a.is_step) {
            const float mom = a.mu * load1(m.momentum, e, m.momentum_bf16) + g;
            store1(m.momentum, e, m.momentum_bf16, mom);
            g = a.nesterov ? g + a.mu * mom : mom;
            m.u[e] = g;
        }
        sum = __builtin_fma((double)g, (double)g, sum);
    }
    sum = block_sum(sum);
    if (threadIdx.x == 0) m.part[chunk] = sum;
}

// X's planes from G, 64 x 64 of X at a time, zeros around it.
__global__ void __launch_bounds__(kThreads) muon_planes_kernel(const Args a) {
    __shared__ float tile[kSquare][kSquare + 1];
    int id = blockIdx.x;
    const Mat m = find(a, kFirstSquare, id);
    double sum = 0.0;
    for (int i = threadIdx.x; i < m.chunks; i += kThreads) sum += m.part[i];
    const double f = (double)a.x_scale / (sqrt(block_sum(sum)) + a.eps);
    const int across = m.np / kSquare;
    const int i0 = id / across * kSquare, j0 = id % across * kSquare;
    const void* src = a.is_step ? (const void*)m.u : m.src;
    const bool bf16 = !a.is_step && m.src_bf16;
    // rows and columns of the source's own square; a tall matrix's is turned on the way to LDS
    const int r0 = m.tall ? j0 : i0, c0 = m.tall ? i0 : j0;
    const bool four = m.cols % 4 == 0 && fours(src, bf16);
    const int c = threadIdx.x % 16 * 4;
#pragma unroll
    for (int r = threadIdx.x / 16; r < kSquare; r += kThreads / 16) {
        f32x4v v = {0.f, 0.f, 0.f, 0.f};
        const int64_t at = (int64_t)(r0 + r) * m.cols + c0 + c;
        if (r0 + r < m.rows) {
            if (four && c0 + c < m.cols) {
                v = load4(src, at, bf16);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c0 + c + e < m.cols) v[e] = load1(src, at + e, bf16);
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) (m.tall ? tile[c + e][r] : tile[r][c + e]) = (float)((double)v[e] * f);
    }
    __syncthreads();
#pragma unroll
    for (int n = threadIdx.x; n < kSquare * kSquare / 8; n += kThreads) {
        const int r = n / 8, p = n % 8 * 8;
        f16x8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            _Float16 h, l;
            split(tile[r][p + e], h, l);
            hi[e] = h, lo[e] = l;
        }
        const int64_t to = (int64_t)(i0 + r) * m.np + j0 + p;
        *reinterpret_cast<f16x8*>(m.x[0] + to) = hi;
        *reinterpret_cast<f16x8*>(m.x[0] + (int64_t)m.mp * m.np + to) = lo;
    }
}

__device__ inline void split4(const float* v, f16x4& hi, f16x4& lo) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        _Float16 h, l;
        split(v[e], h, l);
        hi[e] = h, lo[e] = l;
    }
}

// Tile `id` of the pairs: id = q (q + 1) / 2 + p, p <= q.
template <int TILE>
__device__ inline void pair_place(int id, int& p0, int& q0) {
    int q = (int)((sqrtf(8.f * id + 1.f) - 1.f) * 0.5f);
    while (q * (q + 1) / 2 > id) --q;
    while ((q + 1) * (q + 2) / 2 <= id) ++q;
    q = uniform(q);
    p0 = (id - q * (q + 1) / 2) * TILE, q0 = q * TILE;
}

// The sums of a pair's tile to A or B, on both sides of the diagonal.
template <bool POLY, typename Gram>
__device__ inline void pair_out(const Args& a, const Mat& m, const Gram& g, int p0, int q0, char* smem) {
    const int64_t plane = (int64_t)m.mp * m.mp;
    if (POLY) {
#pragma unroll
        for (int h = 0; h < 2; ++h) Gram::fetch(smem, h, m.a + h * plane, m.mp, p0, q0, m.mp, m.mp);
        __syncthreads();
    }
    _Float16* out = POLY ? m.b : m.a;
    const float from = POLY ? a.a_scale : a.x_scale, to = POLY ? a.b_scale : a.a_scale;
    const float f = (POLY ? a.c : 1.f) * to / from / from, fb = a.b * to / a.a_scale;
#pragma unroll
    for (int j = 0; j < Gram::FQ; ++j)
#pragma unroll
        for (int i = 0; i < Gram::FP; ++i)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                f16x4 &hi = Gram::held(smem, 0, i, j, r), &lo = Gram::held(smem, 1, i, j, r);
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[e] = g.acc[i][j][r + e] * f;
                    if (POLY) v[e] += fb * ((float)hi[e] + (float)lo[e]);
                }
                split4(v, hi, lo);
            }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        Gram::store(smem, h, out + h * plane, m.mp, p0, q0, m.mp, m.mp);
        if (p0 != q0) Gram::store_turned(smem, h, out + h * plane, m.mp, p0, q0, m.mp, m.mp);
    }
}

// POLY: B = b A + c A^2 from A's planes; otherwise A = X X^T.  Matrix instructions bound it: 4 matrices of 2816 x 1024 67 us for
// A (526 TFLOP/s, three products an element, one side of the diagonal counted: 36 tiles of 128 each on 256 CUs), 32 us for B.
template <bool POLY, int TILE>
__global__ void __launch_bounds__(By<TILE>::Gram::kThreads, By<TILE>::Gram::kWaves) muon_pair_kernel(const Args a) {
    typedef typename By<TILE>::Gram Gram;
    static_assert(2 * Gram::kOutPlane <= Gram::kLds, "results go out through LDS");
    extern __shared__ char smem[];
    int id = tile_of(a.runs), p0, q0;
    if (id < 0) return;
    const Mat m = find(a, TILE == 64 ? kFirstPair64 : kFirstPair, id);
    pair_place<TILE>(id, p0, q0);
    const Side side = POLY ? Side{m.a, (int64_t)m.mp * m.mp * 2, m.mp, m.mp} : Side{m.x[a.from], (int64_t)m.mp * m.np * 2, m.np, m.mp};
    Gram g;
    g.run(side, side, p0, q0, 0, POLY ? m.mp : m.np, smem);
    __syncthreads();
    pair_out<POLY>(a, m, g, p0, q0, smem);
}

// A's tiles with k split, for few of them: the sums of a run of k, as the lanes hold them, to `parts` [splits][tiles][4096],
// and a launch that adds them in the runs' order.  A matrix with fewer steps than runs has empty ones, zeros.
typedef By<64>::Gram Part;
static_assert(Part::FP * Part::FQ == 1 && Part::kThreads * 16 == kSquare * kSquare, "a block of 16 values a lane");
__device__ inline f32x4v* part_at(const Args& a, int split, int id) {
    return (f32x4v*)a.parts + ((int64_t)split * a.tiles + id) * (kSquare * kSquare / 4) + threadIdx.x;
}
__global__ void __launch_bounds__(Part::kThreads, Part::kWaves) muon_part_kernel(const Args a) {
    extern __shared__ char smem[];
    int id = tile_of(a.runs), p0, q0;
    if (id < 0) return;
    f32x4v* to = part_at(a, blockIdx.y, id);
    const Mat m = find(a, kFirstPair64, id);
    pair_place<64>(id, p0, q0);
    const int steps = m.np / Part::kStep;
    const int k0 = steps * (int)blockIdx.y / a.splits * Part::kStep, k1 = steps * ((int)blockIdx.y + 1) / a.splits * Part::kStep;
    const Side side = {m.x[a.from], (int64_t)m.mp * m.np * 2, m.np, m.mp};
    Part g;
    if (k1 > k0) g.run(side, side, p0, q0, k0, k1, smem);
    else g.clear();
    const f32x16& v = g.acc[0][0];
#pragma unroll
    for (int r = 0; r < 16; r += 4) to[r / 4 * Part::kThreads] = f32x4v{v[r], v[r + 1], v[r + 2], v[r + 3]};
}
__global__ void __launch_bounds__(Part::kThreads) muon_join_kernel(const Args a) {
    extern __shared__ char smem[];
    int id = blockIdx.x, p0, q0;
    f32x4v v[4] = {};
#pragma unroll 4
    for (int split = 0; split < a.splits; ++split) {
        const f32x4v* from = part_at(a, split, id);
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] += from[r * Part::kThreads];
    }
    const Mat m = find(a, kFirstPair64, id);
    pair_place<64>(id, p0, q0);
    Part g;
#pragma unroll
    for (int r = 0; r < 16; ++r) g.acc[0][0][r] = v[r / 4][r % 4];
    pair_out<false>(a, m, g, p0, q0, smem);
}

// X <- a X + B X.  4 matrices of 2816 x 1024: 97 us, 733 TFLOP/s of three products an element.
template <int TILE>
__global__ void __launch_bounds__(By<TILE>::Apply::kThreads, By<TILE>::Apply::kWaves) muon_apply_kernel(const Args a) {
    typedef typename By<TILE>::Apply Apply;
    static_assert(2 * Apply::kOutPlane <= Apply::kLds && Apply::kOut32 <= Apply::kLds, "results go out through LDS");
    extern __shared__ char smem[];
    int id = tile_of(a.runs);
    if (id < 0) return;
    const Mat m = find(a, TILE == 64 ? kFirstTile64 : kFirstTile, id);
    const int across = (m.np + TILE - 1) / TILE;
    const int p0 = id % across * TILE, q0 = id / across * TILE;
    const int64_t plane = (int64_t)m.mp * m.np;
    const _Float16* x = m.x[a.from];
    Apply g;
    // X's own tile comes by among the rows of X that are multiplied: at k = the lane's row of the result
    f16x4 xh[Apply::FQ][Apply::FP][4], xl[Apply::FQ][Apply::FP][4];
    g.run(Side{x, plane * 2, m.np, m.np}, Side{m.b, (int64_t)m.mp * m.mp * 2, m.mp, m.mp}, p0, q0, 0, m.mp, smem, [&](int k, uint32_t tile) {
#pragma unroll
        for (int j = 0; j < Apply::FQ; ++j) {
            const int i = q0 + Apply::wave_q() + 32 * j - k;
            if (i < 0 || i >= Apply::kStep) continue;
#pragma unroll
            for (int n = 0; n < Apply::FP; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    xh[j][n][r] = Apply::TileP::four(tile, Apply::row(n, 4 * r), i + (threadIdx.x & 31));
                    xl[j][n][r] = Apply::TileP::four(tile + Apply::TileP::kBytes, Apply::row(n, 4 * r), i + (threadIdx.x & 31));
                }
        }
    });
    // a X is added here: as a B with a on its diagonal every sum over k would be rounded at a X's size
    const float out = a.last ? 1.f / a.x_scale : 1.f, f = out / a.b_scale, fx = a.a * out;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < Apply::FQ; ++j)
#pragma unroll
        for (int i = 0; i < Apply::FP; ++i)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[e] = g.acc[i][j][r + e] * f + fx * ((float)xh[j][i][r / 4][e] + (float)xl[j][i][r / 4][e]);
                if (!a.last) split4(v, Apply::held(smem, 0, i, j, r), Apply::held(smem, 1, i, j, r));
                else Apply::held32(smem, i, j, r) = f32x4v{v[0], v[1], v[2], v[3]};
            }
    __syncthreads();
    if (!a.last) {
#pragma unroll
        for (int h = 0; h < 2; ++h) Apply::store(smem, h, m.x[a.to] + h * plane, m.np, p0, q0, m.np, m.mp);
        return;
    }
    // four values of a row of the result a thread, all that a step wants of the old weights on their way at once
    constexpr int kEach = TILE * TILE / 4 / Apply::kThreads;
    const bool four = m.cols % 4 == 0 && fours(m.dst, m.dst_bf16);
    const int r0 = m.tall ? p0 : q0, c0 = m.tall ? q0 : p0;
    f32x4v old[kEach];
    auto place = [&](int n, int& r, int& c) {
        const int i = n * Apply::kThreads + threadIdx.x;
        r = i / (TILE / 4), c = i % (TILE / 4) * 4;
        return (int64_t)(r0 + r) * m.cols + c0 + c;
    };
    if (a.is_step) {
#pragma unroll
        for (int n = 0; n < kEach; ++n) {
            int r, c;
            const int64_t at = place(n, r, c);
            if (r0 + r >= m.rows) continue;
            if (four && c0 + c < m.cols) {
                old[n] = load4(m.dst, at, m.dst_bf16);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) old[n][e] = c0 + c + e < m.cols ? load1(m.dst, at + e, m.dst_bf16) : 0.f;
            }
        }
    }
#pragma unroll
    for (int n = 0; n < kEach; ++n) {
        int r, c;
        const int64_t at = place(n, r, c);
        if (r0 + r >= m.rows) continue;
        f32x4v y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = m.tall ? Apply::out32(smem, c + e, r) : Apply::out32(smem, r, c + e);
        if (a.is_step) y = old[n] * a.keep - (a.lr * m.rate) * y;
        if (four && c0 + c < m.cols) {
            store4(m.dst, at, m.dst_bf16, y);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c0 + c + e < m.cols) store1(m.dst, at + e, m.dst_bf16, y[e]);
        }
    }
}

// ---- small matrices ----------------------------------------------------------------------
//
// Where X's and A's planes fit into a CU's LDS, one workgroup of 16 waves takes a matrix through all steps: what the
// launches of the general case, some 5 us each whatever they do, cost most there.  A wave takes 32 x 32 blocks of each
// product; B stands in A's place and X's new columns in the old ones', after a barrier: 16 blocks at a time.  8 of 128 x 128 in bf16:
// 68 us, the general launches 204.  One CU's matrix instructions take 19 us of that (15 products of 16 blocks, 24 instructions each), its
// LDS reads 26; the rest is waits, for operands that are read right before their use and at the barriers.
constexpr int kSmallThreads = 1024;
constexpr int kSmallLds = 159 * 1024;
constexpr int kSmallEach = kSmallLds / 4 / kSmallThreads;    // elements of a thread, at most

struct SmallArgs {
    Mat m[kMatsOfLaunch];
    Args a;
    int steps;
};
static_assert(sizeof(SmallArgs) <= 4096, "kernel arguments");

__host__ __device__ inline int small_lds(int mp, int np) { return 4 * mp * np + 4 * mp * mp; }

// A matrix's planes in LDS, rows of a multiple of 8 pieces, piece c of row r in the place c ^ swz(r).
struct Held {
    uint32_t lds;       // address of the first plane
    int row, plane;     // bytes
    __device__ int turn(int r) const {
        return row % 256 == 0 ? (r & 3) << 2 | ((r >> 2) & 3) : ((r >> 1) & 1) << 2 | ((r >> 3) & 1) << 1 | ((r >> 2) & 1);
    }
    __device__ uint32_t at(int h, int r, int i) const { return lds + h * plane + r * row + (((i >> 3) ^ turn(r)) << 4) + 2 * (i & 7); }
    // rows r0 + lane % 32, k = k0 + 8 (lane / 32) + 0 .. 7
    __device__ f16x8 rows(int h, int r0, int k0) const {
        const int lane = threadIdx.x & 63;
        return *(__attribute__((address_space(3))) const f16x8*)(uintptr_t)at(h, r0 + (lane & 31), k0 + 8 * (lane >> 5));
    }
    // columns i0 + lane % 32, rows k0 + 8 (lane / 32) + 0 .. 7
    __device__ f16x8 cols(int h, int i0, int k0) const {
        typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
        const int lane = threadIdx.x & 63, r = k0 + 8 * (lane >> 5) + ((lane & 15) >> 2), d = i0 + (lane & 16) + 4 * (lane & 3);
        const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)at(h, r, d));
        const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)at(h, r + 4, d));
        return __builtin_bit_cast(f16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    __device__ f16x4 four(int h, int r, int i) const { return *(__attribute__((address_space(3))) const f16x4*)(uintptr_t)at(h, r, i); }
    __device__ void four(int h, int r, int i, f16x4 v) const { *(__attribute__((address_space(3))) f16x4*)(uintptr_t)at(h, r, i) = v; }
    __device__ void one(int h, int r, int i, _Float16 v) const { *(__attribute__((address_space(3))) _Float16*)(uintptr_t)at(h, r, i) = v; }
};

// A 32 x 32 block: rows p0.. of P (or its columns), rows q0.. of Q, over k.
template <bool COLS>
__device__ inline f32x16 small_block(const Held& p, const Held& q, int p0, int q0, int k) {
    f32x16 x = {}, y = {};
    for (int k0 = 0; k0 < k; k0 += 16) {
        const f16x8 ah = COLS ? p.cols(0, p0, k0) : p.rows(0, p0, k0), al = COLS ? p.cols(1, p0, k0) : p.rows(1, p0, k0);
        const f16x8 bh = q.rows(0, q0, k0), bl = q.rows(1, q0, k0);
        y = mma(al, bh, y);
        x = mma(ah, bh, x);
        y = mma(ah, bl, y);
    }
    return x + y;
}

__global__ void __launch_bounds__(kSmallThreads) muon_small_kernel(const SmallArgs s) {
    extern __shared__ char smem[];
    const Args& a = s.a;
    const Mat& m = s.m[blockIdx.x];
    const int mp = m.mp, np = m.np, lane = threadIdx.x & 63, wave = wave_id(), total = m.rows * m.cols;
    const Held x = {lds_address(smem), 2 * np, 2 * mp * np}, g = {lds_address(smem) + 4 * mp * np, 2 * mp, 2 * mp * mp};
    // G, a few elements a thread, and its norm
    float v[kSmallEach];
    double sum = 0.0;
#pragma unroll
    for (int n = 0; n < kSmallEach; ++n) {
        const int e = n * kSmallThreads + (int)threadIdx.x;
        v[n] = 0.f;
        if (e >= total) continue;
        v[n] = load1(m.src, e, m.src_bf16);
        if (a.is_step) {
            const float mom = a.mu * load1(m.momentum, e, m.momentum_bf16) + v[n];
            store1(m.momentum, e, m.momentum_bf16, mom);
            v[n] = a.nesterov ? v[n] + a.mu * mom : mom;
        }
        sum = __builtin_fma((double)v[n], (double)v[n], sum);
    }
    for (int i = threadIdx.x; i < mp * np / 4; i += kSmallThreads) ((f32x4v*)smem)[i] = f32x4v{0.f, 0.f, 0.f, 0.f};
    const double f = (double)a.x_scale / (sqrt(block_sum(sum)) + a.eps);     // its barriers are those of the zeros, too
#pragma unroll
    for (int n = 0; n < kSmallEach; ++n) {
        const int e = n * kSmallThreads + (int)threadIdx.x;
        if (e >= total) continue;
        const int r = e / m.cols, c = e - r * m.cols;
        _Float16 hi, lo;
        split((float)((double)v[n] * f), hi, lo);
        x.one(0, m.tall ? c : r, m.tall ? r : c, hi);
        x.one(1, m.tall ? c : r, m.tall ? r : c, lo);
    }
    __syncthreads();
    const int bm = mp / 32, bn = np / 32;
    const float to_a = a.a_scale / a.x_scale / a.x_scale, square = a.c * a.b_scale / a.a_scale / a.a_scale, linear = a.b * a.b_scale / a.a_scale;
    const int col = lane & 31, row0 = 4 * (lane >> 5);
    for (int step = 0; step < s.steps; ++step) {
        const bool last = step + 1 == s.steps;
        const int q0 = wave / bm * 32, p0 = wave % bm * 32;      // bm * bm is at most 16
        if (wave < bm * bm) {
            const f32x16 acc = small_block<false>(x, x, p0, q0, np);
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const float w[4] = {acc[r] * to_a, acc[r + 1] * to_a, acc[r + 2] * to_a, acc[r + 3] * to_a};
                f16x4 hi, lo;
                split4(w, hi, lo);
                g.four(0, q0 + col, p0 + 2 * r + row0, hi);
                g.four(1, q0 + col, p0 + 2 * r + row0, lo);
            }
        }
        __syncthreads();
        f16x4 hi[4], lo[4];
        if (wave < bm * bm) {
            const f32x16 acc = small_block<false>(g, g, p0, q0, mp);
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int p = p0 + 2 * r + row0;
                const f16x4 h = g.four(0, q0 + col, p), l = g.four(1, q0 + col, p);
                float w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    w[e] = acc[r + e] * square + linear * ((float)h[e] + (float)l[e]);
                split4(w, hi[r / 4], lo[r / 4]);
            }
        }
        __syncthreads();
        if (wave < bm * bm)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                g.four(0, q0 + col, p0 + 2 * r + row0, hi[r / 4]);
                g.four(1, q0 + col, p0 + 2 * r + row0, lo[r / 4]);
            }
        __syncthreads();
        const float out = last ? 1.f / a.x_scale : 1.f, f = out / a.b_scale, fx = a.a * out;
        const int wide = 16 / bm;                                 // columns' blocks at a time
        for (int b0 = 0; b0 < bn; b0 += wide) {
            const int i0 = wave % bm * 32, j0 = (b0 + wave / bm) * 32;
            const bool mine = wave < bm * wide && j0 < np;
            f32x16 acc = {};
            if (mine) {
                acc = small_block<true>(x, g, j0, i0, mp);
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const f16x4 h = x.four(0, i0 + col, j0 + 2 * r + row0), l = x.four(1, i0 + col, j0 + 2 * r + row0);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[r + e] = acc[r + e] * f + fx * ((float)h[e] + (float)l[e]);
                }
            }
            if (last) {
                const int i = i0 + col;
                if (mine && i < m.m)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int j = j0 + 8 * (r / 4) + row0 + r % 4;
                        if (j >= m.n) continue;
                        const int to = m.tall ? j * m.cols + i : i * m.cols + j;
                        float y = acc[r];
                        if (a.is_step) y = load1(m.dst, to, m.dst_bf16) * a.keep - (a.lr * m.rate) * y;
                        store1(m.dst, to, m.dst_bf16, y);
                    }
                continue;
            }
            __syncthreads();
            if (mine)
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const float w[4] = {acc[r], acc[r + 1], acc[r + 2], acc[r + 3]};
                    f16x4 h, l;
                    split4(w, h, l);
                    x.four(0, i0 + col, j0 + 2 * r + row0, h);
                    x.four(1, i0 + col, j0 + 2 * r + row0, l);
                }
        }
        __syncthreads();
    }
}

// ---- host side ---------------------------------------------------------------------------

struct Stretch {
    uintptr_t from, to;
    bool written;
};

bool code(int64_t dtype) { return dtype == MB_DTYPE_F32 || dtype == MB_DTYPE_BF16; }
int64_t bytes_of(int64_t n, int64_t dtype) { return n * (dtype == MB_DTYPE_F32 ? 4 : 2); }

int check(const char* what, const mb_muon* p) {
    MB_REQUIRE(p, "%s: null args", what);
    MB_REQUIRE(p->count >= 0 && p->count <= (1 << 20) && (p->count == 0 || p->matrices), "%s: count=%lld", what, (long long)p->count);
    MB_REQUIRE(p->steps >= 1 && p->steps <= 100, "%s: steps=%lld (1 to 100)", what, (long long)p->steps);
    for (const int64_t e : {p->x_exponent, p->a_exponent, p->b_exponent})
        MB_REQUIRE(e >= -14 && e <= 15, "%s: an exponent of %lld (-14 to 15)", what, (long long)e);
    MB_REQUIRE(p->eps >= 0, "%s: eps=%g", what, p->eps);
    for (int64_t i = 0; i < p->count; ++i) {
        const mb_muon_matrix& m = p->matrices[i];
        MB_REQUIRE(m.rows >= 0 && m.cols >= 0 && m.rows <= (1 << 20) && m.cols <= (1 << 20) && m.rows * m.cols < ((int64_t)1 << 31)
                       && std::min(m.rows, m.cols) <= (1 << 15),
                   "%s: matrix %lld is %lld x %lld (below 2^31 elements, 2^15 x 2^20 at most)", what, (long long)i, (long long)m.rows,
                   (long long)m.cols);
        MB_REQUIRE(code(m.src_dtype) && code(m.dst_dtype) && (!p->is_step || code(m.momentum_dtype)), "%s: matrix %lld: dtype", what, (long long)i);
    }
    return MB_OK;
}

// What every launch works on; the workspace's size with a null base.
struct Layout {
    std::vector<Mat> mats;
    std::vector<int> first[kFirsts];
    int64_t blocks[kFirsts] = {};
    int splits = 1;
    float* parts = nullptr;

    // The XCDs' runs of a launch whose tiles cost their matrix's n (or m) each, and its grid.
    Runs runs(int which, bool by_n, unsigned& grid) const {
        auto cost = [&](size_t i) { return (int64_t)(by_n ? mats[i].np : mats[i].mp) + 128; };   // and what a tile takes to begin and end
        auto end = [&](size_t i) { return i + 1 < mats.size() ? first[which][i + 1] : (int)blocks[which]; };
        int64_t total = 0, before = 0;
        for (size_t i = 0; i < mats.size(); ++i) total += cost(i) * (end(i) - first[which][i]);
        Runs r = {};
        int x = 1;
        for (size_t i = 0; i < mats.size(); ++i) {
            const int n = end(i) - first[which][i];
            for (; x < kXcds && total * x / kXcds <= before + cost(i) * n; ++x)
                r.from[x] = first[which][i] + (int)((total * x / kXcds - before + cost(i) / 2) / cost(i));
            before += cost(i) * n;
        }
        for (; x <= kXcds; ++x) r.from[x] = (int)blocks[which];
        int most = 0;
        for (x = 0; x < kXcds; ++x) most = std::max(most, r.from[x + 1] - r.from[x]);
        grid = (unsigned)(most * kXcds);
        return r;
    }
};

// Runs of k for A where its tiles of 64 leave places empty: as many as fill these, each of 8 steps at least.  A step is about
// 0.77 us, so that the half of it and more that is saved pays for the join's launch, 5 - 6 us.  Whole calls, not split and
// split: one of 4096 x 1024 616 and 537 us, one of 640 x 4000 462 and 332, 8 of 64 x 2816 215 and 147, one of 48 x 2816 207 and 132.
constexpr int kPlaces = 512;
int64_t splits_of(int64_t tiles, int64_t longest) { return tiles ? std::max<int64_t>(1, std::min(kPlaces / tiles, longest / kPad / 8)) : 1; }

// What a matrix takes of the workspace: two pairs of X's planes and of A's and B's, a step's G, the norm's parts.
int64_t bytes_of_matrix(const mb_muon* p, int64_t i) {
    const mb_muon_matrix& m = p->matrices[i];
    const int64_t mp = pad(std::min(m.rows, m.cols), kPad), np = pad(std::max(m.rows, m.cols), kPad);
    return 8 * mp * (np + mp) + (p->is_step ? 4 * m.rows * m.cols : 0) + m.rows * m.cols / kChunk * 8 + 6 * 256;
}

// The matrices that go through the launches together: all, or as many as this much memory holds; then the next ones with the same memory.
// So much fills the card many times over (some 200 M elements); a list of all of a large model's matrices would want 12 to 20 bytes an element.
constexpr int64_t kGroupBytes = (int64_t)4 << 30;
typedef std::vector<int64_t> Group;
std::vector<Group> groups_of(const mb_muon* p) {
    // the longest products first: what is left at a launch's end is short
    Group order;
    for (int64_t i = 0; i < p->count; ++i)
        if (p->matrices[i].rows && p->matrices[i].cols) order.push_back(i);
    std::stable_sort(order.begin(), order.end(), [&](int64_t i, int64_t j) {
        const mb_muon_matrix &x = p->matrices[i], &y = p->matrices[j];
        return std::max(x.rows, x.cols) > std::max(y.rows, y.cols);
    });
    std::vector<Group> groups;
    int64_t held = 0;
    for (const int64_t i : order) {
        const int64_t bytes = bytes_of_matrix(p, i);
        if (groups.empty() || held + bytes > kGroupBytes) groups.emplace_back(), held = 0;
        groups.back().push_back(i), held += bytes;
    }
    return groups;
}

int64_t lay_out(const mb_muon* p, const Group& group, char* base, Layout* out) {
    int64_t used = 0, tiles = 0, longest = 0;
    auto take = [&](int64_t bytes) {
        char* at = base ? base + used : nullptr;
        used += pad(bytes, 256);
        return at;
    };
    for (const int64_t i : group) {
        const mb_muon_matrix& from = p->matrices[i];
        Mat m = {};
        m.src = from.src, m.dst = from.dst, m.momentum = from.momentum;
        m.rows = (int)from.rows, m.cols = (int)from.cols;
        m.tall = m.rows > m.cols;
        m.m = std::min(m.rows, m.cols), m.n = std::max(m.rows, m.cols);
        m.mp = (int)pad(m.m, kPad), m.np = (int)pad(m.n, kPad);
        m.src_bf16 = from.src_dtype == MB_DTYPE_BF16, m.dst_bf16 = from.dst_dtype == MB_DTYPE_BF16;
        m.momentum_bf16 = from.momentum_dtype == MB_DTYPE_BF16;
        m.rate = (float)from.rate;
        const int64_t elements = from.rows * from.cols, x = 4 * (int64_t)m.mp * m.np, a = 4 * (int64_t)m.mp * m.mp;
        m.chunks = (int)((elements + kChunk - 1) / kChunk);
        m.x[0] = (_Float16*)take(x), m.x[1] = (_Float16*)take(x);
        m.a = (_Float16*)take(a), m.b = (_Float16*)take(a);
        if (p->is_step) m.u = (float*)take(elements * 4);
        m.part = (double*)take(m.chunks * 8);
        tiles += (int64_t)(m.mp / 64) * (m.mp / 64 + 1) / 2, longest = std::max<int64_t>(longest, m.np);
        if (out) {
            const int64_t m64 = m.mp / 64, n64 = m.np / 64, m128 = (m64 + 1) / 2, n128 = (n64 + 1) / 2;
            const int64_t items[kFirsts] = {m.chunks, m64 * n64, m128 * (m128 + 1) / 2, m64 * (m64 + 1) / 2, m128 * n128, m64 * n64};
            for (int f = 0; f < kFirsts; ++f) {
                out->first[f].push_back((int)out->blocks[f]);
                out->blocks[f] += items[f];
            }
            out->mats.push_back(m);
        }
    }
    const int64_t splits = splits_of(tiles, longest);
    float* parts = splits > 1 ? (float*)take(splits * tiles * kSquare * kSquare * 4) : nullptr;
    if (out) out->splits = (int)splits, out->parts = parts;
    return used;
}

bool small_ones(const std::vector<Mat>& mats) {
    return std::all_of(mats.begin(), mats.end(), [](const Mat& m) {
        return m.mp <= 128 && (int64_t)4 * m.mp * (m.np + m.mp) <= kSmallLds && (int64_t)m.rows * m.cols <= kSmallEach * kSmallThreads;
    });
}

int64_t table_bytes(int64_t count) { return pad(count * (int64_t)sizeof(Mat), 256) + pad(count * (int64_t)sizeof(int) * kFirsts, 256); }

int64_t workspace_of(const mb_muon* p, const std::vector<Group>& groups) {
    int64_t most = 0;
    for (const Group& g : groups) most = std::max(most, lay_out(p, g, nullptr, nullptr));
    return table_bytes(p->count) + most;
}

int run(const char* what, const mb_muon* p, const Group& group, hipStream_t st) {
    Layout l;
    const int64_t table = table_bytes(p->count);
    lay_out(p, group, (char*)p->workspace + table, &l);
    const int count = (int)l.mats.size();
    if (count == 0) return MB_OK;
    for (int f = 0; f < kFirsts; ++f)
        MB_REQUIRE(l.blocks[f] <= 0xffffff, "%s: %lld workgroups, too many", what, (long long)l.blocks[f]);
    Args a = {};
    a.mats = (const Mat*)p->workspace;
    a.first = (const int*)((char*)p->workspace + pad(p->count * (int64_t)sizeof(Mat), 256));
    a.count = count;
    a.a = (float)p->a, a.b = (float)p->b, a.c = (float)p->c, a.eps = p->eps;
    a.x_scale = ldexpf(1.f, (int)p->x_exponent), a.a_scale = ldexpf(1.f, (int)p->a_exponent), a.b_scale = ldexpf(1.f, (int)p->b_exponent);
    a.lr = (float)p->lr, a.mu = (float)p->momentum, a.keep = (float)(1.0 - p->lr * p->weight_decay);
    a.nesterov = p->nesterov != 0, a.is_step = p->is_step != 0;
    // Small matrices alone: with larger ones among them the general launches are there anyway, and the small ones cost little in them.
    if (small_ones(l.mats)) {
        static Told told;
        if (const int rc = allow_lds(what, (const void*)muon_small_kernel, kSmallLds, told)) return rc;
        for (int at = 0; at < count; at += kMatsOfLaunch) {
            SmallArgs t = {};
            const int n = std::min(kMatsOfLaunch, count - at);
            t.a = a, t.steps = (int)p->steps;
            int lds = 0;
            for (int i = 0; i < n; ++i) t.m[i] = l.mats[at + i], lds = std::max(lds, small_lds(t.m[i].mp, t.m[i].np));
            hipLaunchKernelGGL(muon_small_kernel, dim3(n), dim3(kSmallThreads), lds, st, t);
        }
        return check_launch(what);
    }
    for (int at = 0; at < count; at += kMatsOfLaunch) {
        TableArgs t = {};
        t.to = (Mat*)a.mats, t.to_first = (int*)a.first, t.at = at, t.n = std::min(kMatsOfLaunch, count - at), t.count = count;
        for (int i = 0; i < t.n; ++i) {
            t.m[i] = l.mats[at + i];
            for (int f = 0; f < kFirsts; ++f) t.first[f][i] = l.first[f][at + i];
        }
        hipLaunchKernelGGL(muon_table_kernel, dim3(1), dim3(64), 0, st, t);
    }
    const dim3 blk(kThreads);
    hipLaunchKernelGGL(muon_norm_kernel, dim3((unsigned)l.blocks[kFirstChunk]), blk, 0, st, a);
    hipLaunchKernelGGL(muon_planes_kernel, dim3((unsigned)l.blocks[kFirstSquare]), blk, 0, st, a);
    // Tiles of 64 or 128, by what a round of them took for 64 k (us; 4 matrices of 2816 x 1024, 3 of 777 x 1234, 48
    // of the six-layer model): pairs 0.8 to 1.0 for up to 512 of 64 and 1.4 for 256 of 128, B X 1.35 for 512 of 64, 2.9 for 512 of 128.
    auto rounds = [](int64_t n, int64_t most) { return (double)((n + most - 1) / most); };
    const bool small_pairs = rounds(l.blocks[kFirstPair64], 512) * 0.8 < rounds(l.blocks[kFirstPair], 256) * 1.4;
    const bool small_tiles = rounds(l.blocks[kFirstTile64], 512) * 1.35 < rounds(l.blocks[kFirstTile], 512) * 2.9;
    const int pairs = small_pairs ? kFirstPair64 : kFirstPair, tiles = small_tiles ? kFirstTile64 : kFirstTile;
    a.parts = l.parts, a.splits = l.splits, a.tiles = (int)l.blocks[kFirstPair64];     // (few tiles are small pairs)
    unsigned gram_grid, poly_grid, apply_grid;
    const Runs gram_runs = l.runs(pairs, true, gram_grid), poly_runs = l.runs(pairs, false, poly_grid),
               apply_runs = l.runs(tiles, false, apply_grid);
    for (int step = 0; step < p->steps; ++step) {
        a.from = step & 1, a.to = a.from ^ 1, a.last = step + 1 == p->steps;
        const auto pair = [&](auto tile) {
            constexpr int TILE = decltype(tile)::value;
            static Told told[2];
            constexpr int lds = By<TILE>::Gram::kLds;
            const dim3 blk(By<TILE>::Gram::kThreads);
            if (const int rc = allow_lds(what, (const void*)muon_pair_kernel<false, TILE>, lds, told[0])) return rc;
            if (const int rc = allow_lds(what, (const void*)muon_pair_kernel<true, TILE>, lds, told[1])) return rc;
            a.runs = gram_runs;
            if (TILE == 64 && a.splits > 1) {
                static Told part;
                if (const int rc = allow_lds(what, (const void*)muon_part_kernel, lds, part)) return rc;
                hipLaunchKernelGGL(muon_part_kernel, dim3(gram_grid, a.splits), blk, lds, st, a);
                hipLaunchKernelGGL(muon_join_kernel, dim3(a.tiles), blk, 2 * Part::kOutPlane, st, a);
            } else {
                hipLaunchKernelGGL((muon_pair_kernel<false, TILE>), dim3(gram_grid), blk, lds, st, a);
            }
            a.runs = poly_runs;
            hipLaunchKernelGGL((muon_pair_kernel<true, TILE>), dim3(poly_grid), blk, lds, st, a);
            return MB_OK;
        };
        const auto apply = [&](auto tile) {
            constexpr int TILE = decltype(tile)::value;
            static Told told;
            constexpr int lds = By<TILE>::Apply::kLds;
            const dim3 blk(By<TILE>::Apply::kThreads);
            if (const int rc = allow_lds(what, (const void*)muon_apply_kernel<TILE>, lds, told)) return rc;
            a.runs = apply_runs;
            hipLaunchKernelGGL((muon_apply_kernel<TILE>), dim3(apply_grid), blk, lds, st, a);
            return MB_OK;
        };
        typedef std::integral_constant<int, 64> T64;
        typedef std::integral_constant<int, 128> T128;
        int rc = small_pairs ? pair(T64()) : pair(T128());
        if (rc == MB_OK) rc = small_tiles ? apply(T64()) : apply(T128());
        if (rc != MB_OK) return rc;
    }
    return check_launch(what);
}

}  // namespace
}  // namespace mb

using namespace mb;

extern "C" int64_t mb_muon_workspace(const mb_muon* p) try {
    if (check("mb_muon_workspace", p)) return -1;
    return workspace_of(p, groups_of(p));
} catch (const std::bad_alloc&) {
    fail(MB_ERR_INVALID_ARGUMENT, "mb_muon_workspace: no host memory");
    return -1;
}

extern "C" int mb_muon_run(const mb_muon* p, void* stream) try {
    const char* what = "mb_muon_run";
    if (const int rc = check(what, p)) return rc;
    std::vector<Stretch> s;
    for (int64_t i = 0; i < p->count; ++i) {
        const mb_muon_matrix& m = p->matrices[i];
        const int64_t n = m.rows * m.cols;
        if (n == 0) continue;
        MB_REQUIRE(m.src && m.dst && (!p->is_step || m.momentum), "%s: matrix %lld: null pointer argument", what, (long long)i);
        s.push_back({(uintptr_t)m.src, (uintptr_t)m.src + bytes_of(n, m.src_dtype), false});
        s.push_back({(uintptr_t)m.dst, (uintptr_t)m.dst + bytes_of(n, m.dst_dtype), true});
        if (p->is_step) s.push_back({(uintptr_t)m.momentum, (uintptr_t)m.momentum + bytes_of(n, m.momentum_dtype), true});
    }
    std::sort(s.begin(), s.end(), [](const Stretch& x, const Stretch& y) { return x.from < y.from; });
    uintptr_t any = 0, written = 0;
    for (const Stretch& x : s) {
        MB_REQUIRE(x.from >= (x.written ? any : written), "%s: tensors share memory that the call writes", what);
        any = std::max(any, x.to);
        if (x.written) written = std::max(written, x.to);
    }
    const std::vector<Group> groups = groups_of(p);
    const int64_t need = workspace_of(p, groups);
    MB_REQUIRE(((uintptr_t)p->workspace & 255) == 0, "%s: the workspace has to begin at a multiple of 256 bytes", what);
    if (s.empty()) return MB_OK;
    if (!p->workspace || p->workspace_bytes < need)
        return fail(MB_ERR_WORKSPACE, "%s: workspace of %lld bytes, %lld are needed", what, (long long)p->workspace_bytes, (long long)need);
    for (const Group& g : groups)
        if (const int rc = run(what, p, g, (hipStream_t)stream)) return rc;
    return MB_OK;
} catch (const std::bad_alloc&) {
    return fail(MB_ERR_INVALID_ARGUMENT, "mb_muon_run: no host memory");
}
