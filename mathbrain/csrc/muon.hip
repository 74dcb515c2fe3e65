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
struct By {
    typedef Product<_Float16, 2, TILE, TILE, kRows, kRows> Gram;
    typedef Product<_Float16, 2, TILE, TILE, kCols, kRows> Apply;
    static_assert(Gram::kThreads == kThreads && Apply::kThreads == kThreads, "");
    static_assert(2 * Gram::kOutPlane <= Gram::kLds && Apply::kOut32 <= Apply::kLds, "results go out through LDS");
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

// Fewer tiles of 128 than this in a launch leave most of the card idle: tiles of 64 then.
constexpr int64_t kFewTiles = 300;

struct Args {
    const Mat* mats;
    const int* first;            // [kFirsts][count]
    int count;
    int from, to;                // X's buffers
    float a, b, c;               // X <- X (a + b A + c A^2)
    float x_scale, a_scale, b_scale;
    double eps;
    float lr, mu, keep;          // keep = 1 - lr decay
    int nesterov, is_step, last;
};

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

// Sums of squares in 64 bits; a step's momentum and G first.
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

// POLY: B = a + b A + c A^2 from A's planes; otherwise A = X X^T.
template <bool POLY, int TILE>
__global__ void __launch_bounds__(kThreads, By<TILE>::Gram::kWaves) muon_pair_kernel(const Args a) {
    typedef typename By<TILE>::Gram Gram;
    extern __shared__ char smem[];
    int id = blockIdx.x;
    const Mat m = find(a, TILE == 64 ? kFirstPair64 : kFirstPair, id);
    int q = (int)((sqrtf(8.f * id + 1.f) - 1.f) * 0.5f);   // id = q (q + 1) / 2 + p, p <= q
    while (q * (q + 1) / 2 > id) --q;
    while ((q + 1) * (q + 2) / 2 <= id) ++q;
    q = uniform(q);
    const int p = id - q * (q + 1) / 2, p0 = p * TILE, q0 = q * TILE;
    const int64_t plane = (int64_t)m.mp * m.mp;
    const Side side = POLY ? Side{m.a, plane * 2, m.mp, m.mp} : Side{m.x[a.from], (int64_t)m.mp * m.np * 2, m.np, m.mp};
    Gram g;
    g.run(side, side, p0, q0, 0, POLY ? m.mp : m.np, smem);
    __syncthreads();
    if (POLY) {
#pragma unroll
        for (int h = 0; h < 2; ++h) Gram::fetch(smem, h, m.a + h * plane, m.mp, p0, q0, m.mp, m.mp);
        __syncthreads();
    }
    _Float16* out = POLY ? m.b : m.a;
    const float from = POLY ? a.a_scale : a.x_scale, to = POLY ? a.b_scale : a.a_scale;
    const float f = (POLY ? a.c : 1.f) * to / from / from, fb = a.b * to / a.a_scale, one = a.a * to;
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
                    if (POLY) {
                        v[e] += fb * ((float)hi[e] + (float)lo[e]);
                        if (p0 + Gram::row(i, r) + e == q0 + Gram::col(j)) v[e] += one;
                    }
                }
                split4(v, hi, lo);
            }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        Gram::store(smem, h, out + h * plane, m.mp, p0, q0, m.mp, m.mp);
        if (p != q) Gram::store_turned(smem, h, out + h * plane, m.mp, p0, q0, m.mp, m.mp);
    }
}

template <int TILE>
__global__ void __launch_bounds__(kThreads, By<TILE>::Apply::kWaves) muon_apply_kernel(const Args a) {
    typedef typename By<TILE>::Apply Apply;
    extern __shared__ char smem[];
    int id = blockIdx.x;
    const Mat m = find(a, TILE == 64 ? kFirstTile64 : kFirstTile, id);
    const int across = (m.np + TILE - 1) / TILE;
    const int p0 = id % across * TILE, q0 = id / across * TILE;
    const int64_t plane = (int64_t)m.mp * m.np;
    Apply g;
    g.run(Side{m.x[a.from], plane * 2, m.np, m.np}, Side{m.b, (int64_t)m.mp * m.mp * 2, m.mp, m.mp}, p0, q0, 0, m.mp, smem);
    const float f = (a.last ? 1.f / a.x_scale : 1.f) / a.b_scale;
    __syncthreads();
    if (!a.last) {
#pragma unroll
        for (int j = 0; j < Apply::FQ; ++j)
#pragma unroll
            for (int i = 0; i < Apply::FP; ++i)
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const float v[4] = {g.acc[i][j][r] * f, g.acc[i][j][r + 1] * f, g.acc[i][j][r + 2] * f, g.acc[i][j][r + 3] * f};
                    split4(v, Apply::held(smem, 0, i, j, r), Apply::held(smem, 1, i, j, r));
                }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < 2; ++h) Apply::store(smem, h, m.x[a.to] + h * plane, m.np, p0, q0, m.np, m.mp);
        return;
    }
#pragma unroll
    for (int j = 0; j < Apply::FQ; ++j)
#pragma unroll
        for (int i = 0; i < Apply::FP; ++i)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                Apply::held32(smem, i, j, r) = f32x4v{g.acc[i][j][r], g.acc[i][j][r + 1], g.acc[i][j][r + 2], g.acc[i][j][r + 3]} * f;
    __syncthreads();
    // lanes next to each other along the result's own rows
#pragma unroll 4
    for (int n = threadIdx.x; n < TILE * TILE; n += kThreads) {
        const int q = m.tall ? n % TILE : n / TILE, p = m.tall ? n / TILE : n % TILE;
        if (q0 + q >= m.m || p0 + p >= m.n) continue;
        const int64_t to = m.tall ? (int64_t)(p0 + p) * m.cols + q0 + q : (int64_t)(q0 + q) * m.cols + p0 + p;
        float y = Apply::out32(smem, q, p);
        if (a.is_step) y = load1(m.dst, to, m.dst_bf16) * a.keep - a.lr * m.rate * y;
        store1(m.dst, to, m.dst_bf16, y);
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
    int64_t bytes = 0;
};

int64_t lay_out(const mb_muon* p, char* base, Layout* out) {
    int64_t used = 0;
    auto take = [&](int64_t bytes) {
        char* at = base ? base + used : nullptr;
        used += pad(bytes, 256);
        return at;
    };
    // the longest products first: what is left at a launch's end is short
    std::vector<int64_t> order;
    for (int64_t i = 0; i < p->count; ++i)
        if (p->matrices[i].rows && p->matrices[i].cols) order.push_back(i);
    std::stable_sort(order.begin(), order.end(), [&](int64_t i, int64_t j) {
        const mb_muon_matrix &x = p->matrices[i], &y = p->matrices[j];
        return std::max(x.rows, x.cols) > std::max(y.rows, y.cols);
    });
    for (const int64_t i : order) {
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
    return used;
}

int64_t table_bytes(int64_t count) { return pad(count * (int64_t)sizeof(Mat), 256) + pad(count * (int64_t)sizeof(int) * kFirsts, 256); }

int run(const char* what, const mb_muon* p, hipStream_t st) {
    Layout l;
    const int64_t table = table_bytes(p->count);
    lay_out(p, (char*)p->workspace + table, &l);
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
    const bool small_pairs = l.blocks[kFirstPair] < kFewTiles, small_tiles = l.blocks[kFirstTile] < kFewTiles;
    for (int step = 0; step < p->steps; ++step) {
        a.from = step & 1, a.to = a.from ^ 1, a.last = step + 1 == p->steps;
        const auto pair = [&](auto tile, unsigned blocks) {
            constexpr int TILE = decltype(tile)::value;
            static Told told[2];
            constexpr int lds = By<TILE>::Gram::kLds;
            if (const int rc = allow_lds(what, (const void*)muon_pair_kernel<false, TILE>, lds, told[0])) return rc;
            if (const int rc = allow_lds(what, (const void*)muon_pair_kernel<true, TILE>, lds, told[1])) return rc;
            hipLaunchKernelGGL((muon_pair_kernel<false, TILE>), dim3(blocks), blk, lds, st, a);
            hipLaunchKernelGGL((muon_pair_kernel<true, TILE>), dim3(blocks), blk, lds, st, a);
            return MB_OK;
        };
        const auto apply = [&](auto tile, unsigned blocks) {
            constexpr int TILE = decltype(tile)::value;
            static Told told;
            constexpr int lds = By<TILE>::Apply::kLds;
            if (const int rc = allow_lds(what, (const void*)muon_apply_kernel<TILE>, lds, told)) return rc;
            hipLaunchKernelGGL((muon_apply_kernel<TILE>), dim3(blocks), blk, lds, st, a);
            return MB_OK;
        };
        typedef std::integral_constant<int, 64> T64;
        typedef std::integral_constant<int, 128> T128;
        int rc = small_pairs ? pair(T64(), (unsigned)l.blocks[kFirstPair64]) : pair(T128(), (unsigned)l.blocks[kFirstPair]);
        if (rc == MB_OK) rc = small_tiles ? apply(T64(), (unsigned)l.blocks[kFirstTile64]) : apply(T128(), (unsigned)l.blocks[kFirstTile]);
        if (rc != MB_OK) return rc;
    }
    return check_launch(what);
}

}  // namespace
}  // namespace mb

using namespace mb;

extern "C" int64_t mb_muon_workspace(const mb_muon* p) try {
    if (check("mb_muon_workspace", p)) return -1;
    return table_bytes(p->count) + lay_out(p, nullptr, nullptr);
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
    const int64_t need = table_bytes(p->count) + lay_out(p, nullptr, nullptr);
    MB_REQUIRE(((uintptr_t)p->workspace & 255) == 0, "%s: the workspace has to begin at a multiple of 256 bytes", what);
    if (s.empty()) return MB_OK;
    if (!p->workspace || p->workspace_bytes < need)
        return fail(MB_ERR_WORKSPACE, "%s: workspace of %lld bytes, %lld are needed", what, (long long)p->workspace_bytes, (long long)need);
    return run(what, p, (hipStream_t)stream);
} catch (const std::bad_alloc&) {
    return fail(MB_ERR_INVALID_ARGUMENT, "mb_muon_run: no host memory");
}
