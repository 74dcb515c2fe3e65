// Rotary positions: the first `turned` channels of every query and key head, in pairs, turned by the
// angles of the row's position, the others copied, on gfx950.
//
//   y[a] = x[a] c - x[b] s,   y[b] = x[a] s + x[b] c,   c, s = cos, sin[position, i]
//   pair i is (a, b) = (2i, 2i + 1) (interleaved) or (i, i + turned / 2) (half); the gradient is the
//   same with -s.
//
// HBM-bound: q and k are read once and written once, in one launch.  A thread holds 16 bytes of a
// head's row (half: 16 bytes of each half), with the cosines and sines of its channels in registers
// for several heads of the token: the tables are read once for them.  Products and sums are rounded
// one by one (no fused multiply-add), as elementwise tensor operations round them.
#include "common.h"

#include <algorithm>

namespace mb {
namespace {

constexpr int kRotThreads = 256;
constexpr int64_t kRotMost = (int64_t)1 << 31;   // threads of a launch (counted in 32 bits)

struct RotArgs {
    const void *q, *k;
    int64_t q_sb, q_sl, q_sh, k_sb, k_sl, k_sh;
    const float *cos, *sin;
    int64_t table_rows;
    const void* start;
    int64_t start0, t0;          // t0: the launch's first token
    unsigned tokens;             // of the launch
    int start_bytes, per_token;
    int L, H, Hk, hd, turned, groups, turn_jobs, jobs;
    float sign;
    void *q_out, *k_out;
};

template <typename T, int N>
struct Piece {
    T v[N];
};
template <typename T, int N>
__device__ inline Piece<T, N> load_piece(const T* p) {
    Piece<T, N> x;
    if constexpr (N * sizeof(T) == 16) {
        typedef T vec __attribute__((ext_vector_type(N)));
        const vec q = *reinterpret_cast<const vec*>(p);
#pragma unroll
        for (int i = 0; i < N; ++i) x.v[i] = q[i];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x.v[i] = p[i];
    }
    return x;
}
template <typename T, int N>
__device__ inline void store_piece(T* p, const Piece<T, N>& x) {
    if constexpr (N * sizeof(T) == 16) {
        typedef T vec __attribute__((ext_vector_type(N)));
        vec q;
#pragma unroll
        for (int i = 0; i < N; ++i) q[i] = x.v[i];
        *reinterpret_cast<vec*>(p) = q;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = x.v[i];
    }
}

// One pair, every product and sum rounded by itself.
template <typename T>
__device__ inline void turn(T& xa, T& xb, float c, float s) {
#pragma clang fp contract(off)
    const float a = (float)xa, b = (float)xb;
    const float ac = a * c, bs = b * s, as = a * s, bc = b * c;
    xa = (T)(ac - bs);
    xb = (T)(as + bc);
}

// N: channels of a piece (16 bytes, or single channels, with pairs of them where they are next to each
// other).  PER: heads in flight at once.
template <typename T, int N, bool HALF, int PER>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const RotArgs a) {
    constexpr int W = HALF ? N : (N < 2 ? 2 : N);   // channels of a turning piece
    constexpr int P = HALF ? W : W / 2;             // its pairs
    const unsigned id = blockIdx.x * kRotThreads + threadIdx.x;
    const unsigned rest = id / (unsigned)a.jobs, job = id - rest * (unsigned)a.jobs;
    const unsigned at = rest / (unsigned)a.groups, group = rest - at * (unsigned)a.groups;
    if (at >= a.tokens) return;
    const int64_t token = a.t0 + at;
    const int64_t b = token / a.L;
    const int l = (int)(token - b * a.L);
    const int heads = a.H + a.Hk;
    const T* qrow = (const T*)a.q + b * a.q_sb + l * a.q_sl;
    const T* krow = (const T*)a.k + b * a.k_sb + l * a.k_sl;
    T* qto = (T*)a.q_out + token * a.H * a.hd;
    T* kto = (T*)a.k_out + token * a.Hk * a.hd;
    const bool turns = job < (unsigned)a.turn_jobs;
    const int c0 = turns ? (int)job * W : a.turned + (int)(job - a.turn_jobs) * N;
    const int c1 = HALF ? c0 + a.turned / 2 : c0;
    float c[P], s[P];
    if (turns) {
        int64_t pos;
        if (a.start) {
            const int64_t i = a.per_token ? token : b;
            pos = (a.start_bytes == 8 ? ((const int64_t*)a.start)[i] : (int64_t)((const int32_t*)a.start)[i]) + (a.per_token ? 0 : l);
        } else {
            pos = a.start0 + l;
        }
        if (pos >= 0 && pos < a.table_rows) {
            const int64_t from = pos * (a.turned / 2) + (HALF ? c0 : c0 / 2);
#pragma unroll
            for (int i = 0; i < P; ++i) c[i] = a.cos[from + i], s[i] = a.sin[from + i] * a.sign;
        } else {   // outside the table: NaN, nothing is read out of its bounds
#pragma unroll
            for (int i = 0; i < P; ++i) c[i] = s[i] = __builtin_nanf("");
        }
    }
    for (int h0 = (int)group; h0 < heads; h0 += PER * a.groups) {
        const T* from[PER];
        T* to[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int h = h0 + i * a.groups;
            from[i] = h < a.H ? qrow + h * a.q_sh : krow + (h - a.H) * a.k_sh;
            to[i] = h < a.H ? qto + (int64_t)h * a.hd : kto + (int64_t)(h - a.H) * a.hd;
        }
        if (turns) {
            Piece<T, W> x[PER], y[PER];
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (h0 + i * a.groups < heads) {
                    x[i] = load_piece<T, W>(from[i] + c0);
                    if constexpr (HALF) y[i] = load_piece<T, W>(from[i] + c1);
                }
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (h0 + i * a.groups < heads) {
#pragma unroll
                    for (int e = 0; e < P; ++e) {
                        if constexpr (HALF) turn(x[i].v[e], y[i].v[e], c[e], s[e]);
                        else turn(x[i].v[2 * e], x[i].v[2 * e + 1], c[e], s[e]);
                    }
                    store_piece<T, W>(to[i] + c0, x[i]);
                    if constexpr (HALF) store_piece<T, W>(to[i] + c1, y[i]);
                }
        } else {
            Piece<T, N> x[PER];
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (h0 + i * a.groups < heads) x[i] = load_piece<T, N>(from[i] + c0);
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (h0 + i * a.groups < heads) store_piece<T, N>(to[i] + c0, x[i]);
        }
    }
}

template <typename T, int N, bool HALF>
void launch(RotArgs& a, int64_t tokens, hipStream_t st) {
    constexpr int W = HALF ? N : (N < 2 ? 2 : N);
    a.turn_jobs = a.turned / (HALF ? 2 : 1) / W;
    a.jobs = a.turn_jobs + (a.hd - a.turned) / N;
    const int heads = a.H + a.Hk;
    a.groups = heads;
    const int64_t per = (int64_t)a.jobs * a.groups;
    const int64_t most = std::max<int64_t>(1, kRotMost / per);
    for (a.t0 = 0; a.t0 < tokens; a.t0 += most) {
        a.tokens = (unsigned)std::min(tokens - a.t0, most);
        const dim3 grid((unsigned)((a.tokens * per + kRotThreads - 1) / kRotThreads));
        hipLaunchKernelGGL((rotary_kernel<T, N, HALF, 1>), grid, dim3(kRotThreads), 0, st, a);
    }
}

template <typename T>
void dispatch(RotArgs& a, bool half, bool pieces, int64_t tokens, hipStream_t st) {
    constexpr int N = 16 / sizeof(T);
    if (pieces) {
        if (half) launch<T, N, true>(a, tokens, st);
        else launch<T, N, false>(a, tokens, st);
    } else {
        if (half) launch<T, 1, true>(a, tokens, st);
        else launch<T, 1, false>(a, tokens, st);
    }
}

bool rows16(const void* p, const int64_t* st, int size) {
    return (((uintptr_t)p | (uint64_t)(st[0] * size) | (uint64_t)(st[1] * size) | (uint64_t)(st[2] * size)) & 15) == 0;
}

}  // namespace
}  // namespace mb

using namespace mb;

extern "C" int mb_apply_rotary(const mb_rotary* p, void* stream) {
    const char* what = "mb_apply_rotary";
    MB_REQUIRE(p, "%s: null args", what);
    const int64_t top = 0x7fffffff;
    MB_REQUIRE(p->B >= 0 && p->B <= top && p->L >= 0 && p->L <= top && p->H >= 0 && p->H <= 0xffff && p->Hk >= 0 && p->Hk <= 0xffff
                   && p->H + p->Hk >= 1, "%s: B=%lld L=%lld H=%lld Hk=%lld", what, (long long)p->B, (long long)p->L,
               (long long)p->H, (long long)p->Hk);
    MB_REQUIRE(p->hd >= 1 && p->hd <= 8192, "%s: head_dim=%lld (1 to 8192)", what, (long long)p->hd);
    MB_REQUIRE(p->turned >= 0 && p->turned <= p->hd && p->turned % 2 == 0, "%s: %lld of %lld channels turned (an even number of them)",
               what, (long long)p->turned, (long long)p->hd);
    MB_REQUIRE(p->layout == 0 || p->layout == 1, "%s: layout=%lld", what, (long long)p->layout);
    MB_REQUIRE(p->dtype == MB_DTYPE_F32 || p->dtype == MB_DTYPE_BF16, "%s: dtype=%lld", what, (long long)p->dtype);
    MB_REQUIRE(!p->start || p->start_bytes == 4 || p->start_bytes == 8, "%s: start_bytes=%lld (4 or 8)", what, (long long)p->start_bytes);
    MB_REQUIRE(p->table_rows >= 0, "%s: table_rows=%lld", what, (long long)p->table_rows);
    if (!p->start)
        MB_REQUIRE(p->start0 >= 0 && p->start0 <= p->table_rows - p->L, "%s: positions %lld to %lld pass the table's %lld rows",
                   what, (long long)p->start0, (long long)(p->start0 + p->L), (long long)p->table_rows);
    const int64_t tokens = p->B * p->L;
    if (tokens == 0) return MB_OK;
    MB_REQUIRE((p->H == 0 || (p->q && p->q_out)) && (p->Hk == 0 || (p->k && p->k_out)) && (p->turned == 0 || (p->cos && p->sin)),
               "%s: null pointer argument", what);
    RotArgs a = {};
    a.q = p->q, a.q_sb = p->q_st[0], a.q_sl = p->q_st[1], a.q_sh = p->q_st[2];
    a.k = p->k, a.k_sb = p->k_st[0], a.k_sl = p->k_st[1], a.k_sh = p->k_st[2];
    a.cos = p->cos, a.sin = p->sin, a.table_rows = p->table_rows;
    a.start = p->start, a.start0 = p->start0, a.start_bytes = (int)p->start_bytes, a.per_token = p->start_per_token != 0;
    a.L = (int)p->L, a.H = (int)p->H, a.Hk = (int)p->Hk, a.hd = (int)p->hd, a.turned = (int)p->turned;
    a.sign = p->inverse ? -1.f : 1.f;
    a.q_out = p->q_out, a.k_out = p->k_out;
    // 16 bytes a thread where rows and the parts of them allow it, single channels otherwise
    const int size = p->dtype == MB_DTYPE_F32 ? 4 : 2, n = 16 / size;
    const bool half = p->layout == 1;
    const bool pieces = p->hd % n == 0 && p->turned % (half ? 2 * n : n) == 0 && (p->H == 0 || rows16(p->q, p->q_st, size))
                        && (p->Hk == 0 || rows16(p->k, p->k_st, size)) && (((uintptr_t)p->q_out | (uintptr_t)p->k_out) & 15) == 0;
    if (p->dtype == MB_DTYPE_F32) dispatch<float>(a, half, pieces, tokens, (hipStream_t)stream);
    else dispatch<__bf16>(a, half, pieces, tokens, (hipStream_t)stream);
    return check_launch(what);
}
