// Rotary positions: the first `turned` channels of every query and key head, in pairs, turned by the
// angles of the row's position, the others copied, on gfx950.
//
//   y[a] = x[a] c - x[b] s,   y[b] = x[a] s + x[b] c,   c, s = cos, sin[position, i]
//   pair i is (a, b) = (2i, 2i + 1) (interleaved) or (i, i + turned / 2) (half); the gradient is the
//   same with -s.
//
// HBM-bound: q and k are read once and written once, in one launch.  A thread takes 16 bytes of a
// head's row (half: 16 bytes of each half); the tables' rows, shared by the heads of a token and by the
// batch, come out of the caches.  Products and sums are rounded one by one (no fused multiply-add), as
// elementwise tensor operations round them.  A direction, replayed on the same tensors (which the last-level
// cache partly holds): 56 x 512 tokens, 8 + 8 heads of 64 in bf16 20.8 us, 5.6 TB/s; 2 x 16384, 8 + 2 heads of 128
// 28.9 us, 5.8 TB/s.  16 tokens: 3.1 us, a launch.
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
    int L, H, Hk, hd, turned, turn_jobs, jobs;
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
// other).
template <typename T, int N, bool HALF>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const RotArgs a) {
    constexpr int W = HALF ? N : (N < 2 ? 2 : N);   // channels of a turning piece
    constexpr int P = HALF ? W : W / 2;             // its pairs
    const unsigned id = blockIdx.x * kRotThreads + threadIdx.x, heads = (unsigned)(a.H + a.Hk);
    const unsigned rest = id / (unsigned)a.jobs, job = id - rest * (unsigned)a.jobs;
    const unsigned at = rest / heads;
    const int h = (int)(rest - at * heads);
    if (at >= a.tokens) return;
    const int64_t token = a.t0 + at;
    const int64_t b = token / a.L;
    const int l = (int)(token - b * a.L);
    const T* from = h < a.H ? (const T*)a.q + b * a.q_sb + l * a.q_sl + h * a.q_sh : (const T*)a.k + b * a.k_sb + l * a.k_sl + (h - a.H) * a.k_sh;
    T* to = h < a.H ? (T*)a.q_out + (token * a.H + h) * a.hd : (T*)a.k_out + (token * a.Hk + h - a.H) * a.hd;
    if (job >= (unsigned)a.turn_jobs) {
        const int c = a.turned + (int)(job - a.turn_jobs) * N;
        store_piece<T, N>(to + c, load_piece<T, N>(from + c));
        return;
    }
    const int c0 = (int)job * W, c1 = HALF ? c0 + a.turned / 2 : c0;
    Piece<T, W> x = load_piece<T, W>(from + c0), y;
    if constexpr (HALF) y = load_piece<T, W>(from + c1);
    int64_t pos;
    if (a.start) {
        const int64_t i = a.per_token ? token : b;
        pos = (a.start_bytes == 8 ? ((const int64_t*)a.start)[i] : (int64_t)((const int32_t*)a.start)[i]) + (a.per_token ? 0 : l);
    } else {
        pos = a.start0 + l;
    }
    float c[P], s[P];
    if (pos >= 0 && pos < a.table_rows) {   // asked once: asked at each pair, the tables come in single floats (29 -> 57 us below)
        const int64_t row = pos * (a.turned / 2) + (HALF ? c0 : c0 / 2);
#pragma unroll
        for (int e = 0; e < P; ++e) c[e] = a.cos[row + e], s[e] = a.sin[row + e] * a.sign;
    } else {   // outside the table: NaN, nothing is read out of its bounds
#pragma unroll
        for (int e = 0; e < P; ++e) c[e] = s[e] = __builtin_nanf("");
    }
#pragma unroll
    for (int e = 0; e < P; ++e) {
        if constexpr (HALF) turn(x.v[e], y.v[e], c[e], s[e]);
        else turn(x.v[2 * e], x.v[2 * e + 1], c[e], s[e]);
    }
    store_piece<T, W>(to + c0, x);
    if constexpr (HALF) store_piece<T, W>(to + c1, y);
}

template <typename T, int N, bool HALF>
void launch(RotArgs& a, int64_t tokens, hipStream_t st) {
    constexpr int W = HALF ? N : (N < 2 ? 2 : N);
    a.turn_jobs = a.turned / (HALF ? 2 : 1) / W;
    a.jobs = a.turn_jobs + (a.hd - a.turned) / N;
    const int64_t per = (int64_t)a.jobs * (a.H + a.Hk);
    const int64_t most = std::max<int64_t>(1, kRotMost / per);
    for (a.t0 = 0; a.t0 < tokens; a.t0 += most) {
        a.tokens = (unsigned)std::min(tokens - a.t0, most);
        const dim3 grid((unsigned)((a.tokens * per + kRotThreads - 1) / kRotThreads));
        hipLaunchKernelGGL((rotary_kernel<T, N, HALF>), grid, dim3(kRotThreads), 0, st, a);
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

// Of a strided input [B, L, H, hd].
Span input_span(const void* p, const int64_t* st, const int64_t* n, int64_t hd, int64_t size) {
    int64_t from = 0, to = hd;
    for (int i = 0; i < 3; ++i) (st[i] < 0 ? from : to) += st[i] * (n[i] - 1);
    return span(p ? (const char*)p + from * size : nullptr, (to - from) * size);
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
    const int size = p->dtype == MB_DTYPE_F32 ? 4 : 2, n = 16 / size;
    const int64_t q_n[3] = {p->B, p->L, p->H}, k_n[3] = {p->B, p->L, p->Hk}, table = p->table_rows * (p->turned / 2) * 4;
    const Span out[] = {span(p->q_out, tokens * p->H * p->hd * size), span(p->k_out, tokens * p->Hk * p->hd * size)};
    const Span in[] = {p->H ? input_span(p->q, p->q_st, q_n, p->hd, size) : Span{}, p->Hk ? input_span(p->k, p->k_st, k_n, p->hd, size) : Span{},
                       span(p->cos, table), span(p->sin, table), span(p->start, (p->start_per_token ? tokens : p->B) * p->start_bytes)};
    for (const Span& x : out)
        for (const Span& y : in) MB_REQUIRE(!touch(x, y), "%s: an output's memory is shared with an input", what);
    MB_REQUIRE(!touch(out[0], out[1]), "%s: the outputs share memory", what);
    RotArgs a = {};
    a.q = p->q, a.q_sb = p->q_st[0], a.q_sl = p->q_st[1], a.q_sh = p->q_st[2];
    a.k = p->k, a.k_sb = p->k_st[0], a.k_sl = p->k_st[1], a.k_sh = p->k_st[2];
    a.cos = p->cos, a.sin = p->sin, a.table_rows = p->table_rows;
    a.start = p->start, a.start0 = p->start0, a.start_bytes = (int)p->start_bytes, a.per_token = p->start_per_token != 0;
    a.L = (int)p->L, a.H = (int)p->H, a.Hk = (int)p->Hk, a.hd = (int)p->hd, a.turned = (int)p->turned;
    a.sign = p->inverse ? -1.f : 1.f;
    a.q_out = p->q_out, a.k_out = p->k_out;
    // 16 bytes a thread where rows and the parts of them allow it, single channels otherwise (56 x 512: 20.8 against 50 us, 2 x 16384:
    // 28.9 against 67; 6 x 1021 in fp32, 10 + 5 heads of 64 of which half turns: 9.1 against 18)
    const bool half = p->layout == 1;
    const bool pieces = p->hd % n == 0 && p->turned % (half ? 2 * n : n) == 0 && (p->H == 0 || rows16(p->q, p->q_st, size))
                        && (p->Hk == 0 || rows16(p->k, p->k_st, size)) && (((uintptr_t)p->q_out | (uintptr_t)p->k_out) & 15) == 0;
    if (p->dtype == MB_DTYPE_F32) dispatch<float>(a, half, pieces, tokens, (hipStream_t)stream);
    else dispatch<__bf16>(a, half, pieces, tokens, (hipStream_t)stream);
    return check_launch(what);
}
