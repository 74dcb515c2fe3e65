// RMS norm of every query and key head with the position rotation in the same pass, forward
// and backward, on gfx950.
//
//   n = x rsqrt(mean(x^2) + eps),  y = w n,  (y_2i, y_2i+1) -> (y_2i c - y_2i+1 s, y_2i s + y_2i+1 c)
//   backward:  g = the inverse rotation of dy,  dx = r (w g - n mean(w g n)),  dw = sum_rows g n
//
// HBM-bound: x is read once and y written once (backward: x and dy read, dx written).  One
// wave takes a token: a lane holds 16 bytes of a head's row, hd * size / 16 lanes share a row
// and sum its squares over DPP/LDS-free shuffles, and the wave walks the token's H + Hk rows
// (queries, then keys) in steps of 64 / lanes rows.  A lane's channels are the same in every
// row, so the token's cosines and sines and the weights are loaded once for all its heads.
#include "common.h"

#include <algorithm>

namespace mb {
namespace {

constexpr int kQkThreads = 256;
constexpr int kQkWaves = kQkThreads / 64;
constexpr int kQkBwdBlocks = 1024;  // four workgroups per CU, each walking tokens

typedef __attribute__((__ext_vector_type__(8))) __bf16 bf16x8v;

// 16 bytes of a row as floats, and back with one rounding to nearest
template <typename T>
struct Row16;
template <>
struct Row16<float> {
    static constexpr int N = 4;
    static __device__ void load(const void* p, float* v) {
        const f32x4v q = *reinterpret_cast<const f32x4v*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = q[i];
    }
    static __device__ void store(void* p, const float* v) {
        const f32x4v q = {v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4v*>(p) = q;
    }
};
template <>
struct Row16<__bf16> {
    static constexpr int N = 8;
    static __device__ void load(const void* p, float* v) {
        const bf16x8v q = *reinterpret_cast<const bf16x8v*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)q[i];
    }
    static __device__ void store(void* p, const float* v) {
        bf16x8v q;
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = (__bf16)v[i];
        *reinterpret_cast<bf16x8v*>(p) = q;
    }
};

struct QkArgs {
    const void *q, *k, *dqo, *dko;            // inputs, and the output gradients (backward)
    int64_t q_sb, q_sl, q_sh, k_sb, k_sl, k_sh;
    int64_t dq_sb, dq_sl, dq_sh, dk_sb, dk_sl, dk_sh;
    const float *wq, *wk, *cos, *sin;
    const void* start;                         // [B] int32 / int64 or NULL
    int64_t start0, table_rows;
    int64_t tokens;
    int start_bytes, L, H, Hk;
    float eps;
    void *q_out, *k_out;                       // [B, L, H, hd], [B, L, Hk, hd]
    float* part;                               // backward: [blocks, 2, hd] partial dw
};

template <int LPR>
__device__ inline float row_sum(float v) {
#pragma unroll
    for (int o = LPR / 2; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// The cosines and sines of a lane's channel pairs at token (b, l).  A position outside the
// table gives NaN: nothing is read out of its bounds.
template <int N>
__device__ inline void load_angles(const QkArgs& a, int64_t b, int64_t l, int half, int chunk, float* c, float* s) {
    int64_t pos = a.start0 + l;
    if (a.start) pos = l + (a.start_bytes == 8 ? ((const int64_t*)a.start)[b] : (int64_t)((const int32_t*)a.start)[b]);
    const bool in = pos >= 0 && pos < a.table_rows;
    const int64_t at = (in ? pos : 0) * half + chunk * (N / 2);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        c[i] = in ? a.cos[at + i] : __builtin_nanf("");
        s[i] = in ? a.sin[at + i] : __builtin_nanf("");
    }
}

template <typename T, int HD>
__global__ void __launch_bounds__(kQkThreads) qk_norm_fwd_kernel(QkArgs a) {
    constexpr int N = Row16<T>::N;
    constexpr int LPR = HD / N;     // lanes of a row
    constexpr int RPW = 64 / LPR;   // rows of a wave's step
    const int lane = threadIdx.x & 63;
    const int chunk = lane % LPR;
    const int64_t t = (int64_t)blockIdx.x * kQkWaves + (threadIdx.x >> 6);
    if (t >= a.tokens) return;
    const int64_t b = t / a.L, l = t - b * a.L;
    float c[N / 2], s[N / 2], wq[N], wk[N];
    load_angles<N>(a, b, l, HD / 2, chunk, c, s);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        wq[i] = a.wq[chunk * N + i];
        wk[i] = a.wk[chunk * N + i];
    }
    const int rows = a.H + a.Hk;
    for (int r0 = 0; r0 < rows; r0 += RPW) {
        const int r = r0 + lane / LPR;
        const bool isq = r < a.H;
        if (r >= rows) continue;
        const T* x = isq ? (const T*)a.q + b * a.q_sb + l * a.q_sl + r * a.q_sh
                         : (const T*)a.k + b * a.k_sb + l * a.k_sl + (r - a.H) * a.k_sh;
        float v[N];
        Row16<T>::load(x + chunk * N, v);
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) ss = __builtin_fmaf(v[i], v[i], ss);
        const float rs = rsqrtf(row_sum<LPR>(ss) * (1.0f / HD) + a.eps);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (isq ? wq[i] : wk[i]) * (v[i] * rs);
        float y[N];
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            y[i] = v[i] * c[i / 2] - v[i + 1] * s[i / 2];
            y[i + 1] = v[i] * s[i / 2] + v[i + 1] * c[i / 2];
        }
        T* o = isq ? (T*)a.q_out + (t * a.H + r) * HD : (T*)a.k_out + (t * a.Hk + (r - a.H)) * HD;
        Row16<T>::store(o + chunk * N, y);
    }
}

// The norm's statistics are taken again from x, which the backward reads anyway.  dw: every
// lane sums its channels over its rows in registers, the workgroup's lanes of one channel are
// added in a fixed order into a row of `part`, and qk_norm_dw_kernel adds the rows in order.
template <typename T, int HD>
__global__ void __launch_bounds__(kQkThreads) qk_norm_bwd_kernel(QkArgs a) {
    constexpr int N = Row16<T>::N;
    constexpr int LPR = HD / N;
    constexpr int RPW = 64 / LPR;
    __shared__ float sums[kQkWaves][2][HD];
    const int lane = threadIdx.x & 63;
    const int wave = threadIdx.x >> 6;
    const int chunk = lane % LPR;
    const int rows = a.H + a.Hk;
    float wq[N], wk[N], accq[N], acck[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        wq[i] = a.wq[chunk * N + i];
        wk[i] = a.wk[chunk * N + i];
        accq[i] = acck[i] = 0.f;
    }
    for (int64_t t = (int64_t)blockIdx.x * kQkWaves + wave; t < a.tokens; t += (int64_t)gridDim.x * kQkWaves) {
        const int64_t b = t / a.L, l = t - b * a.L;
        float c[N / 2], s[N / 2];
        load_angles<N>(a, b, l, HD / 2, chunk, c, s);
        for (int r0 = 0; r0 < rows; r0 += RPW) {
            const int r = r0 + lane / LPR;
            const bool isq = r < a.H;
            if (r >= rows) continue;
            const int rk = r - a.H;
            const T* x = isq ? (const T*)a.q + b * a.q_sb + l * a.q_sl + r * a.q_sh
                             : (const T*)a.k + b * a.k_sb + l * a.k_sl + rk * a.k_sh;
            const T* dy = isq ? (const T*)a.dqo + b * a.dq_sb + l * a.dq_sl + r * a.dq_sh
                              : (const T*)a.dko + b * a.dk_sb + l * a.dk_sl + rk * a.dk_sh;
            float v[N], g[N];
            Row16<T>::load(x + chunk * N, v);
            Row16<T>::load(dy + chunk * N, g);
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i) ss = __builtin_fmaf(v[i], v[i], ss);
            const float rs = rsqrtf(row_sum<LPR>(ss) * (1.0f / HD) + a.eps);
            float dot = 0.f;
#pragma unroll
            for (int i = 0; i < N; i += 2) {
                const float g0 = g[i] * c[i / 2] + g[i + 1] * s[i / 2];
                const float g1 = g[i + 1] * c[i / 2] - g[i] * s[i / 2];
                g[i] = g0;
                g[i + 1] = g1;
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                v[i] *= rs;
                const float gn = g[i] * v[i];
                accq[i] += isq ? gn : 0.f;
                acck[i] += isq ? 0.f : gn;
                g[i] *= isq ? wq[i] : wk[i];
                dot = __builtin_fmaf(g[i], v[i], dot);
            }
            dot = row_sum<LPR>(dot) * (1.0f / HD);
#pragma unroll
            for (int i = 0; i < N; ++i) g[i] = rs * (g[i] - v[i] * dot);
            T* o = isq ? (T*)a.q_out + (t * a.H + r) * HD : (T*)a.k_out + (t * a.Hk + rk) * HD;
            Row16<T>::store(o + chunk * N, g);
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
        for (int o = LPR; o < 64; o <<= 1) {
            accq[i] += __shfl_xor(accq[i], o, 64);
            acck[i] += __shfl_xor(acck[i], o, 64);
        }
        if (lane < LPR) {
            sums[wave][0][chunk * N + i] = accq[i];
            sums[wave][1][chunk * N + i] = acck[i];
        }
    }
    __syncthreads();
    for (int d = threadIdx.x; d < 2 * HD; d += kQkThreads) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kQkWaves; ++w) v += sums[w][d / HD][d % HD];
        a.part[(int64_t)blockIdx.x * 2 * HD + d] = v;
    }
}

// Columns of part [n, 2 hd], summed in a fixed order: 8 columns and 128 strips a workgroup, eight
// loads of a strip on their way together (16 strips of 64 loads one after another: 20 us at 1024
// rows; this way 5).
constexpr int kDwCols = 8, kDwStrips = 128;
__global__ void __launch_bounds__(kDwCols * kDwStrips) qk_norm_dw_kernel(const float* __restrict__ part, int n, int hd,
                                                                        float* __restrict__ dwq, float* __restrict__ dwk) {
    __shared__ float sums[kDwStrips][kDwCols];
    const int col = threadIdx.x % kDwCols, strip = threadIdx.x / kDwCols;
    const int d = blockIdx.x * kDwCols + col;
    float v = 0.f;
    for (int r0 = strip; r0 < n; r0 += 8 * kDwStrips) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = r0 + i * kDwStrips < n ? part[(int64_t)(r0 + i * kDwStrips) * 2 * hd + d] : 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) v += x[i];
    }
    sums[strip][col] = v;
#pragma unroll
    for (int half = kDwStrips / 2; half >= 1; half >>= 1) {
        __syncthreads();
        if (strip < half) sums[strip][col] = v = v + sums[strip + half][col];
    }
    if (strip == 0) (d < hd ? dwq : dwk)[d % hd] = v;
}

int64_t bwd_blocks(int64_t tokens) {
    return std::min<int64_t>((tokens + kQkWaves - 1) / kQkWaves, kQkBwdBlocks);
}

bool aligned16(const void* p, int64_t a, int64_t b, int64_t c, int size) {
    return (((uintptr_t)p | (uint64_t)(a * size) | (uint64_t)(b * size) | (uint64_t)(c * size)) & 15) == 0;
}

// The checks that both directions share; 0 or an error code.
int check(const char* what, const QkArgs& a, int B, int hd, int dtype) {
    MB_REQUIRE(B >= 0 && a.L >= 0 && a.H >= 1 && a.Hk >= 1, "%s: B=%d L=%d H=%d Hk=%d", what, B, a.L, a.H, a.Hk);
    if (hd != 32 && hd != 64 && hd != 128)
        return fail(MB_ERR_UNSUPPORTED, "%s: head_dim=%d (supported: 32, 64, 128)", what, hd);
    MB_REQUIRE(dtype == MB_DTYPE_F32 || dtype == MB_DTYPE_BF16, "%s: dtype=%d", what, dtype);
    MB_REQUIRE(!a.start || a.start_bytes == 4 || a.start_bytes == 8, "%s: start_bytes=%d (4 or 8)", what, a.start_bytes);
    MB_REQUIRE(a.table_rows >= 0, "%s: table_rows=%lld", what, (long long)a.table_rows);
    if (!a.start)
        MB_REQUIRE(a.start0 >= 0 && a.start0 <= a.table_rows - a.L, "%s: positions %lld to %lld pass the table's %lld rows",
                   what, (long long)a.start0, (long long)a.start0 + a.L, (long long)a.table_rows);
    if (a.tokens == 0) return MB_OK;
    MB_REQUIRE(a.q && a.k && a.wq && a.wk && a.cos && a.sin && a.q_out && a.k_out, "%s: null pointer argument", what);
    const int size = dtype == MB_DTYPE_F32 ? 4 : 2;
    MB_REQUIRE(aligned16(a.q, a.q_sb, a.q_sl, a.q_sh, size) && aligned16(a.k, a.k_sb, a.k_sl, a.k_sh, size)
                   && aligned16(a.q_out, 0, 0, 0, size) && aligned16(a.k_out, 0, 0, 0, size),
               "%s: rows must begin at multiples of 16 bytes", what);
    return MB_OK;
}

template <typename T>
void launch_fwd(int hd, dim3 grid, hipStream_t st, const QkArgs& a) {
    const dim3 blk(kQkThreads);
    if (hd == 32) hipLaunchKernelGGL((qk_norm_fwd_kernel<T, 32>), grid, blk, 0, st, a);
    else if (hd == 64) hipLaunchKernelGGL((qk_norm_fwd_kernel<T, 64>), grid, blk, 0, st, a);
    else hipLaunchKernelGGL((qk_norm_fwd_kernel<T, 128>), grid, blk, 0, st, a);
}

template <typename T>
void launch_bwd(int hd, dim3 grid, hipStream_t st, const QkArgs& a) {
    const dim3 blk(kQkThreads);
    if (hd == 32) hipLaunchKernelGGL((qk_norm_bwd_kernel<T, 32>), grid, blk, 0, st, a);
    else if (hd == 64) hipLaunchKernelGGL((qk_norm_bwd_kernel<T, 64>), grid, blk, 0, st, a);
    else hipLaunchKernelGGL((qk_norm_bwd_kernel<T, 128>), grid, blk, 0, st, a);
}

}  // namespace
}  // namespace mb

using namespace mb;

extern "C" int mb_qk_norm_rotary_fwd(const void* q, int64_t q_sb, int64_t q_sl, int64_t q_sh, const void* k,
                                     int64_t k_sb, int64_t k_sl, int64_t k_sh, const float* wq, const float* wk,
                                     const float* cos, const float* sin, int64_t table_rows, const void* start,
                                     int start_bytes, int64_t start0, int B, int L, int H, int Hk, int hd, float eps,
                                     int dtype, void* q_out, void* k_out, void* stream) {
    QkArgs a = {};
    a.q = q, a.q_sb = q_sb, a.q_sl = q_sl, a.q_sh = q_sh;
    a.k = k, a.k_sb = k_sb, a.k_sl = k_sl, a.k_sh = k_sh;
    a.wq = wq, a.wk = wk, a.cos = cos, a.sin = sin, a.table_rows = table_rows;
    a.start = start, a.start_bytes = start_bytes, a.start0 = start0;
    a.tokens = (int64_t)B * L, a.L = L, a.H = H, a.Hk = Hk, a.eps = eps, a.q_out = q_out, a.k_out = k_out;
    if (const int rc = check("mb_qk_norm_rotary_fwd", a, B, hd, dtype)) return rc;
    if (a.tokens == 0) return MB_OK;
    const int64_t blocks = (a.tokens + kQkWaves - 1) / kQkWaves;
    MB_REQUIRE(blocks <= 0x7fffffff, "mb_qk_norm_rotary_fwd: %lld tokens are too many", (long long)a.tokens);
    if (dtype == MB_DTYPE_F32) launch_fwd<float>(hd, dim3((unsigned)blocks), (hipStream_t)stream, a);
    else launch_fwd<__bf16>(hd, dim3((unsigned)blocks), (hipStream_t)stream, a);
    return check_launch("mb_qk_norm_rotary_fwd");
}

extern "C" int64_t mb_qk_norm_rotary_bwd_workspace(int B, int L, int hd) {
    if (B < 1 || L < 1 || hd < 1) return 0;
    return bwd_blocks((int64_t)B * L) * 2 * hd * (int64_t)sizeof(float);
}

extern "C" int mb_qk_norm_rotary_bwd(const void* q, int64_t q_sb, int64_t q_sl, int64_t q_sh, const void* k,
                                     int64_t k_sb, int64_t k_sl, int64_t k_sh, const void* dq_out, int64_t dq_sb,
                                     int64_t dq_sl, int64_t dq_sh, const void* dk_out, int64_t dk_sb, int64_t dk_sl,
                                     int64_t dk_sh, const float* wq, const float* wk, const float* cos,
                                     const float* sin, int64_t table_rows, const void* start, int start_bytes,
                                     int64_t start0, int B, int L, int H, int Hk, int hd, float eps, int dtype,
                                     void* dq, void* dk, float* dwq, float* dwk, void* workspace,
                                     int64_t workspace_bytes, void* stream) {
    QkArgs a = {};
    a.q = q, a.q_sb = q_sb, a.q_sl = q_sl, a.q_sh = q_sh;
    a.k = k, a.k_sb = k_sb, a.k_sl = k_sl, a.k_sh = k_sh;
    a.dqo = dq_out, a.dq_sb = dq_sb, a.dq_sl = dq_sl, a.dq_sh = dq_sh;
    a.dko = dk_out, a.dk_sb = dk_sb, a.dk_sl = dk_sl, a.dk_sh = dk_sh;
    a.wq = wq, a.wk = wk, a.cos = cos, a.sin = sin, a.table_rows = table_rows;
    a.start = start, a.start_bytes = start_bytes, a.start0 = start0;
    a.tokens = (int64_t)B * L, a.L = L, a.H = H, a.Hk = Hk, a.eps = eps, a.q_out = dq, a.k_out = dk;
    a.part = (float*)workspace;
    if (const int rc = check("mb_qk_norm_rotary_bwd", a, B, hd, dtype)) return rc;
    MB_REQUIRE(dwq && dwk, "mb_qk_norm_rotary_bwd: null pointer argument");
    hipStream_t st = (hipStream_t)stream;
    const int64_t blocks = bwd_blocks(a.tokens);
    if (a.tokens > 0) {
        const int size = dtype == MB_DTYPE_F32 ? 4 : 2;
        MB_REQUIRE(dq_out && dk_out, "mb_qk_norm_rotary_bwd: null pointer argument");
        MB_REQUIRE(aligned16(dq_out, dq_sb, dq_sl, dq_sh, size) && aligned16(dk_out, dk_sb, dk_sl, dk_sh, size),
                   "mb_qk_norm_rotary_bwd: rows must begin at multiples of 16 bytes");
        if (!workspace || workspace_bytes < mb_qk_norm_rotary_bwd_workspace(B, L, hd))
            return fail(MB_ERR_WORKSPACE, "mb_qk_norm_rotary_bwd: workspace of %lld bytes, %lld are needed",
                        (long long)workspace_bytes, (long long)mb_qk_norm_rotary_bwd_workspace(B, L, hd));
        if (dtype == MB_DTYPE_F32) launch_bwd<float>(hd, dim3((unsigned)blocks), st, a);
        else launch_bwd<__bf16>(hd, dim3((unsigned)blocks), st, a);
    }
    hipLaunchKernelGGL(qk_norm_dw_kernel, dim3(2 * hd / kDwCols), dim3(kDwCols * kDwStrips), 0, st, a.part, (int)blocks, hd, dwq, dwk);
    return check_launch("mb_qk_norm_rotary_bwd");
}
