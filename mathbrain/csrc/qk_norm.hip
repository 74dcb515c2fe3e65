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
constexpr int64_t kQkMost = 1 << 25;  // tokens of a forward launch, whose threads are counted in 32 bits

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
    int64_t t0, tokens;                        // the launch's first token (forward), the end
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
    const int64_t t = a.t0 + (int64_t)blockIdx.x * kQkWaves + (threadIdx.x >> 6);
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

bool aligned16(const void* p, const int64_t* st, int size) {
    return (((uintptr_t)p | (uint64_t)(st[0] * size) | (uint64_t)(st[1] * size) | (uint64_t)(st[2] * size)) & 15) == 0;
}

// Checks what both directions take and fills the kernels' arguments; 0 or an error code.
int fill(const char* what, const mb_qk_norm_rotary* p, QkArgs& a) {
    MB_REQUIRE(p, "%s: null args", what);
    const int64_t top = 0x7fffffff;
    MB_REQUIRE(p->B >= 0 && p->B <= top && p->L >= 0 && p->L <= top && p->H >= 1 && p->H <= top / 2 && p->Hk >= 1 && p->Hk <= top / 2,
               "%s: B=%lld L=%lld H=%lld Hk=%lld", what, (long long)p->B, (long long)p->L, (long long)p->H, (long long)p->Hk);
    if (p->hd != 32 && p->hd != 64 && p->hd != 128)
        return fail(MB_ERR_UNSUPPORTED, "%s: head_dim=%lld (supported: 32, 64, 128)", what, (long long)p->hd);
    MB_REQUIRE(p->dtype == MB_DTYPE_F32 || p->dtype == MB_DTYPE_BF16, "%s: dtype=%lld", what, (long long)p->dtype);
    MB_REQUIRE(!p->start || p->start_bytes == 4 || p->start_bytes == 8, "%s: start_bytes=%lld (4 or 8)", what, (long long)p->start_bytes);
    MB_REQUIRE(p->table_rows >= 0, "%s: table_rows=%lld", what, (long long)p->table_rows);
    if (!p->start)
        MB_REQUIRE(p->start0 >= 0 && p->start0 <= p->table_rows - p->L, "%s: positions %lld to %lld pass the table's %lld rows",
                   what, (long long)p->start0, (long long)(p->start0 + p->L), (long long)p->table_rows);
    a.tokens = p->B * p->L;
    if (a.tokens == 0) return MB_OK;
    MB_REQUIRE(p->q && p->k && p->wq && p->wk && p->cos && p->sin, "%s: null pointer argument", what);
    const int size = p->dtype == MB_DTYPE_F32 ? 4 : 2;
    MB_REQUIRE(aligned16(p->q, p->q_st, size) && aligned16(p->k, p->k_st, size), "%s: rows must begin at multiples of 16 bytes", what);
    a.q = p->q, a.q_sb = p->q_st[0], a.q_sl = p->q_st[1], a.q_sh = p->q_st[2];
    a.k = p->k, a.k_sb = p->k_st[0], a.k_sl = p->k_st[1], a.k_sh = p->k_st[2];
    a.wq = p->wq, a.wk = p->wk, a.cos = p->cos, a.sin = p->sin, a.table_rows = p->table_rows;
    a.start = p->start, a.start_bytes = (int)p->start_bytes, a.start0 = p->start0;
    a.L = (int)p->L, a.H = (int)p->H, a.Hk = (int)p->Hk, a.eps = (float)p->eps;
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

extern "C" int mb_qk_norm_rotary_fwd(const mb_qk_norm_rotary* p, void* stream) {
    QkArgs a = {};
    if (const int rc = fill("mb_qk_norm_rotary_fwd", p, a)) return rc;
    if (a.tokens == 0) return MB_OK;
    MB_REQUIRE(p->q_out && p->k_out, "mb_qk_norm_rotary_fwd: null pointer argument");
    MB_REQUIRE((((uintptr_t)p->q_out | (uintptr_t)p->k_out) & 15) == 0, "mb_qk_norm_rotary_fwd: rows must begin at multiples of 16 bytes");
    a.q_out = p->q_out, a.k_out = p->k_out;
    for (; a.t0 < a.tokens; a.t0 += kQkMost) {
        const dim3 grid((unsigned)((std::min(a.tokens - a.t0, kQkMost) + kQkWaves - 1) / kQkWaves));
        if (p->dtype == MB_DTYPE_F32) launch_fwd<float>((int)p->hd, grid, (hipStream_t)stream, a);
        else launch_fwd<__bf16>((int)p->hd, grid, (hipStream_t)stream, a);
    }
    return check_launch("mb_qk_norm_rotary_fwd");
}

extern "C" int64_t mb_qk_norm_rotary_bwd_workspace(int B, int L, int hd) {
    if (B < 1 || L < 1 || hd < 1) return 0;
    return bwd_blocks((int64_t)B * L) * 2 * hd * (int64_t)sizeof(float);
}

extern "C" int mb_qk_norm_rotary_bwd(const mb_qk_norm_rotary* p, void* stream) {
    QkArgs a = {};
    if (const int rc = fill("mb_qk_norm_rotary_bwd", p, a)) return rc;
    MB_REQUIRE(p->dwq && p->dwk, "mb_qk_norm_rotary_bwd: null pointer argument");
    hipStream_t st = (hipStream_t)stream;
    const int hd = (int)p->hd;
    const int64_t blocks = bwd_blocks(a.tokens);
    if (a.tokens > 0) {
        const int size = p->dtype == MB_DTYPE_F32 ? 4 : 2;
        MB_REQUIRE(p->dq_out && p->dk_out && p->dq && p->dk, "mb_qk_norm_rotary_bwd: null pointer argument");
        MB_REQUIRE(aligned16(p->dq_out, p->dq_st, size) && aligned16(p->dk_out, p->dk_st, size)
                       && (((uintptr_t)p->dq | (uintptr_t)p->dk) & 15) == 0,
                   "mb_qk_norm_rotary_bwd: rows must begin at multiples of 16 bytes");
        const int64_t need = mb_qk_norm_rotary_bwd_workspace((int)p->B, (int)p->L, hd);
        if (!p->workspace || p->workspace_bytes < need)
            return fail(MB_ERR_WORKSPACE, "mb_qk_norm_rotary_bwd: workspace of %lld bytes, %lld are needed",
                        (long long)p->workspace_bytes, (long long)need);
        a.dqo = p->dq_out, a.dq_sb = p->dq_st[0], a.dq_sl = p->dq_st[1], a.dq_sh = p->dq_st[2];
        a.dko = p->dk_out, a.dk_sb = p->dk_st[0], a.dk_sl = p->dk_st[1], a.dk_sh = p->dk_st[2];
        a.q_out = p->dq, a.k_out = p->dk, a.part = (float*)p->workspace;
        if (p->dtype == MB_DTYPE_F32) launch_bwd<float>(hd, dim3((unsigned)blocks), st, a);
        else launch_bwd<__bf16>(hd, dim3((unsigned)blocks), st, a);
    }
    hipLaunchKernelGGL(qk_norm_dw_kernel, dim3(2 * hd / kDwCols), dim3(kDwCols * kDwStrips), 0, st, a.part, (int)blocks, hd,
                       p->dwq, p->dwk);
    return check_launch("mb_qk_norm_rotary_bwd");
}
