// Forward of the attention with a learned bias by distance buckets.
#include "bias_attn_host.h"

#include <algorithm>

namespace mb {
namespace battn {
namespace {

// A workgroup takes 128 queries of one head, 32 to a wave, and walks the keys in tiles that all
// four waves read out of LDS; the next tile's rows are on their way from memory meanwhile.
// Running maximum, sum and output are in fp32; the probabilities are rounded to bf16 for the
// product with V where the inputs are bf16 (half a step of 2^-8 of each), the sum is not.
//
// SETS = 2: a second set of four waves takes every second tile for the same queries, and the two
// are joined through LDS in the end.  A workgroup's walk, which takes 1.2 us (heads of 128: 1.5) a
// tile with nothing beside it on the CU, is then half as long.
//
// In fp32 the walk may be split into o_parts runs, a workgroup each (o_parts_of), whose maxima, sums
// and outputs bias_attn_join_kernel joins through memory.
template <typename T, int HD, int SETS>
__global__ void __launch_bounds__(SETS * kThreads, (waves_per_simd<T, HD>())) bias_attn_fwd_kernel(const Args a) {
    using X = Ty<T>;
    using Tl = Tile<T, HD>;
    constexpr int KT = Tl::kN;
    constexpr int kStage = 2 * Tl::kBytes;            // a tile of K and one of V
    extern __shared__ __attribute__((aligned(16))) char smem[];
    float* tab = reinterpret_cast<float*>(smem + SETS * Tl::kStages * kStage);

    const int lane = threadIdx.x & 63, wave = wave_id() % 4, set = wave_id() / 4;
    int bh, qb;
    constexpr bool kRuns = sizeof(T) == 4 && SETS == 1;   // the walk may be split into runs
    const int parts = kRuns ? a.o_parts : 1;
    place(blockIdx.x, a.B * a.H, a.nq * parts, false, bh, qb);
    const int part = qb % parts;
    qb /= parts;
    const int b = bh / a.H, h = bh % a.H, hk = h / (a.H / a.Hk);
    const Reach reach(a);
    const int len = key_count(a, b), p0 = first_position(a, b);
    const int w0 = qb * kRows + wave * kWaveRows;   // the wave's first query
    const int i = w0 + (lane & 31), pos = p0 + i;
    const int last = min(a.Lq, (qb + 1) * kRows) - 1;
    const int kend = a.causal ? min(len, p0 + last + 1) : len;
    const int wend = w0 >= a.Lq ? 0 : a.causal ? min(len, p0 + min(a.Lq, w0 + kWaveRows)) : len;
    const int tiles = kend > 0 ? (kend + KT - 1) / KT : 0;
    // the workgroup's run of them (at most 2^24 tiles and 8 parts)
    const int t0 = (int)((uint32_t)(tiles * part) / (uint32_t)parts), t1 = (int)((uint32_t)(tiles * (part + 1)) / (uint32_t)parts);
    const float sl2 = a.scale * kLog2e;

    const T* kbase = (const T*)a.k + b * a.k_sb + hk * a.k_sh;
    const T* vbase = (const T*)a.v + b * a.v_sb + hk * a.v_sh;
    typename X::Frag qf[HD / 16];
    load_frags<T, HD>((const T*)a.q + b * a.q_sb + h * a.q_sh, a.q_sl, w0, a.Lq, qf);

    f32x16 o[HD / 32];
#pragma unroll
    for (int d = 0; d < HD / 32; ++d) o[d] = zero16();
    float m = -INFINITY, l = 0.f;

    const uint32_t lds = lds_address(smem) + set * kStage;
    const typename Tl::Lane at;
    const typename Tl::Offsets koff(a.k_sl), voff(a.v_sl);
    auto load = [&](int n) {   // the set's n-th tiles
        const uint32_t tile = lds + n % Tl::kStages * (SETS * kStage);
        const int j0 = (t0 + n * SETS + set) * KT;
        Tl::load(tile, kbase, a.k_sl, j0, len, koff);
        Tl::load(tile + Tl::kBytes, vbase, a.v_sl, j0, len, voff);
    };
    if (t0 < t1)
        for (int n = 0; n < Tl::kStages - 1; ++n) load(n);
    fill_table(a, h, tab);   // while the first tiles are on their way
    loads_done();
    for (int n = 0; t0 + n * SETS < t1; ++n) {
        // the n-th tiles are there, and nobody reads those before them any longer
        wait_and_meet<(Tl::kStages - 2) * 2 * Tl::kLoads>();
        load(n + Tl::kStages - 1);   // past the end too: the waits count loads
        const uint32_t ktile = lds + n % Tl::kStages * (SETS * kStage), vtile = ktile + Tl::kBytes;
        const int j0 = (t0 + n * SETS + set) * KT;
        if (j0 < wend) {
            f32x16 x[KT / 32];
#pragma unroll
            for (int u = 0; u < KT / 32; ++u) x[u] = zero16();
            typename X::Frag kf[KT / 32][HD / 16];
#pragma unroll
            for (int c = 0; c < HD / 16; ++c)
#pragma unroll
                for (int u = 0; u < KT / 32; ++u) kf[u][c] = Tl::rows(ktile, at, 32 * u, c);
            if constexpr (sizeof(T) == 2) __builtin_amdgcn_sched_group_barrier(0x100, KT / 32 * HD / 16, 0);
#pragma unroll
            for (int c = 0; c < HD / 16; ++c)
#pragma unroll
                for (int u = 0; u < KT / 32; ++u) x[u] = X::mma(kf[u][c], qf[c], x[u]);
            if constexpr (sizeof(T) == 2) __builtin_amdgcn_sched_group_barrier(0x008, KT / 32 * HD / 16, 0);
            const int dlo = p0 + w0 - j0 - (KT - 1), dhi = p0 + w0 + 31 - j0;
            float mul = sl2, add = 0.f;   // the scores in log2 units are mul x + add
            if (dlo >= reach.hi || dhi <= reach.lo) {
                add = tab[kPad + (dlo >= reach.hi ? reach.hi - reach.lo : 0)];   // one bias for the whole tile
            } else {
                // dlo > lo - 95 and dhi < hi + 95: within the padded table, masked pairs too
                const float* near = tab + kPad - reach.lo + (pos - j0);
#pragma unroll
                for (int u = 0; u < KT / 32; ++u)
#pragma unroll
                    for (int r = 0; r < 16; ++r) x[u][r] = __builtin_fmaf(x[u][r], sl2, near[-32 * u - row_of(r)]);
                mul = 1.f;
            }
            if ((a.causal && dlo < 0) || j0 + KT > len) {
                const int most = (a.causal ? min(len, pos + 1) : len) - j0 - 4 * (lane >> 5);
#pragma unroll
                for (int u = 0; u < KT / 32; ++u)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (32 * u + 8 * (r / 4) + r % 4 >= most) x[u][r] = -INFINITY;
            }
            float top = x[0][0];
#pragma unroll
            for (int u = 0; u < KT / 32; ++u)
#pragma unroll
                for (int r = 0; r < 16; ++r) top = fmaxf(top, x[u][r]);
            top = __builtin_fmaf(half_max(top), mul, add);   // mul > 0
            if (__any(top > m + kSlack)) {
                const float mn = fmaxf(m, top);
                const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
                m = mn;
                l *= alpha;
#pragma unroll
                for (int d = 0; d < HD / 32; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
            }
            const float mu = m == -INFINITY ? 0.f : m;   // no key yet: every term is 0
#pragma unroll
            for (int u = 0; u < KT / 32; ++u)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    x[u][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[u][r], mul, add - mu));
                    l += x[u][r];
                }
#pragma unroll
            for (int u = 0; u < KT / 32; ++u)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const typename X::Frag p = to_frag<T>(x[u], c);
#pragma unroll
                    for (int d = 0; d < HD / 32; ++d)
                        o[d] = X::mma(Tl::cols(vtile, at, 32 * u + 16 * c, d), p, o[d]);
                }
        }
    }
    wait_and_meet<0>();   // LDS is written until then
    l = half_sum(l);
    if constexpr (SETS == 2) {
        // the second set's maximum, sum and output, a column a lane
        float* other = reinterpret_cast<float*>(smem) + wave * (HD + 2) * 33 + (lane & 31);
        if (set == 1) {
            if (lane < 32) other[HD * 33] = m, other[(HD + 1) * 33] = l;
#pragma unroll
            for (int d = 0; d < HD / 32; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) other[(32 * d + row_of(r)) * 33] = o[d][r];
        }
        __syncthreads();
        if (set == 1) return;
        const float m1 = other[HD * 33], l1 = other[(HD + 1) * 33];
        const float mn = fmaxf(m, m1), mu = mn == -INFINITY ? 0.f : mn;
        const float f0 = __builtin_amdgcn_exp2f(m - mu), f1 = __builtin_amdgcn_exp2f(m1 - mu);
        m = mn;
        l = l * f0 + l1 * f1;
#pragma unroll
        for (int d = 0; d < HD / 32; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[d][r] = o[d][r] * f0 + other[(32 * d + row_of(r)) * 33] * f1;
    }
    if (parts > 1) {
        if (i < a.Lq) {
            const int G = a.H / a.Hk;
            float* p = a.o_part + ((((int64_t)(b * a.Hk + hk) * a.Lq + i) * G + h % G) * parts + part) * (HD + 2);
            typedef __attribute__((__ext_vector_type__(2))) float f32x2;   // rows begin at multiples of 8 bytes
#pragma unroll
            for (int d = 0; d < HD / 32; ++d)
#pragma unroll
                for (int r = 0; r < 16; r += 2) {
                    const f32x2 v = {o[d][r], o[d][r + 1]};
                    *reinterpret_cast<f32x2*>(p + 32 * d + row_of(r)) = v;
                }
            if (lane < 32) p[HD] = m, p[HD + 1] = l;
        }
    } else if (i < a.Lq) {
        const float inv = l == 0.f ? 0.f : 1.0f / l;   // a row without keys: zeros; NaN stays NaN
        T* row = (T*)a.out + b * a.out_sb + h * a.out_sh + (int64_t)i * a.out_sl;
#pragma unroll
        for (int d = 0; d < HD / 32; ++d) store_block<T>(row, 32 * d, o[d], inv);
        if (a.lse && lane < 32)
            a.lse[(int64_t)bh * a.Lq + i] = l == 0.f ? INFINITY : m + __builtin_amdgcn_logf(l);
    }
}

template <typename T, int HD, int SETS>
int launch_sets(const Args& a, hipStream_t st) {
    using Tl = Tile<T, HD>;
    static_assert(SETS == 1 || 4 * (HD + 2) * 33 * 4 <= SETS * 2 * Tl::kStages * Tl::kBytes, "the sets are joined where the tiles were");
    const int lds = SETS * 2 * Tl::kStages * Tl::kBytes + Reach(a).entries() * (int)sizeof(float);
    static Told told;
    if (const int rc = allow_lds((const void*)bias_attn_fwd_kernel<T, HD, SETS>, lds, told)) return rc;
    hipLaunchKernelGGL((bias_attn_fwd_kernel<T, HD, SETS>), dim3((unsigned)(a.B * a.H * a.nq * a.o_parts)), dim3(SETS * kThreads), lds, st, a);
    return check_launch("mb_bias_attn_fwd");
}

// Two sets of waves where the grid leaves room for them on its CUs and the walks are long.  Measured in a
// captured graph, two sets against one, causal, 8 heads: bf16 of 64: 2 x 2048 (256 workgroups) 28 us against 35, 3 x 2048
// 29 against 35, 12 x 512 18 against 15, 4 x 2048 42 against 37; of 128: 2 x 2048 38 against 45, 3 x 2048 43 against
// 49, 12 x 512 27 against 23; of 32: 4 x 2048 25 against 32; fp32 of 64: 3 x 400 35 against 39; of 32, both directions: 23
// against 26; of 128: 4 x 1100 152 against 177, but 8 x 1000 (512 workgroups) 200 against 168.
template <typename T, int HD>
int launch(const Args& a, hipStream_t st) {
    const int blocks = a.B * a.H * a.nq;
    if (a.o_parts == 1 && a.Lk >= 256 && (blocks <= 256 || (a.Lk >= 1024 && blocks <= (HD == 32 ? 512 : 384)))) return launch_sets<T, HD, 2>(a, st);
    return launch_sets<T, HD, 1>(a, st);
}

// Runs that a workgroup's walk is split into, in fp32, where a tile takes three times as long as in
// bf16 and uneven shares of the CUs cost as much more.  Measured in a captured graph, with the launch that joins the
// runs, against one run of two sets of waves: 2 x 2854 both directions, 6 heads of 32 (276 workgroups), 3 runs
// 159 us against 210; 1 x 1102 queries of 1936, 16 heads of 64, 5 runs 81 against 139; 10 x 1466, 2 heads
// of 64, 3 runs 81 against 107; 1 x 1081 both directions, 16 heads of 128, 3 runs 116 against 150 (4 runs 134);
// 2 x 700, 4 heads of 128, 8 runs 39 against 97 (5 runs 39; both directions 48 and 42 against 99); 1 x 383, 5 heads of 128,
// 5 runs 27 against 60; 4 x 553, 4 heads of 64, 4 runs 30 against 45; but 8 x 400, 6 heads of 64 (192 workgroups), 3 runs
// 42 against 36.  bf16 at these sizes: 2 runs 2 to 50 % slower.
int o_parts_of(int B, int H, int Lq, int Lk, int hd, int dtype) {
    const int64_t blocks = (int64_t)B * H * (((int64_t)Lq + kRows - 1) / kRows);
    const bool early = hd == 128 || blocks <= 64;
    if (dtype != MB_DTYPE_F32 || blocks < 1 || blocks > 400 || Lk < (early ? 192 : 448)) return 1;
    const int64_t n = hd == 128 ? 512 / blocks : (640 + blocks - 1) / blocks;
    return (int)std::max<int64_t>(1, std::min<int64_t>(n, std::min(Lk / (early ? 64 : 128), 8)));
}

}  // namespace
}  // namespace battn
}  // namespace mb

using namespace mb;
using namespace mb::battn;

extern "C" int64_t mb_bias_attn_fwd_workspace(int B, int H, int Hk, int Lq, int Lk, int hd, int causal, int dtype) {
    if (B < 1 || H < 1 || Hk < 1 || H % Hk || Lq < 1 || Lk < 0 || hd < 1) return 0;
    int64_t splits = splits_of(B, H, Hk, Lq, Lk, hd, causal);
    if (splits == 0) splits = o_parts_of(B, H, Lq, Lk, hd, dtype);
    return splits > 1 ? (int64_t)B * H * Lq * splits * (hd + 2) * (int64_t)sizeof(float) : 0;
}

extern "C" int mb_bias_attn_fwd(const mb_bias_attn* p, void* stream) {
    Args a = {};
    if (const int rc = fill_args("mb_bias_attn_fwd", p, a)) return rc;
    if (a.B == 0 || a.Lq == 0) return MB_OK;
    const int hd = (int)p->hd, dtype = (int)p->dtype;
    MB_REQUIRE(p->o, "mb_bias_attn_fwd: null pointer argument");
    MB_REQUIRE(rows16(p->o, p->o_st, dtype), "mb_bias_attn_fwd: o's rows must begin at multiples of 16 bytes");
    a.out = p->o, a.out_sb = p->o_st[0], a.out_sh = p->o_st[1], a.out_sl = p->o_st[2];
    a.lse = p->lse;
    const int64_t need = mb_bias_attn_fwd_workspace(a.B, a.H, a.Hk, a.Lq, a.Lk, hd, a.causal, dtype);
    if (need > 0 && (!p->workspace || p->workspace_bytes < need))
        return fail(MB_ERR_WORKSPACE, "mb_bias_attn_fwd: workspace of %lld bytes, %lld are needed",
                    (long long)p->workspace_bytes, (long long)need);
    MB_REQUIRE(need == 0 || ((uintptr_t)p->workspace & 15) == 0, "mb_bias_attn_fwd: the workspace must begin at a multiple of 16 bytes");
    hipStream_t st = (hipStream_t)stream;
    if (const int splits = splits_of(a.B, a.H, a.Hk, a.Lq, a.Lk, hd, a.causal)) return split_launch(a, hd, dtype, splits, p->workspace, st);
    a.o_parts = o_parts_of(a.B, a.H, a.Lq, a.Lk, hd, dtype);
    a.o_part = (float*)p->workspace;
    const int rc = dtype == MB_DTYPE_F32
                       ? (hd == 32 ? launch<float, 32>(a, st) : hd == 64 ? launch<float, 64>(a, st) : launch<float, 128>(a, st))
                       : (hd == 32 ? launch<__bf16, 32>(a, st) : hd == 64 ? launch<__bf16, 64>(a, st) : launch<__bf16, 128>(a, st));
    return rc == MB_OK && a.o_parts > 1 ? join_launch(a, hd, dtype, a.o_parts, a.o_part, st) : rc;
}
