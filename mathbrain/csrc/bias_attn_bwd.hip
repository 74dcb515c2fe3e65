// Backward of the attention with a learned bias by distance buckets.
//
//   p_ij = exp2(t_ij - lse_i),  delta_i = dO_i . o_i,  ds_ij = p_ij (dO_i . v_j - delta_i)
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij dO_i,
//   dbias[n, h] = sum over the pairs of bucket n of ds_ij
//
// Two passes over the pairs, one that owns queries (dq, delta, dbias) and one that owns keys (dk,
// dv), so that every sum has one owner and a fixed order: 7 products of a pair instead of 5, and
// neither atomics in memory nor fp32 copies of dq.
#include "bias_attn_host.h"

#include <algorithm>
#include <cmath>

namespace mb {
namespace battn {
namespace {

// What the keys' pass needs of a row's lse (log2 units).  In bf16 its products start from -lse in
// units of the scores.  In fp32 -lse is added after the product instead: the sum of a product that
// starts from a number of another size is rounded to that one's (dk and dv off by 1.6e-6 of their
// norms at 2 x 1500 tokens).
template <typename T>
__device__ inline float statistic(float lse, float sl2) {
    return sizeof(T) == 2 ? -lse / sl2 : -lse;
}

// Sum of a value over the wave's 64 lanes.
__device__ inline float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// Sums of a wave's 32 x 32 block of ds along its diagonals.  The block goes through LDS (four
// 16-byte writes a lane); then lane t of a half wave reads, for its 16 of the 32 rows i, column
// (i - t) mod 32: distance t of the block where i >= t, distance t - 32 elsewhere.  The keys go up
// by 32 a block, so the latter distances are the next block's t: they are carried over, and an
// entry of `sums` (one for each distance and wave) is written once, when it is whole.
// LDS atomics on the distances' entries took 226 cycles for an instruction of 64 lanes: 250 us of
// this kernel at 56 x 512 tokens, 8 heads x 64.
struct Diagonals {
    static constexpr int kStride = 36;
    typedef __attribute__((address_space(3))) const float lds_float;
    float* block;    // the wave's [32][kStride]
    float* sums;     // the wave's entry of distance 0 + lane % 32
    // of this lane's 16 values: where they lie in LDS, and 1 where the value is of distance t (0: t - 32)
    uint32_t at[16];
    float here[16];
    float carry = 0.f;
    bool open = false;

    __device__ void start(float* block_, float* sums_) {
        const int lane = threadIdx.x & 63, t = lane & 31, g = lane >> 5;
        block = block_;
        sums = sums_ + t;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const int i = 16 * g + k;
            at[k] = lds_address(block + i * kStride + ((i - t) & 31));
            here[k] = i >= t ? 1.f : 0.f;
        }
    }

    // The block into LDS; take() follows, with the products that need the block between them.
    __device__ void give(const f32x16& x) {
        const int lane = threadIdx.x & 63, t = lane & 31, g = lane >> 5;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const f32x4 v = {x[4 * r], x[4 * r + 1], x[4 * r + 2], x[4 * r + 3]};
            *reinterpret_cast<f32x4*>(block + t * kStride + 8 * r + 4 * g) = v;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    __device__ void take(int d0) {
        const int t = threadIdx.x & 31, g = (threadIdx.x >> 5) & 1;
        float mine = carry, next = 0.f;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const float v = *(lds_float*)(uintptr_t)at[k];
            mine = __builtin_fmaf(v, here[k], mine);
            next += 16 * g + k >= t ? 0.f : v;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        put(d0, mine);
        carry = next;
        open = true;
    }
    __device__ void put(int d, float v) {
        v = half_sum(v);
        if ((threadIdx.x & 63) < 32) sums[d] = v;
    }
    // After the last block (d0): what was carried out of it.
    __device__ void close(int d0) {
        if (open) put(d0 - 32, carry);
        open = false;
        carry = 0.f;
    }
};

// Heads of 128 leave registers for 32 keys at a time in the queries' pass (8 x 1024 tokens, 8 heads, bf16: 71 us against
// 112 with 64 keys, which spill).
template <typename T, int HD>
using QueryTile = Tile<T, HD, HD == 128 ? 32 : Ty<T>::kKeys>;

// A workgroup takes 128 queries of a head and walks their keys, or one of q_parts equal runs of this
// walk; bias_attn_add_q_kernel then adds what the runs found.
// dbias: a block of pairs that lies within one bucket adds to a register, any other adds to its
// distances' entries in LDS (Diagonals).  In the end the entries are added by buckets, into the
// workgroup's own row of a workspace.
template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, (waves_per_simd<T, HD, sizeof(T) == 4>())) bias_attn_dq_kernel(const Args a) {
    using X = Ty<T>;
    using Tl = QueryTile<T, HD>;
    constexpr int KT = Tl::kN;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const Reach reach(a);
    const int entries = reach.entries();
    float* tab = reinterpret_cast<float*>(smem + 2 * Tl::kStages * Tl::kBytes);
    float* hist = tab + entries;   // [wave][entries], then the waves' blocks

    const int lane = threadIdx.x & 63, wave = wave_id();
    int bh, qb;
    place(blockIdx.x, a.B * a.H, a.nq * a.q_parts, false, bh, qb);
    const int part = qb % a.q_parts;
    qb /= a.q_parts;
    const int b = bh / a.H, h = bh % a.H, hk = h / (a.H / a.Hk);
    const int len = key_count(a, b), p0 = first_position(a, b);
    const int w0 = qb * kRows + wave * kWaveRows;
    const int i = w0 + (lane & 31), pos = p0 + i;
    const int last = min(a.Lq, (qb + 1) * kRows) - 1;
    const int kend = a.causal ? min(len, p0 + last + 1) : len;
    const int wend = w0 >= a.Lq ? 0 : a.causal ? min(len, p0 + min(a.Lq, w0 + kWaveRows)) : len;
    const int tiles = kend > 0 ? (kend + KT - 1) / KT : 0;
    const float sl2 = a.scale * kLog2e;
    const bool want_bias = a.dbias_part != nullptr;

    const T* kbase = (const T*)a.k + b * a.k_sb + hk * a.k_sh;
    const T* vbase = (const T*)a.v + b * a.v_sb + hk * a.v_sh;
    typename X::Frag qf[HD / 16], gf[HD / 16];
    load_frags<T, HD>((const T*)a.d_o + b * a.do_sb + h * a.do_sh, a.do_sl, w0, a.Lq, gf);
    load_frags<T, HD>((const T*)a.q + b * a.q_sb + h * a.q_sh, a.q_sl, w0, a.Lq, qf);
    const float lse = i < a.Lq ? a.lse[(int64_t)bh * a.Lq + i] : INFINITY;
    // delta is dO . o, but o and the probabilities in it are rounded where the inputs are bf16, and
    // delta's error is that of every ds of its row.  It falls with the number of keys that share
    // the row's weight; where there are few of them delta is taken from the pairs themselves, in a
    // walk of its own (64 sequences of 3 tokens, heads of 64: dbias off by 5e-3 of its norm with dO . o).
    const bool from_pairs = sizeof(T) == 2 && kend <= kRows;
    float delta = 0.f;
    const uint32_t lds = lds_address(smem);
    const typename Tl::Offsets koff(a.k_sl), voff(a.v_sl);
    auto load = [&](int t) {
        const uint32_t tile = lds + t % Tl::kStages * (2 * Tl::kBytes);
        Tl::load(tile, kbase, a.k_sl, t * KT, len, koff);
        Tl::load(tile + Tl::kBytes, vbase, a.v_sl, t * KT, len, voff);
    };
    // the first of the tiles t0 .. t1 - 1
    auto begin = [&](int t0, int t1) {
        if (t0 < t1)
            for (int t = t0; t < t0 + Tl::kStages - 1; ++t) load(t);
    };
    // (at most 2^24 tiles and 8 parts)
    const int run0 = (int)((uint32_t)(tiles * part) / (uint32_t)a.q_parts), run1 = (int)((uint32_t)(tiles * (part + 1)) / (uint32_t)a.q_parts);
    if (!from_pairs) {
        typename X::Frag of[HD / 16];
        load_frags<T, HD>((const T*)a.o + b * a.o_sb + h * a.o_sh, a.o_sl, w0, a.Lq, of);
        begin(run0, run1);
        fill_table(a, h, tab);   // while all of these are on their way
#pragma unroll
        for (int c = 0; c < HD / 16; ++c)
#pragma unroll
            for (int e = 0; e < 8; ++e) delta = __builtin_fmaf((float)of[c][e], (float)gf[c][e], delta);
        delta = half_sum(delta);
    } else {
        begin(0, tiles);
        fill_table(a, h, tab);
    }
    // In bf16 with heads of 64 the products' results start from -lse (in units of the scores) and
    // -delta, in two blocks of registers that leave two waves a SIMD room: p is then
    // exp2(scale x + bias) and ds is p y.
    constexpr bool kStart = HD == 64 && sizeof(T) == 2;
    const float nlse = statistic<T>(lse, sl2);
    if (i < a.Lq && lane < 32) a.rows[(int64_t)bh * a.Lq + i] = nlse;
    f32x16 x0, y0;
#pragma unroll
    for (int r = 0; r < 16; ++r) x0[r] = kStart ? nlse : 0.f, y0[r] = kStart ? -delta : 0.f;
    if (want_bias)
        for (int n = threadIdx.x; n < 4 * entries; n += kThreads) hist[n] = 0.f;
    Diagonals diag;
    if (want_bias)
        diag.start(reinterpret_cast<float*>(smem + 2 * Tl::kStages * Tl::kBytes) + ((5 * entries + 3) & ~3) + wave * 32 * Diagonals::kStride,
                   hist + wave * entries + kPad - reach.lo);
    // Keys go up, so the blocks at or above the reach come first, those at or below its lower end last.
    float far_hi = 0.f, far_sum = 0.f, row_sum = 0.f;
    float far_p_hi = 0.f, far_p = 0.f;   // the blocks' probabilities
    bool first_part = true;
    int last_d0 = 0;

    f32x16 dq[HD / 32];
#pragma unroll
    for (int d = 0; d < HD / 32; ++d) dq[d] = zero16();
    const typename Tl::Lane at;
    // block(ktile, vtile, u, jb) for the wave's blocks of 32 keys from jb on, in rows 32 u of the tiles
    // t0 .. t1 - 1, whose first are on their way
    auto walk = [&](int t0, int t1, auto&& block) {
        for (int t = t0; t < t1; ++t) {
            wait_and_meet<(Tl::kStages - 2) * 2 * Tl::kLoads>();   // as in the forward
            load(t + Tl::kStages - 1);
            const uint32_t ktile = lds + t % Tl::kStages * (2 * Tl::kBytes), vtile = ktile + Tl::kBytes;
#pragma unroll
            for (int u = 0; u < KT / 32; ++u) {
                const int jb = t * KT + 32 * u;
                if (jb >= wend) break;
                block(ktile, vtile, u, jb);
            }
        }
        wait_and_meet<0>();   // LDS is written until then
    };
    // A block's exponents (log2 of p, but for lse where the products do not start from it) and dO . v
    // (less delta where they do).
    auto products = [&](uint32_t ktile, uint32_t vtile, int u, int jb, f32x16& x, f32x16& y) {
        x = x0, y = y0;
        typename X::Frag kr[HD / 16], vr[HD / 16];
#pragma unroll
        for (int c = 0; c < HD / 16; ++c) kr[c] = Tl::rows(ktile, at, 32 * u, c), vr[c] = Tl::rows(vtile, at, 32 * u, c);
        // all reads before the first product (heads of 64: 92 -> 90 us at 56 x 512; others have no room)
        if constexpr (kStart) __builtin_amdgcn_sched_group_barrier(0x100, HD / 8, 0);
#pragma unroll
        for (int c = 0; c < HD / 16; ++c) {
            x = X::mma(kr[c], qf[c], x);
            y = X::mma(vr[c], gf[c], y);
        }
        if constexpr (kStart) __builtin_amdgcn_sched_group_barrier(0x008, HD / 8, 0);
        const int dlo = p0 + w0 - jb - 31, dhi = p0 + w0 + 31 - jb;
        if (dlo >= reach.hi || dhi <= reach.lo) {
            const float bias = tab[kPad + (dlo >= reach.hi ? reach.hi - reach.lo : 0)];
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] = __builtin_fmaf(x[r], sl2, bias);
        } else {
            const float* near = tab + kPad - reach.lo + (pos - jb);
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] = __builtin_fmaf(x[r], sl2, near[-row_of(r)]);
        }
        if ((a.causal && dlo < 0) || jb + 32 > len) {
            const int most = a.causal ? min(len, pos + 1) : len;
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (jb + row_of(r) >= most) x[r] = -INFINITY;
        }
    };
    loads_done();
    if (from_pairs) {
        walk(0, tiles, [&](uint32_t ktile, uint32_t vtile, int u, int jb) {
            f32x16 x, y;
            products(ktile, vtile, u, jb, x, y);
#pragma unroll
            for (int r = 0; r < 16; ++r) delta = __builtin_fmaf(__builtin_amdgcn_exp2f(kStart ? x[r] : x[r] - lse), y[r], delta);
        });
        begin(run0, run1);
        delta = half_sum(delta);
        if (kStart)
#pragma unroll
            for (int r = 0; r < 16; ++r) y0[r] = -delta;
    }
    walk(run0, run1, [&](uint32_t ktile, uint32_t vtile, int u, int jb) {
        const int dlo = p0 + w0 - jb - 31, dhi = p0 + w0 + 31 - jb;
        const bool above = dlo >= reach.hi, one = above || dhi <= reach.lo;
        if (first_part && !above) {
            first_part = false;
            far_hi = far_sum, far_sum = 0.f;
            far_p_hi = far_p, far_p = 0.f;
        }
        f32x16 x, y;
        products(ktile, vtile, u, jb, x, y);
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = __builtin_amdgcn_exp2f(kStart ? x[r] : x[r] - lse);
        if (sizeof(T) == 2 && want_bias && one) {
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int r = 0; r < 16; ++r) sum[r % 4] += x[r];
            far_p += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] *= kStart ? y[r] : y[r] - delta;
        if (want_bias && !one) diag.give(x);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const typename X::Frag f = to_frag<T>(x, c);
#pragma unroll
            for (int d = 0; d < HD / 32; ++d) dq[d] = X::mma(Tl::cols(ktile, at, 32 * u + 16 * c, d), f, dq[d]);
        }
        // while the products run:
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int r = 0; r < 16; ++r) sum[r % 4] += x[r];
        const float all = (sum[0] + sum[1]) + (sum[2] + sum[3]);
        row_sum += all;
        if (want_bias) {
            if (one) {
                diag.close(last_d0);
                far_sum += all;
            } else {
                last_d0 = dlo + 31;
                diag.take(last_d0);
            }
        }
    });
    // A row's ds sum to zero but for delta's error, which comes from o's rounding and that of the
    // probabilities in it: for the keys' pass delta is put right by what is left.
    row_sum = half_sum(row_sum);
    float far_lo = far_sum;
    if (first_part) far_hi = far_lo, far_lo = 0.f, far_p_hi = far_p, far_p = 0.f;
    if (i < a.Lq && a.q_parts > 1) {
        const int64_t all = (int64_t)a.B * a.H * a.Lq, at = (int64_t)bh * a.Lq + i;
        const float p_hi = half_sum(far_p_hi), p_lo = half_sum(far_p);
        float* stat = a.q_stat + 4 * part * all + at;
        if (lane < 32) stat[0] = row_sum, stat[all] = p_hi, stat[2 * all] = p_lo, stat[3 * all] = delta;
        float* row = a.q_part + (part * all + at) * HD;
#pragma unroll
        for (int d = 0; d < HD / 32; ++d) store_block<float>(row, 32 * d, dq[d], a.scale);
    } else if (i < a.Lq) {
        if (lane < 32) a.rows[((int64_t)a.B * a.H + bh) * a.Lq + i] = -(delta + row_sum);
        T* row = (T*)a.out + b * a.out_sb + h * a.out_sh + (int64_t)i * a.out_sl;
#pragma unroll
        for (int d = 0; d < HD / 32; ++d) store_block<T>(row, 32 * d, dq[d], a.scale);
    }
    if (!want_bias) return;
    diag.close(last_d0);
    // delta's error again: what is left of a row's sum belongs to its pairs by their probability.  The
    // blocks of one bucket, which have most of it in long rows, are put right here.
    if (sizeof(T) == 2 && a.q_parts == 1) far_hi -= row_sum * far_p_hi, far_lo -= row_sum * far_p;
    // The whole blocks' sums go where no diagonal reaches: the padding's 63rd entries and on.
    far_hi = half_sum(far_hi);
    far_lo = half_sum(far_lo);
    if (lane < 32) diag.sums[reach.hi + 63] = far_hi, diag.sums[reach.lo - 94] = far_lo;
    __syncthreads();
    float* sums = a.dbias_part + (h * a.bias_rows + ((int64_t)b * a.nq + qb) * a.q_parts + part) * a.buckets;
    for (int n = threadIdx.x / 8; n < a.buckets; n += kThreads / 8) {   // eight lanes a bucket
        const bool back = n >= a.n_starts;        // keys behind the query's position
        const int m = back ? n - a.n_starts : n;
        const bool end = m == a.n_starts - 1;
        // its distances' entries, those of the padding with the last bucket's (and, in a causal table,
        // the first one's: a whole block at or below distance 0 has nothing else that counts)
        int e0 = a.starts[m], e1 = end ? reach.hi + kPad : a.starts[m + 1] - 1;
        if (back) {
            const int near = max(e0, 1);
            e0 = -e1, e1 = -near;
        } else if (a.causal && n == 0) {
            e0 = -kPad;
        }
        e0 += kPad - reach.lo, e1 += kPad - reach.lo;
        float v = 0.f;
        for (int e = e0 + (lane & 7); e <= e1; e += 16) {
            const int next = e + 8 <= e1 ? e + 8 : e;
            float x = 0.f, y = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) x += hist[w * entries + e], y += hist[w * entries + next];
            v += next > e ? x + y : x;
        }
#pragma unroll
        for (int o = 4; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
        if ((lane & 7) == 0) sums[n] = v;
    }
}

// Where the queries' pass is split: dq and the rows' sums of ds from the runs', in order, and in bf16
// what delta's error left in the blocks of one bucket, as a row of dbias's parts of its own.  Four
// workgroups take 128 queries of a head, 32 each; the first of them has all the sums of ds.
template <typename T, int HD>
__global__ void __launch_bounds__(kThreads) bias_attn_add_q_kernel(const Args a) {
    __shared__ float left[kThreads / 64][2];
    const int quarter = blockIdx.x % 4, qb = blockIdx.x / 4 % a.nq, bh = blockIdx.x / 4 / a.nq, b = bh / a.H, h = bh % a.H;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t all = (int64_t)a.B * a.H * a.Lq, first = (int64_t)bh * a.Lq + (int64_t)qb * kRows;
    const int rows = min(kRows, a.Lq - qb * kRows);
    float hi = 0.f, lo = 0.f;
    if (quarter == 0 && (int)threadIdx.x < rows) {
        const float* stat = a.q_stat + first + threadIdx.x;
        float sum = 0.f;
        for (int s = 0; s < a.q_parts; ++s, stat += 4 * all) sum += stat[0], hi += stat[all], lo += stat[2 * all];
        a.rows[all + first + threadIdx.x] = -(a.q_stat[3 * all + first + threadIdx.x] + sum);
        hi *= sum, lo *= sum;
    }
    const bool correct = sizeof(T) == 2 && a.dbias_part && quarter == 0;
    if (correct) {
        hi = wave_sum(hi), lo = wave_sum(lo);
        if (lane == 0) left[wave][0] = hi, left[wave][1] = lo;
        __syncthreads();
        float* sums = a.dbias_part + (h * a.bias_rows + (int64_t)a.B * a.nq * a.q_parts + (int64_t)b * a.nq + qb) * a.buckets;
        for (int n = threadIdx.x; n < a.buckets; n += kThreads) {
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < kThreads / 64; ++w) {
                if (n == a.n_starts - 1) v -= left[w][0];
                if (n == (a.causal ? 0 : a.buckets - 1)) v -= left[w][1];
            }
            sums[n] = v;
        }
    }
    for (int n = threadIdx.x; n < min(kWaveRows, rows - quarter * kWaveRows) * (HD / 4); n += kThreads) {
        const int r = quarter * kWaveRows + n / (HD / 4), d = n % (HD / 4) * 4;
        const float* p = a.q_part + (first + r) * HD + d;
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
        for (int s0 = 0; s0 < a.q_parts; s0 += 4) {   // four loads on their way together
            f32x4 x[4];
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
                x[s] = zero;
                if (s0 + s < a.q_parts) x[s] = *reinterpret_cast<const f32x4*>(p + (s0 + s) * all * HD);
            }
#pragma unroll
            for (int s = 0; s < 4; ++s) sum += x[s];
        }
        typename Ty<T>::Quad v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (T)sum[e];
        *reinterpret_cast<typename Ty<T>::Quad*>((T*)a.out + b * a.out_sb + h * a.out_sh + (int64_t)(qb * kRows + r) * a.out_sl + d) = v;
    }
}

// dbias[n, h] = the sum of part[h, :, n], in a fixed order, by a workgroup: strips of rows.
__device__ inline void add_parts(const Args& a, int h, float* sums) {
    const int rows = (int)a.bias_rows;
    const int strips = kThreads / a.buckets;   // at least one: buckets <= 256
    const int n = threadIdx.x % a.buckets, strip = threadIdx.x / a.buckets;
    const float* part = a.dbias_part + (int64_t)h * rows * a.buckets + n;
    float v = 0.f;
    if (strip < strips)
        for (int r = strip; r < rows; r += strips) v += part[(int64_t)r * a.buckets];
    sums[threadIdx.x] = v;
    __syncthreads();
    if (strip == 0) {
        for (int k = 1; k < strips; ++k) v += sums[k * a.buckets + n];
        const int64_t at = (int64_t)n * a.H + h;
        if (a.bias_bf16) ((__bf16*)a.dbias)[at] = (__bf16)v;
        else ((float*)a.dbias)[at] = v;
    }
}
static_assert(2 * kMaxStarts <= kThreads, "a thread for every bucket");

// A workgroup takes 128 keys of one key head, 32 to a wave, and walks the queries of all query
// heads that share it, or one of kv_parts equal runs of this walk; the runs' sums are then added by
// bias_attn_add_kv_kernel.  Where dbias is wanted, H workgroups before these add the queries' pass's
// parts of it.
template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, (waves_per_simd<T, HD, true>())) bias_attn_dkv_kernel(const Args a) {
    using X = Ty<T>;
    using Tl = Tile<T, HD>;
    constexpr int QT = Tl::kN;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ __attribute__((aligned(16))) float stat[Tl::kStages][2][64];   // rows' -lse and -delta
    float* tab = reinterpret_cast<float*>(smem + 2 * Tl::kStages * Tl::kBytes);

    const int nk = (a.Lk + kRows - 1) / kRows;
    const int id = (int)blockIdx.x - (a.dbias ? a.H : 0);
    if (id < 0) {
        add_parts(a, blockIdx.x, reinterpret_cast<float*>(smem));
        return;
    }
    const int lane = threadIdx.x & 63, wave = wave_id(), g = lane >> 5;
    int bh, kb;
    place(id, a.B * a.Hk, nk * a.kv_parts, true, bh, kb);
    const int part = kb % a.kv_parts;
    kb /= a.kv_parts;
    const int b = bh / a.Hk, hk = bh % a.Hk, group = a.H / a.Hk;
    const Reach reach(a);
    const int len = key_count(a, b), p0 = first_position(a, b);
    const int k0 = kb * kRows, w0 = k0 + wave * kWaveRows;
    const int j = w0 + (lane & 31);
    // queries from the first one that sees key k0
    const int first = a.causal ? max(0, k0 - p0) / QT : 0;
    const int tiles = k0 < len ? (a.Lq + QT - 1) / QT : 0;
    const int steps = max(0, tiles - first);   // of a head
    const bool whole = a.kv_parts == 1;
    const int64_t all = (int64_t)group * steps, step0 = whole ? 0 : all * part / a.kv_parts, step1 = whole ? all : all * (part + 1) / a.kv_parts;
    const float sl2 = a.scale * kLog2e;

    typename X::Frag kf[HD / 16], vf[HD / 16];
    load_frags<T, HD>((const T*)a.k + b * a.k_sb + hk * a.k_sh, a.k_sl, w0, len, kf);
    load_frags<T, HD>((const T*)a.v + b * a.v_sb + hk * a.v_sh, a.v_sl, w0, len, vf);
    f32x16 dk[HD / 32], dv[HD / 32];
#pragma unroll
    for (int d = 0; d < HD / 32; ++d) dk[d] = zero16(), dv[d] = zero16();

    const uint32_t lds = lds_address(smem);
    const typename Tl::Lane at;
    const typename Tl::Offsets qoff(a.q_sl), goff(a.do_sl);
    for (int hh = 0; hh < group; ++hh) {
        const int h = hk * group + hh;
        const T* qbase = (const T*)a.q + b * a.q_sb + h * a.q_sh;
        const T* gbase = (const T*)a.d_o + b * a.do_sb + h * a.do_sh;
        const float* nlse = a.rows + ((int64_t)b * a.H + h) * a.Lq;
        const float* ndelta = nlse + (int64_t)a.B * a.H * a.Lq;
        auto load = [&](int t) {
            const int s = t % Tl::kStages;
            if (wave < 2)   // one wave the rows' -lse, another their -delta; the last row's past the end
                dma4(lds_address(&stat[s][wave][0]), 4u * (uint32_t)min(t * QT + lane, a.Lq - 1),
                     wave ? ndelta : nlse);
            const uint32_t tile = lds + s * (2 * Tl::kBytes);
            Tl::load(tile, qbase, a.q_sl, t * QT, a.Lq, qoff);
            Tl::load(tile + Tl::kBytes, gbase, a.do_sl, t * QT, a.Lq, goff);
        };
        // the run's share of this head
        const int64_t at0 = step0 - (int64_t)hh * steps, at1 = step1 - (int64_t)hh * steps;
        const int t0 = first + (int)(at0 < 0 ? 0 : at0 < steps ? at0 : steps), t1 = first + (int)(at1 < 0 ? 0 : at1 < steps ? at1 : steps);
        if (t0 >= t1) continue;
        // the previous head's last barrier lies behind its reads
        for (int t = t0; t < t0 + Tl::kStages - 1; ++t) load(t);
        fill_table(a, h, tab);   // while these are on their way
        loads_done();
        for (int t = t0; t < t1; ++t) {
            const int s = t % Tl::kStages;
            // (two waves have a load more on their way: they wait for that one of the next tile too)
            wait_and_meet<(Tl::kStages - 2) * 2 * Tl::kLoads>();
            load(t + Tl::kStages - 1);
            const uint32_t qtile = lds + s * (2 * Tl::kBytes), gtile = qtile + Tl::kBytes;
#pragma unroll
            for (int u = 0; u < QT / 32; ++u) {
                const int ib = t * QT + 32 * u;
                if (ib >= a.Lq || w0 >= len || (a.causal && p0 + ib + 31 < w0)) continue;
                f32x16 x, y;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const f32x4 nl = *reinterpret_cast<const f32x4*>(&stat[s][0][32 * u + 8 * r + 4 * g]);
                    const f32x4 nd = *reinterpret_cast<const f32x4*>(&stat[s][1][32 * u + 8 * r + 4 * g]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[4 * r + e] = sizeof(T) == 2 ? nl[e] : 0.f, y[4 * r + e] = nd[e];
                }
                typename X::Frag qr[HD / 16], gr[HD / 16];
#pragma unroll
                for (int c = 0; c < HD / 16; ++c) qr[c] = Tl::rows(qtile, at, 32 * u, c), gr[c] = Tl::rows(gtile, at, 32 * u, c);
                // all reads before the first product (heads of 64: 81 -> 76 us at 56 x 512)
                if constexpr (sizeof(T) == 2) __builtin_amdgcn_sched_group_barrier(0x100, HD / 8 + 8, 0);
#pragma unroll
                for (int c = 0; c < HD / 16; ++c) {
                    x = X::mma(qr[c], kf[c], x);
                    y = X::mma(gr[c], vf[c], y);
                }
                if constexpr (sizeof(T) == 2) __builtin_amdgcn_sched_group_barrier(0x008, HD / 8, 0);
                const int dlo = p0 + ib - w0 - 31, dhi = p0 + ib + 31 - w0;
                const bool above = dlo >= reach.hi;
                if (above || dhi <= reach.lo) {
                    const float bias = tab[kPad + (above ? reach.hi - reach.lo : 0)];
#pragma unroll
                    for (int r = 0; r < 16; ++r) x[r] = __builtin_fmaf(x[r], sl2, bias);
                } else {
                    const float* near = tab + kPad - reach.lo + (p0 + ib - j);
#pragma unroll
                    for (int r = 0; r < 16; ++r) x[r] = __builtin_fmaf(x[r], sl2, near[row_of(r)]);
                }
                if ((a.causal && dlo < 0) || w0 + 32 > len || ib + 32 > a.Lq) {
                    const int least = j >= len ? 0x7fffffff : a.causal ? j - p0 : -0x7fffffff;
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int i = ib + row_of(r);
                        if (i < least || i >= a.Lq) x[r] = -INFINITY;
                    }
                }
                if constexpr (sizeof(T) == 4) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const f32x4 nl = *reinterpret_cast<const f32x4*>(&stat[s][0][32 * u + 8 * r + 4 * g]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[4 * r + e] += nl[e];
                    }
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    x[r] = __builtin_amdgcn_exp2f(x[r]);
                    y[r] *= x[r];
                }
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const typename X::Frag p = to_frag<T>(x, c), ds = to_frag<T>(y, c);
#pragma unroll
                    for (int d = 0; d < HD / 32; ++d) {
                        dv[d] = X::mma(Tl::cols(gtile, at, 32 * u + 16 * c, d), p, dv[d]);
                        dk[d] = X::mma(Tl::cols(qtile, at, 32 * u + 16 * c, d), ds, dk[d]);
                    }
                }
            }
        }
        wait_and_meet<0>();   // the next head's loads and table go where this one's were
    }
    if (j < a.Lk && a.kv_parts > 1) {
        float* row = a.kv_part + (((int64_t)part * a.B * a.Hk + bh) * a.Lk + j) * 2 * HD;
#pragma unroll
        for (int d = 0; d < HD / 32; ++d) {
            store_block<float>(row, 32 * d, dk[d], a.scale);
            store_block<float>(row + HD, 32 * d, dv[d], 1.f);
        }
    } else if (j < a.Lk) {
        T* krow = (T*)a.dk + b * a.dk_sb + hk * a.dk_sh + (int64_t)j * a.dk_sl;
        T* vrow = (T*)a.dv + b * a.dv_sb + hk * a.dv_sh + (int64_t)j * a.dv_sl;
#pragma unroll
        for (int d = 0; d < HD / 32; ++d) {
            store_block<T>(krow, 32 * d, dk[d], a.scale);
            store_block<T>(vrow, 32 * d, dv[d], 1.f);
        }
    }
}

// dk and dv where the keys' pass is split: the runs' sums in order, four channels a thread.
template <typename T, int HD>
__global__ void __launch_bounds__(kThreads) bias_attn_add_kv_kernel(const Args a) {
    const int64_t rows = (int64_t)a.B * a.Hk * a.Lk, n = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (n >= rows * (HD / 2)) return;
    const int64_t row = n / (HD / 2);
    const int c = (int)(n % (HD / 2)) * 4, which = c / HD, d = c % HD;
    const float* p = a.kv_part + row * 2 * HD + c;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < a.kv_parts; s0 += 4) {   // four loads on their way together
        f32x4 x[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
            x[s] = zero;
            if (s0 + s < a.kv_parts) x[s] = *reinterpret_cast<const f32x4*>(p + (s0 + s) * rows * 2 * HD);
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) sum += x[s];
    }
    const int64_t bh = row / a.Lk, j = row - bh * a.Lk, b = bh / a.Hk, h = bh - b * a.Hk;
    T* out = which ? (T*)a.dv + b * a.dv_sb + h * a.dv_sh + j * a.dv_sl : (T*)a.dk + b * a.dk_sb + h * a.dk_sh + j * a.dk_sl;
    typename Ty<T>::Quad v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (T)sum[e];
    *reinterpret_cast<typename Ty<T>::Quad*>(out + d) = v;
}

template <typename T, int HD>
int launch(const Args& a, hipStream_t st) {
    const int entries = Reach(a).entries();
    const int table = entries * (int)sizeof(float);
    const int base = 2 * Tile<T, HD>::kStages * Tile<T, HD>::kBytes + table;
    const int lds_q = 2 * QueryTile<T, HD>::kStages * QueryTile<T, HD>::kBytes + table + (a.dbias_part ? (4 * entries + 3 + 4 * 32 * Diagonals::kStride) * (int)sizeof(float) : 0);
    if (a.B > 0 && a.Lq > 0) {
        static Told told;
        if (const int rc = allow_lds((const void*)bias_attn_dq_kernel<T, HD>, lds_q, told)) return rc;
        hipLaunchKernelGGL((bias_attn_dq_kernel<T, HD>), dim3((unsigned)(a.B * a.H * a.nq * a.q_parts)), dim3(kThreads), lds_q, st, a);
        if (a.q_parts > 1)
            hipLaunchKernelGGL((bias_attn_add_q_kernel<T, HD>), dim3((unsigned)(a.B * a.H * a.nq * 4)), dim3(kThreads), 0, st, a);
    }
    const int nk = (a.Lk + kRows - 1) / kRows, blocks = a.B * a.Hk * nk * a.kv_parts + (a.dbias ? a.H : 0);
    if (blocks > 0) {
        static Told told;
        if (const int rc = allow_lds((const void*)bias_attn_dkv_kernel<T, HD>, base, told)) return rc;
        hipLaunchKernelGGL((bias_attn_dkv_kernel<T, HD>), dim3((unsigned)blocks), dim3(kThreads), base, st, a);
    }
    if (a.kv_parts > 1) {
        const int64_t threads = (int64_t)a.B * a.Hk * a.Lk * (HD / 2);
        hipLaunchKernelGGL((bias_attn_add_kv_kernel<T, HD>), dim3((unsigned)((threads + kThreads - 1) / kThreads)), dim3(kThreads), 0,
                           st, a);
    }
    return check_launch("mb_bias_attn_bwd");
}

int64_t padded(int64_t floats) { return (floats + 3) & ~(int64_t)3; }

// Runs that a pass splits each walk into, for `groups` workgroups of `steps` 64-row tiles each: where
// there are few, most of the device would wait for the longest.  The time is counted in tiles: a run's
// own start and end, that of the launch which adds the runs, and what two workgroups of a CU take
// from each other.  Measured, split against not, dq / dk and dv, launches that add included:
// causal bf16 heads of 64, 2 x 1310, 8 heads (176 workgroups, 21 tiles) 32 us against 41 / 31 against
// 38; 9 x 2259, one head 40 against 63 / 39 against 59; heads of 128, 2 x 1516, 4 heads on 2 key
// heads 41 against 72 / 45 against 122; fp32 heads of 64, 3 x 1000, 8 heads 77 against 124 / 100 against
// 160; fp32 heads of 128, 1 x 1081 both directions, 16 heads on 4 key heads 193 against 252 / 204 against 1180;
// 1 x 383, 5 heads of 128, runs of 64 rows 37 against 47 / 36 against 52 with three runs.
int parts_of(int64_t groups, int64_t steps, int per_cu, bool causal, int dtype) {
    if (groups < 1 || groups > 512) return 1;
    const bool f32 = dtype == MB_DTYPE_F32;   // whose tiles keep a CU busy by one workgroup
    const double start = f32 ? causal ? 1.0 : 1.5 : 4.0, join = 1.2 * start;
    int best = 1;
    double least = INFINITY;
    for (int n = 1; n <= 8 && (n == 1 || n <= (f32 ? steps : steps / 2)); ++n) {
        const double wgs = (causal ? 0.95 : 1.0) * groups * n;
        const double run = (double)steps / n + start;
        const double cost = (f32 && causal ? std::max(run, groups * (0.5 * steps + n * start) / 256)
                                           : std::ceil(wgs / (256 * per_cu)) * run * (wgs > 256 && per_cu == 2 ? 1.6 : 1.0))
                            + (n > 1 ? join : 0.0);
        if (cost < (best == 1 ? 0.95 : 1.0) * least) least = cost, best = n;
    }
    // the longest walk is twice the mean under a causal mask (3 x 3461, 5 heads of 32, 420 workgroups of 55 tiles: 64 us
    // against 89 / 58 against 72; but 448 of 16 tiles: 49 against 38 / 50 against 35; fp32, 9 x 900, 6 heads of 64, 432 of 15
    // tiles: 147 against 150 / 164 against 193)
    if (best == 1 && causal && per_cu == 2 && groups > 256 && steps >= (f32 ? 12 : 24)) best = 2;
    return best;
}

// The workspace's parts in floats: the rows' statistics, dbias's sums (and how many for each bucket and
// head), and what the passes' runs find where they are split.
struct Space {
    int q_parts, kv_parts;
    int64_t bias_rows, rows, bias, q, q_stat, kv;
    Space(int B, int H, int Hk, int Lq, int Lk, int hd, bool causal, int dtype, int buckets) {
        const int64_t all = (int64_t)B * H * Lq, nq = ((int64_t)Lq + kRows - 1) / kRows, nk = ((int64_t)Lk + kRows - 1) / kRows;
        q_parts = parts_of(B * H * nq, ((int64_t)Lk + 63) / 64, dtype == MB_DTYPE_F32 && hd == 128 ? 1 : 2, causal, dtype);
        kv_parts = parts_of(B * Hk * nk, (int64_t)(H / Hk) * (((int64_t)Lq + 63) / 64), hd == 128 ? 1 : 2, causal, dtype);
        bias_rows = B * nq * (q_parts > 1 ? q_parts + 1 : 1);
        rows = padded(2 * all);
        bias = padded(H * bias_rows * buckets);
        q = q_parts > 1 ? q_parts * all * hd : 0;
        q_stat = q_parts > 1 ? padded(4 * q_parts * all) : 0;
        kv = kv_parts > 1 ? (int64_t)kv_parts * B * Hk * Lk * 2 * hd : 0;
    }
    int64_t floats() const { return rows + bias + q + q_stat + kv; }
};

}  // namespace
}  // namespace battn
}  // namespace mb

using namespace mb;
using namespace mb::battn;

extern "C" int64_t mb_bias_attn_bwd_workspace(int B, int H, int Hk, int Lq, int Lk, int hd, int causal, int dtype, int buckets) {
    if (B < 1 || H < 1 || Hk < 1 || H % Hk || Lq < 1 || Lk < 0 || hd < 1 || buckets < 1) return 0;
    return Space(B, H, Hk, Lq, Lk, hd, causal != 0, dtype, buckets).floats() * (int64_t)sizeof(float);
}

extern "C" int mb_bias_attn_bwd(const mb_bias_attn* p, void* stream) {
    Args a = {};
    if (const int rc = fill_args("mb_bias_attn_bwd", p, a)) return rc;
    const int hd = (int)p->hd, dtype = (int)p->dtype;
    const int64_t need = mb_bias_attn_bwd_workspace(a.B, a.H, a.Hk, a.Lq, a.Lk, hd, a.causal, dtype, a.buckets);
    if (need > 0 && (!p->workspace || p->workspace_bytes < need))
        return fail(MB_ERR_WORKSPACE, "mb_bias_attn_bwd: workspace of %lld bytes, %lld are needed",
                    (long long)p->workspace_bytes, (long long)need);
    MB_REQUIRE(need == 0 || ((uintptr_t)p->workspace & 15) == 0, "mb_bias_attn_bwd: the workspace must begin at a multiple of 16 bytes");
    if (a.B > 0 && a.Lq > 0) {
        MB_REQUIRE(p->o && p->d_o && p->lse && p->dq, "mb_bias_attn_bwd: null pointer argument");
        MB_REQUIRE(rows16(p->o, p->o_st, dtype) && rows16(p->d_o, p->do_st, dtype) && rows16(p->dq, p->dq_st, dtype),
                   "mb_bias_attn_bwd: rows must begin at multiples of 16 bytes");
        MB_REQUIRE(p->do_st[2] >= 0 && p->do_st[2] <= (1 << 24) / (dtype == MB_DTYPE_F32 ? 4 : 2),
                   "mb_bias_attn_bwd: d_o's rows are %lld elements apart", (long long)p->do_st[2]);
        a.o = p->o, a.o_sb = p->o_st[0], a.o_sh = p->o_st[1], a.o_sl = p->o_st[2];
        a.d_o = p->d_o, a.do_sb = p->do_st[0], a.do_sh = p->do_st[1], a.do_sl = p->do_st[2];
        a.out = p->dq, a.out_sb = p->dq_st[0], a.out_sh = p->dq_st[1], a.out_sl = p->dq_st[2];
    }
    if (a.B > 0 && a.Lk > 0) {
        MB_REQUIRE(p->dk && p->dv, "mb_bias_attn_bwd: null pointer argument");
        MB_REQUIRE(rows16(p->dk, p->dk_st, dtype) && rows16(p->dv, p->dv_st, dtype), "mb_bias_attn_bwd: rows must begin at multiples of 16 bytes");
        a.dk = p->dk, a.dk_sb = p->dk_st[0], a.dk_sh = p->dk_st[1], a.dk_sl = p->dk_st[2];
        a.dv = p->dv, a.dv_sb = p->dv_st[0], a.dv_sh = p->dv_st[1], a.dv_sl = p->dv_st[2];
    }
    a.lse = p->lse;
    a.dbias = p->dbias;
    a.q_parts = a.kv_parts = 1;
    if (need > 0) {
        const Space w(a.B, a.H, a.Hk, a.Lq, a.Lk, hd, a.causal, dtype, a.buckets);
        a.q_parts = w.q_parts, a.kv_parts = w.kv_parts;
        a.bias_rows = dtype == MB_DTYPE_F32 && w.q_parts > 1 ? w.bias_rows / (w.q_parts + 1) * w.q_parts : w.bias_rows;
        a.rows = (float*)p->workspace;
        a.dbias_part = p->dbias ? a.rows + w.rows : nullptr;
        a.q_part = a.rows + w.rows + w.bias;
        a.q_stat = a.q_part + w.q;
        a.kv_part = a.q_stat + w.q_stat;
    }
    hipStream_t st = (hipStream_t)stream;
    return dtype == MB_DTYPE_F32
               ? (hd == 32 ? launch<float, 32>(a, st) : hd == 64 ? launch<float, 64>(a, st) : launch<float, 128>(a, st))
               : (hd == 32 ? launch<__bf16, 32>(a, st) : hd == 64 ? launch<__bf16, 64>(a, st) : launch<__bf16, 128>(a, st));
}
