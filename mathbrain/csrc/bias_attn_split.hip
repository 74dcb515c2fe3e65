// Forward of the attention with a learned bias by distance buckets where there are few queries: the
// keys of a row are split over waves and workgroups, and the parts joined.
#include "bias_attn_host.h"

#include <algorithm>

namespace mb {
namespace battn {
namespace {

// Operand with channels d0 + lane % 32 and rows row0 + (the slots' order) of a tile with padded rows.
template <int STRIDE>
__device__ inline bf16x8 cols_bf16(const __bf16* tile, int row0, int d0) {
    // 16 lanes read 4 rows of 16 channels, 8 bytes each, and get 4 rows of one channel each
    const int lane = threadIdx.x & 63;
    const __bf16* p = tile + (row0 + 4 * (lane >> 5) + ((lane & 15) >> 2)) * STRIDE + d0 + (lane & 16) + 4 * (lane & 3);
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(__attribute__((address_space(3))) void*)p);
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_s16x4*)(__attribute__((address_space(3))) void*)(p + 8 * STRIDE));
    const bf16x4 x = __builtin_bit_cast(bf16x4, a), y = __builtin_bit_cast(bf16x4, b);
    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
}
template <int STRIDE>
__device__ inline f32x8 cols_f32(const float* tile, int row0, int d0) {
    const int lane = threadIdx.x & 63;
    const float* p = tile + (row0 + 4 * (lane >> 5)) * STRIDE + d0 + (lane & 31);
    f32x8 f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = p[(8 * (e / 4) + e % 4) * STRIDE];
    return f;
}

// Rows are the queries of all heads that share a key head, query by query: row r is query r / G of
// head r % G.  A workgroup takes 32 of them (one column of the 32 x 32 products for each, so that 1
// row costs what 32 cost) and one of `splits` parts of the keys that they see; each of its waves
// takes a quarter of the part and walks it alone, 32 keys a step: the keys go from memory straight
// into the registers of the first product, the values through the wave's own corner of LDS, which
// turns them, and both of the next step are on their way meanwhile.  Bound by reading k and v.
template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, (waves_per_simd<T, HD, true>())) bias_attn_split_kernel(const Args a, int splits,
                                                                                                   float* part) {
    using X = Ty<T>;
    constexpr int kVecT = 16 / (int)sizeof(T);
    constexpr int kStride = HD + kVecT;                 // of the values in LDS
    constexpr int kPerRow = HD / kVecT;
    constexpr int kVecs = 32 * kPerRow / 64;
    constexpr int kOut = HD * 33;                       // a wave's output block, [HD][33]
    constexpr int kWaveFloats = kOut > 32 * kStride * (int)sizeof(T) / 4 ? kOut : 32 * kStride * (int)sizeof(T) / 4;
    static_assert(kOut % 4 == 0, "the waves' corners begin at multiples of 16 bytes");
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ float stat[4][2][32];
    float* corner = reinterpret_cast<float*>(smem);     // [4][kWaveFloats]
    float* values = corner + 4 * kWaveFloats;           // near blocks: [buckets][G] biases,
    uint8_t* bucket = reinterpret_cast<uint8_t*>(values + a.buckets * (a.H / a.Hk));  // and each distance's bucket

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 5;
    const int G = a.H / a.Hk, rows = G * a.Lq, tiles = (rows + 31) / 32;
    const int s = blockIdx.x % splits;
    const int tile = (blockIdx.x / splits) % tiles, bhk = blockIdx.x / (splits * tiles);
    const int b = bhk / a.Hk, hk = bhk % a.Hk;
    const Reach reach(a);
    const int len = key_count(a, b), p0 = first_position(a, b);
    const int r = tile * 32 + (lane & 31);
    const int rr = min(r, rows - 1), i = rr / G, hh = rr - i * G, h = hk * G + hh;
    const int pos = p0 + i;
    const int pmin = p0 + tile * 32 / G, pmax = p0 + min(a.Lq - 1, (tile * 32 + 31) / G);
    const int kend = a.causal ? min(len, pmax + 1) : len;
    // the wave's keys: equal parts of those that count, in steps of 32
    const int units = splits * 4;
    const int per = kend > 0 ? ((kend + units - 1) / units + 31) / 32 * 32 : 0;
    const int64_t first = (int64_t)(s * 4 + wave) * per;
    const int j0 = (int)(first < kend ? first : kend), j1 = j0 + per < kend ? j0 + per : kend;
    const float sl2 = a.scale * kLog2e;

    // Does any wave of the workgroup meet a block of several buckets?  (All waves decide alike.)
    const int64_t w0 = (int64_t)s * 4 * per, w1 = w0 + 4 * per < kend ? w0 + 4 * per : kend;
    if (w0 < w1 && pmin - (w1 + 31) < reach.hi && pmax - w0 > reach.lo) {
        for (int n = threadIdx.x; n < a.buckets * G; n += kThreads) {
            const int head = hk * G + n % G;
            const float v = bias_value(a, n / G, head);
            values[n] = in_log2(is_low(v) ? v - taken_off<false>(head) : v);
        }
        for (int n = threadIdx.x; n <= reach.hi - reach.lo; n += kThreads) {
            const int d = n + reach.lo;
            int k;
            buckets_of<1>(a, &d, &k);
            bucket[n] = (uint8_t)k;
        }
    }
    float bias_hi = bias_value(a, a.n_starts - 1, h), bias_lo = bias_value(a, a.causal ? 0 : 2 * a.n_starts - 1, h);

    typename X::Frag qf[HD / 16], kf[HD / 16];
    {
        const T* q = (const T*)a.q + b * a.q_sb + h * a.q_sh + (int64_t)i * a.q_sl;
#pragma unroll
        for (int c = 0; c < HD / 16; ++c) qf[c] = *reinterpret_cast<const typename X::FragMem*>(q + 16 * c + 8 * g);
    }
    const T* kbase = (const T*)a.k + b * a.k_sb + hk * a.k_sh;
    const T* vbase = (const T*)a.v + b * a.v_sb + hk * a.v_sh;
    T* vt = reinterpret_cast<T*>(corner + wave * kWaveFloats);
    f32x4 vv[kVecs];
    auto load = [&](int jb) {   // rows from the part's end on are zero
        load_frags<T, HD>(kbase, a.k_sl, jb, j1, kf);
#pragma unroll
        for (int n = 0; n < kVecs; ++n) {
            const int p = n * 64 + lane, j = jb + p / kPerRow;
            const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
            vv[n] = zero;
            if (j < j1) vv[n] = *reinterpret_cast<const f32x4*>(vbase + (int64_t)j * a.v_sl + (p % kPerRow) * kVecT);
        }
    };
    f32x16 o[HD / 32];
#pragma unroll
    for (int d = 0; d < HD / 32; ++d) o[d] = zero16();
    float m = -INFINITY, l = 0.f;
    if (j0 < j1) load(j0);
    const float off = is_low(bias_hi) || is_low(bias_lo) ? taken_off<false>(h) : 0.f;   // while these are on their way
    bias_hi = in_log2(bias_hi - off), bias_lo = in_log2(bias_lo - off);
    __syncthreads();
    for (int jb = j0; jb < j1; jb += 32) {
        f32x16 x = zero16();
#pragma unroll
        for (int c = 0; c < HD / 16; ++c) x = X::mma(kf[c], qf[c], x);
#pragma unroll
        for (int n = 0; n < kVecs; ++n) {
            const int p = n * 64 + lane;
            *reinterpret_cast<f32x4*>(vt + (p / kPerRow) * kStride + (p % kPerRow) * kVecT) = vv[n];
        }
        if (jb + 32 < j1) load(jb + 32);
        const int dlo = pmin - jb - 31, dhi = pmax - jb;
        if (dlo >= reach.hi || dhi <= reach.lo) {
            const float bias = dlo >= reach.hi ? bias_hi : bias_lo;
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = __builtin_fmaf(x[e], sl2, bias);
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int d = pos - jb - row_of(e);
                const int n = bucket[(d < reach.lo ? reach.lo : d > reach.hi ? reach.hi : d) - reach.lo];
                x[e] = __builtin_fmaf(x[e], sl2, values[n * G + hh]);
            }
        }
        if ((a.causal && dlo < 0) || jb + 32 > j1) {
            const int most = a.causal ? min(j1, pos + 1) : j1;
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (jb + row_of(e) >= most) x[e] = -INFINITY;
        }
        float top = x[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) top = fmaxf(top, x[e]);
        top = half_max(top);
        if (__any(top > m + kSlack)) {
            const float mn = fmaxf(m, top);
            const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < HD / 32; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[d][e] *= alpha;
        }
        const float mu = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            x[e] = __builtin_amdgcn_exp2f(x[e] - mu);
            l += x[e];
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const typename X::Frag p = to_frag<T>(x, c);
#pragma unroll
            for (int d = 0; d < HD / 32; ++d) {
                typename X::Frag f;
                if constexpr (sizeof(T) == 2) f = cols_bf16<kStride>(vt, 16 * c, 32 * d);
                else f = cols_f32<kStride>(vt, 16 * c, 32 * d);
                o[d] = X::mma(f, p, o[d]);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    l = half_sum(l);
    // join the four waves
    if (lane < 32) stat[wave][0][lane] = m, stat[wave][1][lane] = l;
    float* mine = corner + wave * kWaveFloats;
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) mine[(32 * d + row_of(e)) * 33 + (lane & 31)] = o[d][e];
    __syncthreads();
    const int64_t row0 = (int64_t)bhk * rows + tile * 32;
    const int count = min(32, rows - tile * 32);
    for (int n = threadIdx.x; n < count * HD; n += kThreads) {
        const int q = n / HD, d = n % HD;
        float top = -INFINITY, sum = 0.f, acc = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) top = fmaxf(top, stat[w][0][q]);
        const float mu = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = __builtin_amdgcn_exp2f(stat[w][0][q] - mu);
            sum = __builtin_fmaf(stat[w][1][q], f, sum);
            acc = __builtin_fmaf(corner[w * kWaveFloats + d * 33 + q], f, acc);
        }
        const int64_t row = row0 + q;
        if (splits > 1) {
            float* p = part + (row * splits + s) * (HD + 2);
            p[d] = acc;
            if (d == 0) p[HD] = top, p[HD + 1] = sum;
        } else {
            const int iq = (tile * 32 + q) / G, hq = hk * G + (tile * 32 + q) % G;
            ((T*)a.out)[b * a.out_sb + hq * a.out_sh + (int64_t)iq * a.out_sl + d] = (T)(sum == 0.f ? 0.f : acc / sum);   // NaN stays NaN
            if (d == 0 && a.lse)
                a.lse[((int64_t)b * a.H + hq) * a.Lq + iq] = sum == 0.f ? INFINITY : top + __builtin_amdgcn_logf(sum);
        }
    }
}

// Joins the parts of a row, the forward's runs too (bias_attn_fwd.hip): a wave a row, a lane a part for the weights, then a lane a channel.
template <typename T, int HD>
__global__ void __launch_bounds__(kThreads) bias_attn_join_kernel(const Args a, int splits, const float* __restrict__ part) {
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int G = a.H / a.Hk, rows = G * a.Lq;
    if (row >= (int64_t)a.B * a.Hk * rows) return;
    const float* p = part + row * splits * (HD + 2);
    const bool in = lane < splits;
    const float m = in ? p[lane * (HD + 2) + HD] : -INFINITY, l = in ? p[lane * (HD + 2) + HD + 1] : 0.f;
    float top = m;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    const float f = __builtin_amdgcn_exp2f(m - (top == -INFINITY ? 0.f : top));
    float sum = l * f;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, 64);
    const float w = sum == 0.f ? 0.f : f / sum;
    const int bhk = (int)(row / rows), rr = (int)(row - (int64_t)bhk * rows);
    const int b = bhk / a.Hk, h = bhk % a.Hk * G + rr % G, i = rr / G;
    T* out = (T*)a.out + b * a.out_sb + h * a.out_sh + (int64_t)i * a.out_sl;
#pragma unroll
    for (int d0 = 0; d0 < HD; d0 += 64) {
        const int d = d0 + lane;
        float acc = 0.f;
        for (int s0 = 0; s0 < splits; s0 += 8) {   // eight loads on their way together
            float x[8];
#pragma unroll
            for (int s = 0; s < 8; ++s) x[s] = s0 + s < splits && d < HD ? p[(s0 + s) * (HD + 2) + d] : 0.f;
#pragma unroll
            for (int s = 0; s < 8; ++s) acc = __builtin_fmaf(__shfl(w, s0 + s, 64), x[s], acc);
        }
        if (d < HD) out[d] = (T)acc;
    }
    if (lane == 0 && a.lse) a.lse[((int64_t)b * a.H + h) * a.Lq + i] = sum == 0.f ? INFINITY : top + __builtin_amdgcn_logf(sum);
}

template <typename T, int HD>
int join(const Args& a, int splits, const float* part, hipStream_t st) {
    const int64_t total = (int64_t)a.B * a.H * a.Lq;
    hipLaunchKernelGGL((bias_attn_join_kernel<T, HD>), dim3((unsigned)((total + 3) / 4)), dim3(kThreads), 0, st, a, splits, part);
    return check_launch("mb_bias_attn_fwd");
}

template <typename T, int HD>
int launch(const Args& a, int splits, float* part, hipStream_t st) {
    const int G = a.H / a.Hk, rows = G * a.Lq, tiles = (rows + 31) / 32;
    const int corner = std::max(HD * 33 * 4, 32 * (HD * (int)sizeof(T) + 16));
    const Reach r(a);
    const int lds = 4 * corner + a.buckets * G * 4 + (r.hi - r.lo + 1);
    static Told told;
    if (const int rc = allow_lds((const void*)bias_attn_split_kernel<T, HD>, lds, told)) return rc;
    hipLaunchKernelGGL((bias_attn_split_kernel<T, HD>), dim3((unsigned)(a.B * a.Hk * tiles * splits)), dim3(kThreads), lds, st,
                       a, splits, part);
    if (splits > 1) return join<T, HD>(a, splits, part, st);
    return check_launch("mb_bias_attn_fwd");
}

}  // namespace

int split_launch(const Args& a, int hd, int dtype, int splits, void* part, hipStream_t st) {
    float* p = (float*)part;
    if (dtype == MB_DTYPE_F32)
        return hd == 32 ? launch<float, 32>(a, splits, p, st) : hd == 64 ? launch<float, 64>(a, splits, p, st) : launch<float, 128>(a, splits, p, st);
    return hd == 32 ? launch<__bf16, 32>(a, splits, p, st) : hd == 64 ? launch<__bf16, 64>(a, splits, p, st) : launch<__bf16, 128>(a, splits, p, st);
}

int join_launch(const Args& a, int hd, int dtype, int splits, const void* part, hipStream_t st) {
    const float* p = (const float*)part;
    if (dtype == MB_DTYPE_F32) return hd == 32 ? join<float, 32>(a, splits, p, st) : hd == 64 ? join<float, 64>(a, splits, p, st) : join<float, 128>(a, splits, p, st);
    return hd == 32 ? join<__bf16, 32>(a, splits, p, st) : hd == 64 ? join<__bf16, 64>(a, splits, p, st) : join<__bf16, 128>(a, splits, p, st);
}

}  // namespace battn
}  // namespace mb
