// The argument checks that the attention's entry points share (host side).
#pragma once

#include "bias_attn.h"

#include <atomic>

namespace mb {
namespace battn {

// A workgroup may use 160 KiB of LDS; beyond 64 KiB, of which a few are the kernels' static arrays, a
// kernel has to be told, once on each device.  `told` is the kernel's own.
struct Told {
    std::atomic<int> bytes[64] = {};
};
inline int allow_lds(const void* kernel, int bytes, Told& told) {
    if (bytes <= 61440) return MB_OK;
    if (bytes > 163840) return fail(MB_ERR_UNSUPPORTED, "mb_bias_attn: %d bytes of LDS are wanted, 163840 are there", bytes);
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e == hipSuccess && dev < 64 && told.bytes[dev].load(std::memory_order_relaxed) >= bytes) return MB_OK;
    if (e == hipSuccess) e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) return fail((int)e, "mb_bias_attn: %d bytes of LDS: %s", bytes, hipGetErrorString(e));
    if (dev < 64) told.bytes[dev].store(bytes, std::memory_order_relaxed);
    return MB_OK;
}

constexpr int kMostGroups = 0xffffff;   // of a launch, whose threads are counted in 32 bits

inline bool rows16(const void* p, const int64_t* st, int dtype) {
    const int64_t size = dtype == MB_DTYPE_F32 ? 4 : 2;
    return (((uint64_t)(uintptr_t)p | (uint64_t)(st[0] * size) | (uint64_t)(st[1] * size) | (uint64_t)(st[2] * size)) & 15) == 0;
}

// Parts that the keys of a row are split into (bias_attn_split.hip), or 0 for the kernel whose
// workgroups walk all keys for 128 queries of a head.  The latter leaves CUs idle where its grid is
// small, and its time is that of its longest walk; the former takes a few us more to start and
// join, and a time that grows with the pairs.  The one is the shorter where the pairs that a mask
// leaves fill few workgroups and the keys are many.  Measured in bf16 in a captured graph, split against not, 8 heads:
// of 64: 1 x 1024 15 us against 17, 1 x 2048 30 against 27, 4 x 128 queries of 4096 keys 32 against 46, 1 x 256 of 4096
// 18 against 45; of 128: 1 x 2048 71 against 37, 4 x 128 of 4096 50 against 64; of 32: 1 x 2048 21 against 23.  Up to
// 32 rows for a key head are one column block of the split kernel: 16 x 1 of 4096, 8 heads x 64, 29 us against 44, in
// fp32, for which the number of parts was not fitted, 67 against 75 (with 4 parts instead of 6: 58).
inline int splits_of(int B, int H, int Hk, int Lq, int Lk, int hd, int causal) {
    const int64_t G = H / Hk, tiles = (G * Lq + 31) / 32, nq = ((int64_t)Lq + kRows - 1) / kRows;
    if (G > 32 || (double)B * Hk * tiles > kMostGroups) return 0;
    if (G * Lq > 32) {
        // a causal mask leaves Lk - Lq / 2 of Lk keys where the last query sees them all
        const double share = causal && Lk > 0 ? 1.0 - 0.5 * (Lq < Lk ? Lq : Lk) / Lk : 1.0;
        const double most = hd == 128 ? 40.0 : hd == 64 ? 52.0 : 70.0;
        if (Lk <= 400 || (double)B * H * nq * share > most * (1.0 - 400.0 / Lk)) return 0;
    }
    const int64_t wanted = (hd == 128 ? 512 : 768) / ((int64_t)B * Hk * tiles);  // two or three workgroups a CU
    const int64_t most = ((int64_t)Lk + 511) / 512;                              // at least 128 keys a wave
    const int64_t n = wanted < most ? wanted : most;
    return (int)(n < 1 ? 1 : n > 64 ? 64 : n);
}
int split_launch(const Args& a, int hd, int dtype, int splits, void* part, hipStream_t st);
// o and lse from parts [B, Hk, Lq, H / Hk, splits, hd + 2] of rows: sums of p v, the maximum, the sum of p.
int join_launch(const Args& a, int hd, int dtype, int splits, const void* part, hipStream_t st);

// Checks what both directions take and fills the kernels' arguments; 0 or an error code.
inline int fill_args(const char* what, const mb_bias_attn* p, Args& a) {
    MB_REQUIRE(p, "%s: null args", what);
    const int64_t top = kFarthest;
    MB_REQUIRE(p->B >= 0 && p->B <= top && p->Lq >= 0 && p->Lq <= top && p->Lk >= 0 && p->Lk <= top && p->H >= 1 && p->H <= top
                   && p->Hk >= 1 && p->Hk <= top,
               "%s: B=%lld H=%lld Hk=%lld Lq=%lld Lk=%lld", what, (long long)p->B, (long long)p->H, (long long)p->Hk,
               (long long)p->Lq, (long long)p->Lk);
    MB_REQUIRE(p->H % p->Hk == 0, "%s: H=%lld is not a multiple of Hk=%lld", what, (long long)p->H, (long long)p->Hk);
    if (p->hd != 32 && p->hd != 64 && p->hd != 128)
        return fail(MB_ERR_UNSUPPORTED, "%s: head_dim=%lld (supported: 32, 64, 128)", what, (long long)p->hd);
    MB_REQUIRE(p->dtype == MB_DTYPE_F32 || p->dtype == MB_DTYPE_BF16, "%s: dtype=%lld", what, (long long)p->dtype);
    MB_REQUIRE(p->bias_dtype == MB_DTYPE_F32 || p->bias_dtype == MB_DTYPE_BF16, "%s: bias_dtype=%lld", what, (long long)p->bias_dtype);
    MB_REQUIRE(p->scale >= 1e-20 && p->scale <= 1e20, "%s: scale=%g (1e-20 to 1e20)", what, p->scale);
    MB_REQUIRE(p->starts && p->n_starts >= 1 && p->buckets == (p->causal ? p->n_starts : 2 * p->n_starts),
               "%s: %lld buckets for %lld first distances", what, (long long)p->buckets, (long long)p->n_starts);
    if (p->n_starts > kMaxStarts)
        return fail(MB_ERR_UNSUPPORTED, "%s: %lld buckets in a direction (at most %d)", what, (long long)p->n_starts, kMaxStarts);
    const int32_t* starts = p->starts;
    const int n_starts = (int)p->n_starts;
    MB_REQUIRE(starts[0] == 0, "%s: the first bucket begins at distance %d, not at 0", what, starts[0]);
    for (int i = 1; i < n_starts; ++i)
        MB_REQUIRE(starts[i] >= starts[i - 1] && starts[i] > 0, "%s: first distances must not fall, and one alone is 0", what);
    if (starts[n_starts - 1] > kMaxReach)
        return fail(MB_ERR_UNSUPPORTED, "%s: the last bucket begins at distance %d (at most %d)", what, starts[n_starts - 1], kMaxReach);
    MB_REQUIRE((!p->lengths || p->lengths_bytes == 4 || p->lengths_bytes == 8)
                   && (!p->q_start || p->q_start_bytes == 4 || p->q_start_bytes == 8),
               "%s: lengths and q_start hold integers of 4 or 8 bytes", what);
    MB_REQUIRE(p->q_start || (p->q_start0 >= -top && p->q_start0 <= top), "%s: q_start=%lld", what, (long long)p->q_start0);
    const int64_t nq = (p->Lq + kRows - 1) / kRows, nk = (p->Lk + kRows - 1) / kRows;
    MB_REQUIRE((double)p->B * p->H * (nq > 0 ? nq : 1) <= kMostGroups && (double)p->B * p->Hk * nk + p->H <= kMostGroups,
               "%s: B=%lld H=%lld Lq=%lld Lk=%lld are too many", what, (long long)p->B, (long long)p->H, (long long)p->Lq,
               (long long)p->Lk);
    const int dtype = (int)p->dtype;
    const int64_t most = (int64_t)(1 << 24) / (dtype == MB_DTYPE_F32 ? 4 : 2);   // offsets within a tile have 32 bits
    if (p->B > 0 && p->Lq > 0) {
        MB_REQUIRE(p->q && p->bias, "%s: null pointer argument", what);
        MB_REQUIRE(rows16(p->q, p->q_st, dtype), "%s: q's rows must begin at multiples of 16 bytes", what);
        MB_REQUIRE(p->q_st[2] >= 0 && p->q_st[2] <= most, "%s: q's rows are %lld elements apart", what, (long long)p->q_st[2]);
    }
    if (p->B > 0 && p->Lk > 0) {
        MB_REQUIRE(p->k && p->v, "%s: null pointer argument", what);
        MB_REQUIRE(rows16(p->k, p->k_st, dtype) && rows16(p->v, p->v_st, dtype), "%s: k's and v's rows must begin at multiples of 16 bytes", what);
        MB_REQUIRE(p->k_st[2] >= 0 && p->k_st[2] <= most && p->v_st[2] >= 0 && p->v_st[2] <= most,
                   "%s: k's and v's rows are %lld and %lld elements apart", what, (long long)p->k_st[2], (long long)p->v_st[2]);
    }
    a.q = p->q, a.k = p->k, a.v = p->v, a.bias = p->bias;
    a.q_sb = p->q_st[0], a.q_sh = p->q_st[1], a.q_sl = p->q_st[2];
    a.k_sb = p->k_st[0], a.k_sh = p->k_st[1], a.k_sl = p->k_st[2];
    a.v_sb = p->v_st[0], a.v_sh = p->v_st[1], a.v_sl = p->v_st[2];
    a.lengths = p->lengths, a.lengths_bytes = (int)p->lengths_bytes;
    a.start = p->q_start, a.start_bytes = (int)p->q_start_bytes, a.start0 = p->q_start ? 0 : (int)p->q_start0;
    a.B = (int)p->B, a.H = (int)p->H, a.Hk = (int)p->Hk, a.Lq = (int)p->Lq, a.Lk = (int)p->Lk, a.nq = (int)nq;
    a.causal = p->causal != 0, a.bias_bf16 = p->bias_dtype == MB_DTYPE_BF16, a.buckets = (int)p->buckets, a.n_starts = n_starts;
    a.reach = starts[n_starts - 1];
    a.scale = (float)p->scale;
    for (int i = 0; i < kMaxStarts; ++i) a.starts[i] = i < n_starts ? starts[i] : 0x7fffffff;
    return MB_OK;
}

}  // namespace battn
}  // namespace mb
