// The argument checks that the attention's entry points share (host side).
#pragma once

#include "bias_attn.h"

namespace mb {
namespace battn {

// A workgroup may use 160 KiB of LDS; beyond 64 KiB the kernel has to be told.
inline int allow_lds(const void* kernel, int bytes) {
    if (bytes <= 65536) return MB_OK;
    if (bytes > 163840) return fail(MB_ERR_UNSUPPORTED, "mb_bias_attn: %d bytes of LDS are wanted, 163840 are there", bytes);
    const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) return fail((int)e, "mb_bias_attn: %d bytes of LDS: %s", bytes, hipGetErrorString(e));
    return MB_OK;
}

inline bool rows16(const void* p, const int64_t* st, int dtype) {
    const int64_t size = dtype == MB_DTYPE_F32 ? 4 : 2;
    return (((uint64_t)(uintptr_t)p | (uint64_t)(st[0] * size) | (uint64_t)(st[1] * size) | (uint64_t)(st[2] * size)) & 15) == 0;
}

// Parts that the keys of a row are split into (bias_attn_split.hip), or 0 for the kernel whose
// workgroups walk all keys for 128 queries of a head.  The latter leaves CUs idle where its grid is
// small, and its longest workgroup takes 1.2 us (heads of 128: 1.5) for every 64 keys; the former
// takes about 8 us to start and join, and 1.6 ns (3.5) for every 32 queries by 32 keys.  The one is
// the shorter where the pairs that a mask leaves fill less than about 80 (40) workgroups and the
// keys are not few.  Measured in bf16, split against not: 1 x 2048, 8 heads x 64 35 us against 42, 2 x
// 2048 53 against 42, 1 x 512 17 against 21, 8 x 128 15 against 13; 8 heads x 128: 1 x 1024 41
// against 31, 1 x 2048 75 against 50, 4 x 128 queries of 4096 keys 54 against 90.  Up to 32 rows for a key head are one column
// block of the split kernel (16 x 1 of 4096, 8 heads x 64: 27 us against 97).
inline int splits_of(int B, int H, int Hk, int Lq, int Lk, int hd, int causal) {
    const int64_t G = H / Hk, tiles = (G * Lq + 31) / 32, nq = ((int64_t)Lq + kRows - 1) / kRows;
    if (G > 32 || (double)B * Hk * tiles > 0x7fffffff / 64) return 0;
    if (G * Lq > 32) {
        // a causal mask leaves Lk - Lq / 2 of Lk keys where the last query sees them all
        const double share = causal && Lk > 0 ? 1.0 - 0.5 * (Lq < Lk ? Lq : Lk) / Lk : 1.0;
        if (Lk < (hd == 128 ? 2048 : 512) || (double)B * H * nq * share > (hd == 128 ? 40.0 : 80.0)) return 0;
    }
    const int64_t wanted = (hd == 128 ? 512 : 768) / ((int64_t)B * Hk * tiles);  // two or three workgroups a CU
    const int64_t most = ((int64_t)Lk + 511) / 512;                              // at least 128 keys a wave
    const int64_t n = wanted < most ? wanted : most;
    return (int)(n < 1 ? 1 : n > 64 ? 64 : n);
}
int split_launch(const Args& a, int hd, int dtype, int splits, void* part, hipStream_t st);

inline int fill_args(const char* what, Args& a, const void* q, const int64_t* q_st, const void* k, const int64_t* k_st,
                     const void* v, const int64_t* v_st, const void* bias, int bias_dtype, int buckets,
                     const int32_t* starts, int n_starts, const void* lengths, int lengths_bytes, const void* q_start,
                     int q_start_bytes, int64_t q_start0, int B, int H, int Hk, int Lq, int Lk, int hd, float scale,
                     int causal, int dtype) {
    MB_REQUIRE(B >= 0 && Lq >= 0 && Lk >= 0 && H >= 1 && Hk >= 1, "%s: B=%d H=%d Hk=%d Lq=%d Lk=%d", what, B, H, Hk, Lq, Lk);
    MB_REQUIRE(H % Hk == 0, "%s: H=%d is not a multiple of Hk=%d", what, H, Hk);
    if (hd != 32 && hd != 64 && hd != 128)
        return fail(MB_ERR_UNSUPPORTED, "%s: head_dim=%d (supported: 32, 64, 128)", what, hd);
    MB_REQUIRE(dtype == MB_DTYPE_F32 || dtype == MB_DTYPE_BF16, "%s: dtype=%d", what, dtype);
    MB_REQUIRE(bias_dtype == MB_DTYPE_F32 || bias_dtype == MB_DTYPE_BF16, "%s: bias_dtype=%d", what, bias_dtype);
    MB_REQUIRE(scale > 0.f && scale < INFINITY, "%s: scale=%g", what, (double)scale);
    MB_REQUIRE(starts && n_starts >= 1 && buckets == (causal ? n_starts : 2 * n_starts),
               "%s: %d buckets for %d first distances", what, buckets, n_starts);
    if (n_starts > kMaxStarts)
        return fail(MB_ERR_UNSUPPORTED, "%s: %d buckets in a direction (at most %d)", what, n_starts, kMaxStarts);
    MB_REQUIRE(starts[0] == 0, "%s: the first bucket begins at distance %d, not at 0", what, starts[0]);
    for (int i = 1; i < n_starts; ++i)
        MB_REQUIRE(starts[i] >= starts[i - 1], "%s: first distances must not fall", what);
    if (starts[n_starts - 1] > kMaxReach)
        return fail(MB_ERR_UNSUPPORTED, "%s: the last bucket begins at distance %d (at most %d)", what, starts[n_starts - 1], kMaxReach);
    MB_REQUIRE((!lengths || lengths_bytes == 4 || lengths_bytes == 8) && (!q_start || q_start_bytes == 4 || q_start_bytes == 8),
               "%s: lengths and q_start hold integers of 4 or 8 bytes", what);
    MB_REQUIRE(q_start || (q_start0 >= -(1 << 30) && q_start0 <= (1 << 30)), "%s: q_start=%lld", what, (long long)q_start0);
    MB_REQUIRE(Lq <= (1 << 30) && Lk <= (1 << 30), "%s: Lq=%d Lk=%d", what, Lq, Lk);
    const int64_t nq = ((int64_t)Lq + kRows - 1) / kRows;
    MB_REQUIRE((int64_t)B * H * (nq > 0 ? nq : 1) <= 0x7fffffff && (int64_t)B * Hk * (((int64_t)Lk + kRows - 1) / kRows) <= 0x7fffffff,
               "%s: B=%d H=%d Lq=%d Lk=%d are too many", what, B, H, Lq, Lk);
    if (B > 0 && Lq > 0) MB_REQUIRE(q && q_st && bias, "%s: null pointer argument", what);
    if (B > 0 && Lk > 0) MB_REQUIRE(k && k_st && v && v_st, "%s: null pointer argument", what);
    if (B > 0 && Lq > 0) MB_REQUIRE(rows16(q, q_st, dtype), "%s: q's rows must begin at multiples of 16 bytes", what);
    if (B > 0 && Lk > 0)
        MB_REQUIRE(rows16(k, k_st, dtype) && rows16(v, v_st, dtype), "%s: k's and v's rows must begin at multiples of 16 bytes", what);
    // offsets within a tile of 64 rows have 32 bits
    const int64_t most = (int64_t)(1 << 24) / (dtype == MB_DTYPE_F32 ? 4 : 2);
    if (B > 0 && Lq > 0) MB_REQUIRE(q_st[2] >= 0 && q_st[2] <= most, "%s: q's rows are %lld elements apart", what, (long long)q_st[2]);
    if (B > 0 && Lk > 0)
        MB_REQUIRE(k_st[2] >= 0 && k_st[2] <= most && v_st[2] >= 0 && v_st[2] <= most,
                   "%s: k's and v's rows are %lld and %lld elements apart", what, (long long)k_st[2], (long long)v_st[2]);
    a.q = q, a.k = k, a.v = v, a.bias = bias;
    if (q_st) a.q_sb = q_st[0], a.q_sh = q_st[1], a.q_sl = q_st[2];
    if (k_st) a.k_sb = k_st[0], a.k_sh = k_st[1], a.k_sl = k_st[2];
    if (v_st) a.v_sb = v_st[0], a.v_sh = v_st[1], a.v_sl = v_st[2];
    a.lengths = lengths, a.lengths_bytes = lengths_bytes;
    a.start = q_start, a.start_bytes = q_start_bytes, a.start0 = (int)q_start0;
    a.B = B, a.H = H, a.Hk = Hk, a.Lq = Lq, a.Lk = Lk, a.nq = (int)nq;
    a.causal = causal != 0, a.bias_bf16 = bias_dtype == MB_DTYPE_BF16, a.buckets = buckets, a.n_starts = n_starts;
    a.reach = starts[n_starts - 1];
    a.scale = scale;
    for (int i = 0; i < n_starts; ++i) a.starts[i] = (int16_t)starts[i];
    return MB_OK;
}

}  // namespace battn
}  // namespace mb
