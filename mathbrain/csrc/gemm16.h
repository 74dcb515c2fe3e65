// Products of matrices held in 16-bit planes, for the kernels that fuse something around them.
//
//   acc[p][q] = sum_k P[p][k] Q[q][k],  fp32 accumulation in the 32 x 32 x 16 matrix instructions
//
// One plane: bf16 or fp16 values.  Two planes: fp32 values as x = hi + lo, both fp16 (24 bits down
// to 2^-16 of the largest value, see below), from three products lo hi + hi lo + hi hi; the fourth is
// below fp32's own rounding.
//
// A workgroup of four or eight waves takes a TP x TQ tile of the result and walks k in steps of 32 or 64.  Operand tiles go
// from memory straight into LDS, kStages - 1 steps ahead, 16 bytes a lane.  Such a
// load puts its 64 pieces next to each other, so a row has no padding; piece c of row r lies in the
// place c ^ swz(r) instead, which spreads the reads over the banks.  An operand may have its k next to
// each other (kRows) or its free index (kCols: read back by the transposing 16-bit LDS read).
//
// Buffers are padded: kRows operands have whole steps of k (zeros behind the matrix on one side at
// least), kCols operands whole steps of rows and rows of a multiple of 8 elements.  Tiles that pass
// the free index's end read the last rows (or pieces) again; whoever uses acc leaves those out.
//
// What bounds it: power first (under such load the clock falls to 1.6 - 1.85 GHz), then the loads into LDS.  8192^3 in tiles of
// 256 x 256 takes 955 - 1013 us, 1085 - 1150 TFLOP/s; its loads alone take 765 us, its instructions 560, its LDS reads 270.
// kRows operands load best in whole lines of 128 bytes, steps of 64 (out of the L2: 382 us against 540 and more).
//
// A lane holds, of each 32 x 32 block, column q = lane % 32 and the rows p = 8 (r / 4) + 4 (lane / 32) + r % 4.
#pragma once

#include "lds_dma.h"

#include <atomic>
#include <type_traits>

namespace mb {
namespace g16 {

constexpr int kPad = 64;        // what k is padded to: a step of any of the products

typedef __attribute__((__ext_vector_type__(8))) _Float16 f16x8;
typedef __attribute__((__ext_vector_type__(4))) _Float16 f16x4;
typedef __attribute__((__ext_vector_type__(8))) __bf16 bf16x8;
typedef __attribute__((__ext_vector_type__(4))) short s16x4;
typedef __attribute__((__ext_vector_type__(8))) short s16x8;
typedef __attribute__((__ext_vector_type__(16))) float f32x16;

enum Order { kRows, kCols };

// One operand: element (i, k) of a plane at p + i * ld + k (kRows) or p + k * ld + i (kCols).
struct Side {
    const void* p;
    int64_t plane;   // bytes from the first plane (hi) to the second (lo)
    int64_t ld;      // elements
    int n;           // free indices that are there (at least 1)
};

__device__ inline f32x16 mma(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ inline f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
template <typename T>
struct Frag;
template <>
struct Frag<_Float16> { typedef f16x8 type; };
template <>
struct Frag<__bf16> { typedef bf16x8 type; };

// A value that is the same in all lanes, where the compiler cannot see that.
__device__ inline int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
template <typename T>
__device__ inline T* uniform(T* p) {
    const uint64_t x = (uint64_t)p;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x), hi = __builtin_amdgcn_readfirstlane((uint32_t)(x >> 32));
    return (T*)((uint64_t)hi << 32 | lo);
}
__device__ inline int64_t uniform(int64_t x) { return (int64_t)uniform((char*)x); }
__device__ inline Side uniform(const Side& s) { return {uniform((char*)s.p), uniform(s.plane), uniform(s.ld), uniform(s.n)}; }

// A tile of N free indices by STEP k in LDS.
template <typename T, int N, Order ORDER, int STEP, int THREADS>
struct Tile {
    static constexpr int kStep = STEP;
    static constexpr int kBytes = N * kStep * 2;
    static constexpr int kLoads = kBytes / (THREADS * 16);          // of each wave
    static constexpr int kRow = ORDER == kRows ? kStep * 2 : N * 2; // bytes
    static constexpr int kPieces = kRow / 16;
    static_assert(kBytes % (THREADS * 16) == 0 && N % 64 == 0 && STEP % 32 == 0, "a wave's load moves 1 KiB");
    typedef __attribute__((address_space(3))) const char lds_char;

    static __device__ constexpr int swz(int row) {
        if (kPieces == 4) return (row >> 2) & 3;
        if (kPieces == 8) return ((row >> 1) & 1) << 2 | ((row >> 3) & 1) << 1 | ((row >> 2) & 1);
        return (row & 3) << 2 | ((row >> 2) & 3);
    }
    // This lane's offset of each of its wave's loads, from the tile's first element; i0 is the tile's first
    // free index.
    struct Offsets {
        uint32_t v[kLoads];
        __device__ Offsets(const Side& s, int i0) {
            const int left = s.n - 1 - i0;
            const int last = ORDER == kRows ? left : (int)(s.ld - 8) - i0;
#pragma unroll
            for (int j = 0; j < kLoads; ++j) {
                const int slot = j * THREADS + (int)threadIdx.x, row = slot / kPieces;
                const int piece = (slot % kPieces) ^ swz(row);
                if (ORDER == kRows) v[j] = (uint32_t)(min(row, last) * (int64_t)s.ld * 2) + piece * 16;
                else v[j] = (uint32_t)(row * s.ld * 2) + min(piece * 8, last) * 2;
            }
        }
    };
    static __device__ void load(uint32_t tile, int j, const char* base, const Offsets& off) {
        dma16(tile + wave_id() * 1024 + j * THREADS * 16, off.v[j], base);
    }
    // Bytes from the matrix's first element to the tile's.
    static __device__ int64_t at(const Side& s, int i0, int k0) {
        return (ORDER == kRows ? i0 * s.ld + k0 : (int64_t)k0 * s.ld + i0) * 2;
    }
    // Where this lane reads within a tile: the fragment of free indices i0 + lane % 32 (i0 a multiple of 32) and
    // k = 16 c + 8 (lane / 32) + 0 .. 7.
    struct Lane {
        uint32_t v[ORDER == kRows ? STEP / 16 : STEP / 8];
        __device__ Lane() {
            const int lane = threadIdx.x & 63, g = lane >> 5;
            if (ORDER == kRows) {
#pragma unroll
                for (int c = 0; c < STEP / 16; ++c) v[c] = (lane & 31) * kRow + (((2 * c + g) ^ swz(lane & 31)) << 4);
            } else {
                // 16 lanes read 4 rows of 16 free indices, 8 bytes each, and get 4 rows of one index each
                const int d = (lane & 16) + 4 * (lane & 3);
#pragma unroll
                for (int c = 0; c < STEP / 8; ++c) {
                    const int r = 16 * (c / 2) + 8 * g + 4 * (c % 2) + ((lane & 15) >> 2);
                    v[c] = r * kRow + (((d >> 3) ^ swz(r)) << 4) + 2 * (d & 7);
                }
            }
        }
    };
    // Four values of free indices i .. i + 3 (i a multiple of 4) at k of a kCols tile.
    typedef T four_t __attribute__((ext_vector_type(4)));
    static __device__ four_t four(uint32_t tile, int i, int k) {
        static_assert(ORDER == kCols, "");
        return *(__attribute__((address_space(3))) const four_t*)(uintptr_t)(tile + k * kRow + (((i >> 3) ^ swz(k)) << 4) + 2 * (i & 7));
    }
    static __device__ typename Frag<T>::type read(uint32_t tile, const Lane& l, int i0, int c) {
        typedef typename Frag<T>::type F;
        if constexpr (ORDER == kRows) {
            return *(__attribute__((address_space(3))) const F*)((lds_char*)(uintptr_t)(tile + l.v[c]) + i0 * kRow);
        } else {
            typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
            // 32 indices further, piece n becomes n ^ 4
            const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(lds_char*)(uintptr_t)(tile + (l.v[2 * c] ^ (i0 * 2))));
            const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(lds_char*)(uintptr_t)(tile + (l.v[2 * c + 1] ^ (i0 * 2))));
            return __builtin_bit_cast(F, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
};

// NP x NQ waves, each with TP / NP x TQ / NQ of the tile.
template <typename T_, int PLANES, int TP_, int TQ_, Order OP, Order OQ, int NP = 2, int NQ = 2, int STEP = 32>
struct Product {
    typedef T_ T;
    static constexpr int kThreads = 64 * NP * NQ, kStep = STEP;
    static constexpr int TP = TP_, TQ = TQ_;
    static constexpr int WP = TP / NP, WQ = TQ / NQ;   // of a wave
    static constexpr int FP = WP / 32, FQ = WQ / 32;   // its 32 x 32 blocks
    static constexpr int kWavesP = NP;
    typedef Tile<T, TP, OP, STEP, kThreads> TileP;
    typedef Tile<T, TQ, OQ, STEP, kThreads> TileQ;
    static constexpr int kStage = PLANES * (TileP::kBytes + TileQ::kBytes);
    // Two waves a SIMD: two workgroups of four waves a CU, or one of eight.  One wave with twice the block (128 x 128) reads LDS
    // less and stalls more: 8192^3 in tiles of 256 x 256 1013 TFLOP/s with four waves, 1085 - 1116 with eight.
    static constexpr int kWaves = 2;
    static_assert(FP * FQ <= 8, "results and two sets of operands in 256 registers");
    static constexpr int kRoom = 163840 * kThreads / 512;     // bytes of LDS
    // Whether the waves meet before a step's last instructions, with the next step's first fragments on their way during
    // these: with eight waves in one workgroup all wait at the same time (8192^3, 256 x 256: 1146 TFLOP/s against 1120),
    // with two workgroups a CU the one works while the other waits (256 x 128: 1114 against 1081 with this).
    static constexpr bool kAhead = kThreads > 256;
    static constexpr int kStages = kRoom / kStage < 3 ? kRoom / kStage : 3;
    static_assert(kStages >= 2, "a step's operands on their way beside the one in use");
    static constexpr int kLds = kStages * kStage;
    static constexpr int kLoads = PLANES * (TileP::kLoads + TileQ::kLoads);

    f32x16 acc[FP][FQ];

    __device__ static int wave_p() { return wave_id() % NP * WP; }
    __device__ static int wave_q() { return wave_id() / NP * WQ; }
    // the row within the tile of element r of block i, the column of block j
    __device__ static int row(int i, int r) {
        return wave_p() + 32 * i + 8 * (r / 4) + 4 * ((threadIdx.x & 63) >> 5) + r % 4;
    }
    __device__ static int col(int j) { return wave_q() + 32 * j + (threadIdx.x & 31); }

    __device__ void clear() {
#pragma unroll
        for (int i = 0; i < FP; ++i)
#pragma unroll
            for (int j = 0; j < FQ; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    }

    struct Frags {
        typename Frag<T>::type a[PLANES][FP], b[PLANES][FQ];
    };

    // k from k0 to k1, multiples of kStep (k1 > k0).  All waves have to be here; LDS is free again after the next barrier.
    // peek(k, tile) sees every step's operands in LDS (P's planes, then Q's) while they are there.
    __device__ void run(const Side& p, const Side& q, int p0, int q0, int k0, int k1, void* smem) {
        run(p, q, p0, q0, k0, k1, smem, [](int, uint32_t) {});
    }
    template <typename F>
    __device__ void run(const Side& p_, const Side& q_, int p0, int q0, int k0, int k1, void* smem, F peek) {
        const uint32_t lds = lds_address(smem);
        const Side p = uniform(p_), q = uniform(q_);
        p0 = uniform(p0), q0 = uniform(q0), k0 = uniform(k0);
        const typename TileP::Offsets po(p, p0);
        const typename TileQ::Offsets qo(q, q0);
        const typename TileP::Lane pl;
        const typename TileQ::Lane ql;
        const char* pb = (const char*)p.p + TileP::at(p, p0, k0);
        const char* qb = (const char*)q.p + TileQ::at(q, q0, k0);
        const int64_t pstep = TileP::at(p, 0, kStep), qstep = TileQ::at(q, 0, kStep);
        const int steps = uniform((k1 - k0) / kStep);
        // A wave with a single block has two results, of alternate instructions, added at the end: each instruction would
        // wait for the one before.
        constexpr bool kTwo = FP * FQ == 1;
        f32x16 second = {};
        // load n of the wave's for a step
        auto load = [&](uint32_t tile, int n) {
            constexpr int all = PLANES * TileP::kLoads;
            if (n < all) TileP::load(tile + n / TileP::kLoads * TileP::kBytes, n % TileP::kLoads, pb + n / TileP::kLoads * p.plane, po);
            else TileQ::load(tile + PLANES * TileP::kBytes + (n - all) / TileQ::kLoads * TileQ::kBytes, (n - all) % TileQ::kLoads,
                             qb + (n - all) / TileQ::kLoads * q.plane, qo);
        };
        auto stage = [&](int t) { return lds + t % kStages * kStage; };
        clear();
        __builtin_amdgcn_s_waitcnt(0x0F70);   // the compiler's own loads are done: it would wait for the DMA with them
        for (int t = 0; t < kStages - 1 && t < steps; ++t) {
#pragma unroll
            for (int n = 0; n < kLoads; ++n) load(stage(t), n);
            pb += pstep, qb += qstep;
        }
        auto read = [&](Frags& x, uint32_t ptile, int c) {
            const uint32_t qtile = ptile + PLANES * TileP::kBytes;
#pragma unroll
            for (int h = 0; h < PLANES; ++h) {
#pragma unroll
                for (int j = 0; j < FQ; ++j) x.b[h][j] = TileQ::read(qtile + h * TileQ::kBytes, ql, wave_q() + 32 * j, c);
#pragma unroll
                for (int i = 0; i < FP; ++i) x.a[h][i] = TileP::read(ptile + h * TileP::kBytes, pl, wave_p() + 32 * i, c);
            }
        };
        // A step: fragments come out of LDS one k of 16 ahead of the instructions that use them.  The loads for a later
        // step go out between the instructions, a few at a time: a wave that sends all of them at once waits for the
        // others' before it can go on.
        Frags f[2];
        auto step = [&](int t, auto more, auto last) {
            constexpr int C = STEP / 16, kProducts = PLANES == 2 ? 3 : 1, kGroups = (kAhead ? C - 1 : C) * kProducts * FP;
            const uint32_t to = stage(t + kStages - 1);
            if constexpr (!kAhead) {
                wait_and_meet<decltype(more)::value ? (kStages - 2) * kLoads : 0>();
                read(f[0], stage(t), 0);
            }
            peek(k0 + t * kStep, stage(t));
#pragma unroll
            for (int c = 0; c < C; ++c) {
                if (c + 1 < C) {
                    read(f[(c + 1) % 2], stage(t), c + 1);
                } else if constexpr (kAhead && !decltype(last)::value) {
                    wait_and_meet<decltype(more)::value ? (kStages - 2) * kLoads : 0>();
                    read(f[0], stage(t + 1), 0);
                }
                __builtin_amdgcn_sched_barrier(0);
                const Frags& x = f[c % 2];
#pragma unroll
                for (int k = 3 - kProducts; k < 3; ++k)   // lo hi, hi lo, hi hi
#pragma unroll
                    for (int i = 0; i < FP; ++i) {
#pragma unroll
                        for (int j = 0; j < FQ; ++j) {
                            f32x16& to_ = kTwo && (c * kProducts + k) % 2 ? second : acc[i][j];
                            to_ = mma(x.a[k == 0][i], x.b[k == 1][j], to_);
                        }
                        const int g = (c * kProducts + k - 3 + kProducts) * FP + i;
                        if constexpr (decltype(more)::value) {
#pragma unroll
                            for (int n = g * kLoads / kGroups; g < kGroups && n < (g + 1) * kLoads / kGroups; ++n) load(to, n);
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
            }
            if constexpr (decltype(more)::value) pb += pstep, qb += qstep;
        };
        if constexpr (kAhead) {
            if (steps >= kStages - 1) wait_and_meet<(kStages - 2) * kLoads>();
            else wait_and_meet<0>();
            read(f[0], stage(0), 0);
        }
        int t = 0;
        for (; t + kStages - 1 < steps; ++t) step(t, std::true_type(), std::false_type());
        for (; t + 1 < steps; ++t) step(t, std::false_type(), std::false_type());
        step(t, std::false_type(), std::true_type());
        if constexpr (kTwo) acc[0][0] += second;
    }

    // The result as 16-bit values next to each other in p, by way of LDS: a lane's own four of a row would go out in 32
    // pieces of 16 bytes an instruction.  held() is a lane's place there for its elements r .. r + 3 of a block, to be written
    // after a barrier; store() takes a whole tile out, 16 bytes a lane, rows of q (q0 + r < q_end) and pieces of 8 p
    // (p_end a multiple of 8) that are there, fetch() brings one in.
    static constexpr int kOutPieces = TP / 8;
    static constexpr int kOutTurn = kOutPieces % 16 == 0 ? 15 : 7;
    static constexpr int kOutPlane = TP * TQ * 2;
    __device__ static int out_at(int plane, int q, int piece) {
        return plane * kOutPlane + q * (2 * TP) + ((piece ^ (q & kOutTurn)) << 4);
    }
    __device__ static f16x4& held(void* smem, int plane, int i, int j, int r) {
        const int half = (threadIdx.x & 63) >> 5;
        return *(f16x4*)((char*)smem + out_at(plane, col(j), (wave_p() + 32 * i + 8 * (r / 4)) / 8) + half * 8);
    }
    __device__ static void store(const void* smem, int plane, _Float16* out, int64_t ld, int p0, int q0, int p_end, int q_end) {
#pragma unroll 4
        for (int n = threadIdx.x; n < TQ * kOutPieces; n += kThreads) {
            const int q = n / kOutPieces, piece = n % kOutPieces;
            const f16x8 v = *(const f16x8*)((const char*)smem + out_at(plane, q, piece));
            if (q0 + q < q_end && p0 + piece * 8 < p_end) *(f16x8*)(out + (int64_t)(q0 + q) * ld + p0 + piece * 8) = v;
        }
    }
    __device__ static void fetch(void* smem, int plane, const _Float16* in, int64_t ld, int p0, int q0, int p_end, int q_end) {
#pragma unroll 4
        for (int n = threadIdx.x; n < TQ * kOutPieces; n += kThreads) {
            const int q = n / kOutPieces, piece = n % kOutPieces;
            if (q0 + q < q_end && p0 + piece * 8 < p_end)
                *(f16x8*)((char*)smem + out_at(plane, q, piece)) = *(const f16x8*)(in + (int64_t)(q0 + q) * ld + p0 + piece * 8);
        }
    }
    // The tile's transpose: rows of p, pieces of 8 q (q_end a multiple of 8); 16 rows of 64 bytes an instruction.
    __device__ static void store_turned(const void* smem, int plane, _Float16* out, int64_t ld, int p0, int q0, int p_end, int q_end) {
        for (int n = threadIdx.x; n < TP * (TQ / 8); n += kThreads) {
            const int p = n % 16 + n / (2 * TQ) * 16, piece = n / 16 % (TQ / 8);
            f16x8 v;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = *((const _Float16*)((const char*)smem + out_at(plane, piece * 8 + e, p / 8)) + p % 8);
            if (p0 + p < p_end && q0 + piece * 8 < q_end) *(f16x8*)(out + (int64_t)(p0 + p) * ld + q0 + piece * 8) = v;
        }
    }
    // The same for fp32 values, four next to each other, for the blocks j0 .. j0 + n - 1 of every wave: row of LDS
    // (wave's number along q) * 32 n + 32 (j - j0) + lane % 32.
    __device__ static int out32_row(int j, int n) { return wave_id() / NP * 32 * n + 32 * j + (threadIdx.x & 31); }
    __device__ static int out32_col(int row, int j0, int n) { return row / (32 * n) * WQ + 32 * j0 + row % (32 * n); }
    __device__ static int out32_at(int r, int piece) { return r * (4 * TP) + ((piece ^ (r & 15)) << 4); }
    __device__ static f32x4v& held32(void* smem, int i, int j, int r, int n = FQ) {
        return *(f32x4v*)((char*)smem + out32_at(out32_row(j, n), row(i, r) / 4));
    }
    __device__ static f32x4v& out32x4(void* smem, int r, int p) { return *(f32x4v*)((char*)smem + out32_at(r, p / 4)); }
    __device__ static float out32(const void* smem, int r, int p) { return *((const float*)((const char*)smem + out32_at(r, p / 4)) + p % 4); }
    static constexpr int kOut32 = TP * TQ * 4;
};

// ---- planes ------------------------------------------------------------------------------
//
// fp16 holds 11 bits within 2^-14 .. 65504, and multiples of 2^-24 below.  With the power of two that brings the largest value
// to 2^14 .. 2^15 one plane holds bf16 values (8 bits) exactly from 2^-17 on, down to 2^-31 of the largest; two planes are off
// by 2^-23 of a value from 2^-2 on (lo's half step is 2^-25 at least), down to 2^-16 of the largest.  Smaller values are off by 2^-25, 2^-39
// of the largest, in either.

// The scale for a largest (finite) magnitude of these bits, which may be any: 2^-113 to 2^127 (magnitudes below 2^-113 stay below 2^14).
__device__ inline float plane_scale(uint32_t bits) {
    const int e = (int)(bits >> 23);
    return __builtin_bit_cast(float, (uint32_t)(127 + 14 - ((e < 14 ? 14 : e) - 127)) << 23);
}
// x = hi + lo; an infinite hi (or NaN) stands alone.
__device__ inline void split(float x, _Float16& hi, _Float16& lo) {
    hi = (_Float16)x;
    const float rest = x - (float)hi;
    lo = (_Float16)(__builtin_isfinite(rest) ? rest : 0.f);
}

// ---- host side ---------------------------------------------------------------------------

// Beyond 64 KiB of LDS a kernel has to be told, once on each device.  `told` is the kernel's own.
struct Told {
    std::atomic<bool> done[64] = {};
};
inline int allow_lds(const char* what, const void* kernel, int bytes, Told& told) {
    if (bytes <= 65536) return MB_OK;
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e == hipSuccess && dev < 64 && told.done[dev].load(std::memory_order_relaxed)) return MB_OK;
    if (e == hipSuccess) e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) return fail((int)e, "%s: %d bytes of LDS: %s", what, bytes, hipGetErrorString(e));
    if (dev < 64) told.done[dev].store(true, std::memory_order_relaxed);
    return MB_OK;
}

inline int64_t pad(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

}  // namespace g16
}  // namespace mb
