// Attention with a learned bias by distance buckets: what the forward and backward share.
//
//   s_ij = scale q_i . k_j + bias[bucket(pos_i - j), h],   p = softmax_j(s),   o_i = sum_j p_ij v_j
//
// Layout of the products.  All of them run on the 32 x 32 matrix instructions, whose result a
// lane holds as one column (lane % 32) and the 16 rows 8 (r / 4) + 4 (lane / 32) + r % 4.  The
// score block is taken transposed (keys by queries), so that a lane holds 16 keys of one query:
// the row's maximum and sum need one exchange between the two half waves, and the probabilities
// are already the right-hand operand of the next product.  An operand's k index may run in any
// order as long as both operands agree: slot (half wave g, element e) of the 16-deep step c is
// row 16 c + 8 (e / 4) + 4 g + e % 4, which is where the results lie.  The other operand comes
// out of LDS in that order by the transposing 16-bit LDS read (or, in fp32, by element).
#pragma once

#include "common.h"

namespace mb {
namespace battn {

constexpr int kThreads = 256;   // four waves
constexpr int kWaveRows = 32;   // queries (or keys) of a wave
constexpr int kRows = 4 * kWaveRows;
constexpr int kMaxStarts = 128;
constexpr int kStartStep = 16;  // starts[] is filled up to a multiple of it with distances that none reaches
static_assert(kMaxStarts % kStartStep == 0, "");
constexpr int kMaxReach = 1024; // the largest distance with a bucket of its own
constexpr int kPad = 96;        // table entries beyond each end: a 32 x 64 tile's distances that pass it
constexpr float kLog2e = 1.4426950408889634f;
// The running maximum follows a row's scores only where one passes it by more than this (in log2
// units): probabilities up to 2^8 of the maximum's lose nothing in fp32 or bf16, and the output
// is rescaled a few times a row instead of in most tiles.
constexpr float kSlack = 8.f;

typedef __attribute__((__ext_vector_type__(4))) __bf16 bf16x4;
typedef __attribute__((__ext_vector_type__(8))) __bf16 bf16x8;
typedef __attribute__((__ext_vector_type__(4))) short s16x4;
typedef __attribute__((__ext_vector_type__(4))) float f32x4;
typedef __attribute__((__ext_vector_type__(8))) float f32x8;
typedef __attribute__((__ext_vector_type__(16))) float f32x16;
typedef f32x8 f32x8u __attribute__((aligned(16)));  // rows begin at multiples of 16 bytes

template <typename T>
struct Ty;
template <>
struct Ty<__bf16> {
    typedef bf16x8 Frag;
    typedef bf16x8 FragMem;
    typedef bf16x4 Quad;
    static constexpr int kKeys = 64;   // rows of a staged tile
    static __device__ f32x16 mma(Frag a, Frag b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Ty<float> {
    typedef f32x8 Frag;
    typedef f32x8u FragMem;
    typedef f32x4 Quad;
    static constexpr int kKeys = 32;
    // the 16-deep product as eight 2-deep ones: element e of both operands is slot (g, e)
    static __device__ f32x16 mma(Frag a, Frag b, f32x16 c) {
#pragma unroll
        for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
};

// Waves of a SIMD that the registers have to be enough for.  Two (at most 256 registers) keep the
// matrix instructions' results in VGPRs, where the softmax reads them; with one, the compiler puts
// them into AGPRs and moves each of them (forward at 4 x 4096, 8 heads x 64: 279 us instead of
// 131; in fp32 at 8 x 1000, 8 heads x 128: 178 instead of 238).  Heads of 128 do not fit that way with
// two results (`wide`), nor, in fp32, in the queries' pass (178 spills).
template <typename T, int HD, bool WIDE = false>
constexpr int waves_per_simd() { return HD == 128 && WIDE ? 1 : 2; }

struct Args {
    const void *q, *k, *v, *o, *d_o;        // o, d_o: backward
    int64_t q_sb, q_sh, q_sl, k_sb, k_sh, k_sl, v_sb, v_sh, v_sl, o_sb, o_sh, o_sl, do_sb, do_sh, do_sl;
    const void* bias;                        // [buckets, H]
    const void *lengths, *start;             // [B] or NULL
    void *out, *dk, *dv, *dbias;             // out: o (forward) or dq
    int64_t out_sb, out_sh, out_sl, dk_sb, dk_sh, dk_sl, dv_sb, dv_sh, dv_sl;
    float *lse, *rows, *dbias_part;          // [B, H, Lq] (log2 units), [2, B, H, Lq], [H, bias_rows, buckets]
    float* o_part;                           // [B, Hk, Lq, H / Hk, o_parts, hd + 2] where the forward's walks are split
    int o_parts;
    // where the backward's passes are split: [q_parts, B, H, Lq, hd], [q_parts, 4, B, H, Lq], [kv_parts, B, Hk, Lk, 2, hd]
    float *q_part, *q_stat, *kv_part;
    int64_t bias_rows;
    int q_parts, kv_parts;
    int lengths_bytes, start_bytes, start0;
    int B, H, Hk, Lq, Lk, nq;
    int causal, bias_bf16, buckets, n_starts, reach;
    float scale;
    int starts[kMaxStarts];                  // first distance of each bucket of one direction
};

// The distance table covers lo .. hi and is padded by kPad entries on both ends.  Distances from
// hi on have one bucket, and so have those from lo down.
struct Reach {
    int lo, hi;
    __host__ __device__ explicit Reach(const Args& a)
        : lo(a.causal ? 0 : -(a.reach > 1 ? a.reach : 1)), hi(a.reach) {}
    __host__ __device__ int entries() const { return hi - lo + 1 + 2 * kPad; }
};

__device__ inline int row_int(const void* p, int bytes, int b, int lo, int hi) {
    const int64_t v = bytes == 8 ? ((const int64_t*)p)[b] : (int64_t)((const int32_t*)p)[b];
    return (int)(v < lo ? lo : v > hi ? hi : v);
}
constexpr int kFarthest = 1 << 29;   // positions and lengths: sums and differences of them fit 32 bits
// Position of the row's first query.
__device__ inline int first_position(const Args& a, int b) {
    return a.start ? row_int(a.start, a.start_bytes, b, -kFarthest, kFarthest) : a.start0;
}
// How many of the row's keys may be seen: rows from there on are not used at all, so that a cache
// may hold anything behind its last token.
__device__ inline int key_count(const Args& a, int b) {
    const int n = a.lengths ? row_int(a.lengths, a.lengths_bytes, b, 0, a.Lk) : a.Lk;
    return a.causal ? max(0, min(n, first_position(a, b) + a.Lq)) : n;
}

// Buckets of N distances: how many first distances are no larger.  All of them are compared, at
// uniform addresses: a search would take a chain of loads for each lane's own (3 us a workgroup).
template <int N>
__device__ inline void buckets_of(const Args& a, const int* d, int* bucket) {
    int n[N];
#pragma unroll
    for (int i = 0; i < N; ++i) n[i] = d[i] < 0 ? -d[i] : d[i], bucket[i] = -1;
    for (int k0 = 0; k0 < a.n_starts; k0 += kStartStep)
#pragma unroll
        for (int k = 0; k < kStartStep; ++k) {
            const int first = a.starts[k0 + k];
#pragma unroll
            for (int i = 0; i < N; ++i) bucket[i] += first <= n[i] ? 1 : 0;
        }
#pragma unroll
    for (int i = 0; i < N; ++i) bucket[i] += !a.causal && d[i] < 0 ? a.n_starts : 0;
}

// A bias below -2^16 hides its pairs: were it kept, a row that has no others would get a denominator of
// that size, next to which the backward's products lose the scores (at -1e9 p comes out at 2^100).  Where all
// of a head's biases lie down there, its largest, which a softmax does not notice, is taken off first.
constexpr float kHidden = -65536.f;
__device__ inline float bias_value(const Args& a, int n, int h) {
    const int64_t at = (int64_t)n * a.H + h;
    return a.bias_bf16 ? (float)((const __bf16*)a.bias)[at] : ((const float*)a.bias)[at];
}
__device__ inline bool is_low(float v) { return v < kHidden && v > -INFINITY; }
// What is taken off head h's biases where one of them is low; no other thread pays for it.  The kernel's arguments
// (Args is the first one) are read once more from where they came: kept in registers for this, they take dk and dv's
// loop the room to read ahead of its products (heads of 128, 8 x 1024: 84 us against 80).
// UNIFORM: h is the whole wave's.
template <bool UNIFORM>
__device__ inline float taken_off(int h) {
    auto* a = (__attribute__((address_space(4))) const Args*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(a));
    if constexpr (UNIFORM) asm volatile("" : "+s"(h));
    const void* bias = a->bias;
    const int buckets = a->buckets, heads = a->H, bf16 = a->bias_bf16;
    float top = -INFINITY;
#pragma unroll 1
    for (int n = 0; n < buckets; ++n) {
        const int64_t at = (int64_t)n * heads + h;
        top = fmaxf(top, bf16 ? (float)((const __bf16*)bias)[at] : ((const float*)bias)[at]);
    }
    return top < kHidden ? top : 0.f;
}
__device__ inline float in_log2(float v) { return v < kHidden ? -INFINITY : kLog2e * v; }

// tab[i] = log2(e) bias of distance lo - kPad + i (clamped to lo .. hi), by all threads.
__device__ inline void fill_table(const Args& a, int h, float* tab) {
    const Reach r(a);
    for (int i = threadIdx.x; i < r.entries(); i += 2 * blockDim.x) {
        int d[2], n[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            d[e] = r.lo - kPad + i + e * (int)blockDim.x;
            d[e] = d[e] < r.lo ? r.lo : d[e] > r.hi ? r.hi : d[e];
        }
        buckets_of<2>(a, d, n);
        const float x = bias_value(a, n[0], h), y = bias_value(a, n[1], h);
        const float off = __any(is_low(x) || is_low(y)) ? taken_off<true>(h) : 0.f;
        tab[i] = in_log2(x - off);
        if (i + (int)blockDim.x < r.entries()) tab[i + blockDim.x] = in_log2(y - off);
    }
}

// ---- staged tiles ------------------------------------------------------------------------------
//
// Rows go from memory straight into LDS, 16 bytes a lane, two tiles ahead of the one that is used
// (loads through registers, one tile ahead, left the waves waiting: forward at 4 x 4096, 8 heads x
// 64, 117 us against 87 with the loads taken out).  Such a load puts its 64 pieces next to each
// other, so a row has no padding; piece c of row r lies in the row's place c ^ swz(r) instead,
// which spreads both ways of reading the tile over the banks.

// 16 (or 4) bytes a lane from base + voff to LDS at lds + 16 (or 4) * lane.  M0 holds the LDS address; the compiler
// reserves it for its own instructions, which set it before they use it, warns of the clobber for that reason, and
// has to know of it so that it keeps no value there from one of them to the next.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ inline void dma16(uint32_t lds, uint32_t voff, const void* base) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "s"(lds), "v"(voff), "s"(base)
                 : "memory", "m0");
}
__device__ inline void dma4(uint32_t lds, uint32_t voff, const void* base) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2"
                 :
                 : "s"(lds), "v"(voff), "s"(base)
                 : "memory", "m0");
}
#pragma clang diagnostic pop
// Waits until at most N of the wave's loads are on their way, and for the other waves.
template <int N>
__device__ inline void wait_and_meet() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(N) : "memory");
}
// Ends the compiler's own loads before a loop of dma16: it would wait for them at their first use,
// inside the loop, and with them for the loads that are meant to be on their way.
__device__ inline void loads_done() { __builtin_amdgcn_s_waitcnt(0x0F70); }   // vmcnt(0)

__device__ inline int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

__device__ inline uint32_t lds_address(const void* p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}

template <typename T, int HD, int ROWS = Ty<T>::kKeys>
struct Tile {
    static constexpr int kN = ROWS;
    static constexpr int kRow = HD * (int)sizeof(T);               // bytes
    static constexpr int kBytes = kN * kRow;
    static constexpr int kPieces = kRow / 16;
    static constexpr int kLoads = kBytes / 4096;                   // of each of the four waves
    static_assert(kBytes % 4096 == 0, "a wave's load moves 1 KiB");
    // Tiles of each kind in LDS: two on their way beside the one in use, or one where three would leave
    // a CU a single workgroup of the two that its registers hold (heads of 128).
    static constexpr int kStages = kBytes > 8192 ? 2 : 3;

    static __device__ constexpr int swz(int row) {
        if (kPieces == 4) return (row >> 2) & 3;
        if (kPieces == 8) return ((row >> 1) & 1) << 2 | ((row >> 3) & 1) << 1 | ((row >> 2) & 1);
        return (row & 3) << 2 | ((row >> 2) & 3);
    }
    static __device__ int at(int row, int piece) { return row * kRow + ((piece ^ swz(row & 15)) << 4); }

    // This lane's part of each of its wave's loads: the row, and its offset from the tile's first.
    struct Offsets {
        uint32_t v[kLoads];
        __device__ explicit Offsets(int64_t sl) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) v[i] = (uint32_t)(row(i) * (int)(sl * (int)sizeof(T))) + piece(i);
        }
        static __device__ int slot(int i) { return i * kThreads + (int)(threadIdx.x % kThreads); }
        static __device__ int row(int i) { return slot(i) / kPieces; }
        static __device__ uint32_t piece(int i) { return (uint32_t)((slot(i) % kPieces) ^ swz(row(i) & 15)) << 4; }
    };
    // Rows row0 .. row0 + kN - 1 of `base` on their way to the tile; rows from `rows` (at least 1)
    // on are the last one again.
    static __device__ void load(uint32_t tile, const T* base, int64_t sl, int row0, int rows, const Offsets& off) {
        const uint32_t lds = tile + wave_id() % 4 * 1024;
        const int first = min(row0, rows - 1);
        const T* from = base + first * sl;
        if (row0 + kN <= rows) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) dma16(lds + i * 4096, off.v[i], from);
        } else {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int r = min(Offsets::row(i), rows - 1 - first);
                dma16(lds + i * 4096, (uint32_t)(r * (int)(sl * (int)sizeof(T))) + Offsets::piece(i), from);
            }
        }
    }

    // Where this lane reads, relative to a tile: with these kept, several reads cost one addition (the
    // rest is the instruction's constant offset).  In fp32, whose products take 16 times as long, some
    // of them are formed at the read instead of kept.
    typedef __attribute__((address_space(3))) const char lds_char;
    struct Lane {
        uint32_t row[sizeof(T) == 2 ? HD / 16 : 2], col[sizeof(T) == 2 ? HD / 16 : 8];
        __device__ Lane() {
            const int lane = threadIdx.x & 63, g = lane >> 5;
#pragma unroll
            for (int i = 0; i < (sizeof(T) == 2 ? HD / 16 : 2); ++i) row[i] = at(lane & 31, sizeof(T) == 2 ? 2 * i + g : 2 * g + i);
            if constexpr (sizeof(T) == 2) {
                // 16 lanes read 4 rows of 16 channels, 8 bytes each, and get 4 rows of one channel each
                const int r = 4 * g + ((lane & 15) >> 2), d = (lane & 16) + 4 * (lane & 3);
#pragma unroll
                for (int i = 0; i < HD / 16; ++i) col[i] = at(r + 8 * (i % 2), 4 * (i / 2) + (d >> 3)) + 2 * (d & 7);
            } else {
                const int d = lane & 31;
#pragma unroll
                for (int i = 0; i < 8; ++i) col[i] = at(4 * g + 8 * (i / 4) + i % 4, d >> 2) + 4 * (d & 3);
            }
        }
    };
    // Operand with the tile's rows row0 + lane % 32 (row0 a multiple of 32) and channels 16 c ..: a
    // lane's 8 are adjacent.
    static __device__ typename Ty<T>::Frag rows(uint32_t tile, const Lane& l, int row0, int c) {
        if constexpr (sizeof(T) == 2) {
            return *(__attribute__((address_space(3))) const bf16x8*)((lds_char*)(uintptr_t)(tile + l.row[c]) + row0 * kRow);
        } else {
            // channels 16 c further, piece n becomes n ^ 4 c
            typedef __attribute__((address_space(3))) const f32x4 lds_f32x4;
            const f32x4 x = *(lds_f32x4*)((lds_char*)(uintptr_t)(tile + (l.row[0] ^ (c << 6))) + row0 * kRow);
            const f32x4 y = *(lds_f32x4*)((lds_char*)(uintptr_t)(tile + (l.row[1] ^ (c << 6))) + row0 * kRow);
            return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
    // Operand with channels 32 d + lane % 32 and the tile's rows row0 + (the slots' order above), row0
    // a multiple of 16.
    static __device__ typename Ty<T>::Frag cols(uint32_t tile, const Lane& l, int row0, int d) {
        if constexpr (sizeof(T) == 2) {
            typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
            const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_s16x4*)((lds_char*)(uintptr_t)(tile + l.col[2 * d]) + row0 * kRow));
            const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_s16x4*)((lds_char*)(uintptr_t)(tile + l.col[2 * d + 1]) + row0 * kRow));
            return __builtin_shufflevector(__builtin_bit_cast(bf16x4, x), __builtin_bit_cast(bf16x4, y), 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
            f32x8 f;
#pragma unroll
            for (int e = 0; e < 8; ++e)   // 32 channels further, piece c becomes c ^ 8
                f[e] = *(__attribute__((address_space(3))) const float*)((lds_char*)(uintptr_t)(tile + (l.col[e] ^ (d << 7))) + row0 * kRow);
            return f;
        }
    }
};

// Rows of a wave in registers: row r0 + lane % 32, channels 16 c + 8 (lane / 32) ..; rows from
// `rows` on are zero.
template <typename T, int HD>
__device__ inline void load_frags(const T* base, int64_t sl, int r0, int rows, typename Ty<T>::Frag* f) {
    const int lane = threadIdx.x & 63;
    const int r = r0 + (lane & 31);
#pragma unroll
    for (int c = 0; c < HD / 16; ++c) {
        typename Ty<T>::Frag z;
#pragma unroll
        for (int e = 0; e < 8; ++e) z[e] = (T)0.f;
        f[c] = z;
        if (r < rows)
            f[c] = *reinterpret_cast<const typename Ty<T>::FragMem*>(base + (int64_t)r * sl + 16 * c + 8 * (lane >> 5));
    }
}

// Eight of a block's 16 values as an operand of the next product (rounded to nearest in bf16).
template <typename T>
__device__ inline typename Ty<T>::Frag to_frag(const f32x16& x, int c) {
    typename Ty<T>::Frag f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = (T)x[8 * c + e];
    return f;
}

// A 32 x 32 result block (channels d0 .. by rows) into the wave's rows.
template <typename T>
__device__ inline void store_block(T* row, int d0, const f32x16& x, float mul) {
    const int g = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        typename Ty<T>::Quad v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (T)(x[4 * r + e] * mul);
        *reinterpret_cast<typename Ty<T>::Quad*>(row + d0 + 8 * r + 4 * g) = v;
    }
}

// The row block and head of workgroup id.  Blocks with the most pairs go first (`first_most`: block 0,
// else the last one), all heads of a block position one after another: a head's blocks then land
// on one XCD where the heads are a multiple of 8, and read its keys out of that L2.  Every second
// 256 workgroups (one for each CU) run backwards in steps of 8, so that a CU's share of a grid
// that is resident at once comes out even.
__device__ inline void place(int id, int heads, int blocks, bool first_most, int& bh, int& blk) {
    if ((id & 256) && (id | 255) < heads * blocks) id = (id & ~255) + (31 - ((id >> 3) & 31)) * 8 + (id & 7);
    bh = id % heads;
    blk = id / heads;
    if (!first_most) blk = blocks - 1 - blk;
}

// A value of this lane and of the same lane of the other half wave: the first register's upper half
// is swapped with the second's lower half.
__device__ inline void halves(float v, float& lo, float& hi) {
    const int a = __builtin_bit_cast(int, v);
    const auto r = __builtin_amdgcn_permlane32_swap(a, a, false, false);
    const int x = r[0], y = r[1];
    lo = __builtin_bit_cast(float, x);
    hi = __builtin_bit_cast(float, y);
}
__device__ inline float half_max(float v) {
    float lo, hi;
    halves(v, lo, hi);
    return fmaxf(lo, hi);
}
__device__ inline float half_sum(float v) {
    float lo, hi;
    halves(v, lo, hi);
    return lo + hi;
}

__device__ inline f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.f;
    return z;
}

// Row of a block's value r in this lane.
__device__ inline int row_of(int r) { return 8 * (r / 4) + 4 * ((threadIdx.x & 63) >> 5) + r % 4; }

}  // namespace battn
}  // namespace mb
