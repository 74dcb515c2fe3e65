// The 2-norm of many tensors together, and their scaling to a bound, on gfx950.
//
//   norm = sqrt(sum over tensors and elements of g^2),  factor = min(1, max_norm / (norm + 1e-6)),
//   dst = factor * src
//
// HBM-bound: every element is read for the norm, and read again and written for the scaling.
// Up to kTensors tensors share a launch: their addresses and sizes travel in the kernel's
// arguments, so nothing is copied to the device first.  The elements of all of them form one
// row of chunks, and every workgroup takes an equal run of it (a binary search finds the run's
// first tensor).  Squares are summed in 64 bits: no value of an fp32 gradient overflows there,
// and the sum's order is fixed.  The scaling launches follow in the same stream; each of their
// workgroups adds the norm launches' partial sums by itself (8 KiB out of L2), which saves a
// launch between the two.  In place, where the factor is 1, they leave without touching memory.
#include "common.h"

#include <algorithm>
#include <cmath>
#include <new>

namespace mb {
namespace {

constexpr int kClipThreads = 256;
constexpr int kTensors = 120;       // tensors of a launch: 120 * 29 bytes of kernel arguments
constexpr int kChunk = 4096;        // elements
constexpr int kClipBlocks = 1024;   // four workgroups per CU

typedef __attribute__((__ext_vector_type__(4))) __bf16 bf16x4v;

struct ClipArgs {
    const void* src[kTensors];
    void* dst[kTensors];
    int64_t n[kTensors];
    int32_t first[kTensors];        // the tensor's first chunk
    uint8_t kind[kTensors];         // bit 0: src is bf16, bit 1: dst is bf16, bit 2: aligned for vectors
    int count, chunks;
    double* part;                   // norm: [blocks] partial sums of this launch
    int parts;                      // scaling: partial sums of all launches
    float max_norm;
    float* norm_out;
    int in_place, write_norm;
};
static_assert(sizeof(ClipArgs) <= 4096, "kernel arguments");

__device__ inline double block_sum(double v) {
    __shared__ double s[kClipThreads / 64];
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int i = 0; i < kClipThreads / 64; ++i) v += s[i];
    return v;
}

// The workgroup's run of chunks, and the tensor that holds its first one.
__device__ inline void run_of(const ClipArgs& a, int& c0, int& c1, int& t) {
    c0 = (int)((int64_t)a.chunks * blockIdx.x / gridDim.x);
    c1 = (int)((int64_t)a.chunks * (blockIdx.x + 1) / gridDim.x);
    int lo = 0, hi = a.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.first[mid] <= c0) lo = mid;
        else hi = mid - 1;
    }
    t = lo;
}

__device__ inline f32x4v load4(const void* p, int64_t i, bool bf16) {
    if (!bf16) return *reinterpret_cast<const f32x4v*>((const float*)p + i);
    const bf16x4v q = *reinterpret_cast<const bf16x4v*>((const __bf16*)p + i);
    return f32x4v{(float)q[0], (float)q[1], (float)q[2], (float)q[3]};
}
__device__ inline float load1(const void* p, int64_t i, bool bf16) {
    return bf16 ? (float)((const __bf16*)p)[i] : ((const float*)p)[i];
}
__device__ inline void store4(void* p, int64_t i, bool bf16, f32x4v v) {
    if (!bf16) {
        *reinterpret_cast<f32x4v*>((float*)p + i) = v;
    } else {
        const bf16x4v q = {(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
        *reinterpret_cast<bf16x4v*>((__bf16*)p + i) = q;
    }
}
__device__ inline void store1(void* p, int64_t i, bool bf16, float v) {
    if (bf16) ((__bf16*)p)[i] = (__bf16)v;
    else ((float*)p)[i] = v;
}

__global__ void __launch_bounds__(kClipThreads) grad_square_kernel(const ClipArgs a) {
    int c0, c1, t;
    run_of(a, c0, c1, t);
    double sum = 0.0;
    for (int c = c0; c < c1; ++c) {
        while (t + 1 < a.count && a.first[t + 1] <= c) ++t;
        const int64_t e0 = (int64_t)(c - a.first[t]) * kChunk;
        const int64_t e1 = e0 + kChunk < a.n[t] ? e0 + kChunk : a.n[t];
        const void* p = a.src[t];
        const bool bf = a.kind[t] & 1;
        if (e1 - e0 == kChunk && (a.kind[t] & 4)) {
            f32x4v v[kChunk / kClipThreads / 4];
#pragma unroll
            for (int i = 0; i < kChunk / kClipThreads / 4; ++i)
                v[i] = load4(p, e0 + (i * kClipThreads + threadIdx.x) * 4, bf);
#pragma unroll
            for (int i = 0; i < kChunk / kClipThreads / 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) sum = __builtin_fma((double)v[i][j], (double)v[i][j], sum);
        } else {
            for (int64_t e = e0 + threadIdx.x; e < e1; e += kClipThreads) {
                const double v = load1(p, e, bf);
                sum = __builtin_fma(v, v, sum);
            }
        }
    }
    sum = block_sum(sum);
    if (threadIdx.x == 0) a.part[blockIdx.x] = sum;
}

__global__ void __launch_bounds__(kClipThreads) grad_scale_kernel(const ClipArgs a) {
    double sum = 0.0;
    for (int i = threadIdx.x; i < a.parts; i += kClipThreads) sum += a.part[i];
    const double norm = sqrt(block_sum(sum));
    if (a.write_norm && blockIdx.x == 0 && threadIdx.x == 0) *a.norm_out = (float)norm;
    const double f = (double)a.max_norm / (norm + 1e-6);
    const float factor = f >= 1.0 ? 1.0f : (float)f;  // NaN stays NaN, as in a product with it
    if (a.count == 0 || (a.in_place && factor == 1.0f)) return;
    int c0, c1, t;
    run_of(a, c0, c1, t);
    for (int c = c0; c < c1; ++c) {
        while (t + 1 < a.count && a.first[t + 1] <= c) ++t;
        const int64_t e0 = (int64_t)(c - a.first[t]) * kChunk;
        const int64_t e1 = e0 + kChunk < a.n[t] ? e0 + kChunk : a.n[t];
        const void* p = a.src[t];
        void* q = a.dst[t];
        const bool bf = a.kind[t] & 1, obf = a.kind[t] & 2;
        if (e1 - e0 == kChunk && (a.kind[t] & 4)) {
            f32x4v v[kChunk / kClipThreads / 4];
#pragma unroll
            for (int i = 0; i < kChunk / kClipThreads / 4; ++i)
                v[i] = load4(p, e0 + (i * kClipThreads + threadIdx.x) * 4, bf);
#pragma unroll
            for (int i = 0; i < kChunk / kClipThreads / 4; ++i)
                store4(q, e0 + (i * kClipThreads + threadIdx.x) * 4, obf, v[i] * factor);
        } else {
            for (int64_t e = e0 + threadIdx.x; e < e1; e += kClipThreads)
                store1(q, e, obf, load1(p, e, bf) * factor);
        }
    }
}

// A stretch of memory, and whether it is written.
struct Stretch {
    uintptr_t from, to;
    bool written;
};

int64_t chunks_of(int64_t n) { return (n + kChunk - 1) / kChunk; }

}  // namespace
}  // namespace mb

using namespace mb;

extern "C" int64_t mb_grad_clip_workspace(int count) {
    if (count < 0) return 0;
    return ((int64_t)(count + kTensors - 1) / kTensors + 1) * kClipBlocks * (int64_t)sizeof(double);
}

extern "C" int mb_grad_clip(const void* const* src, const int32_t* src_dtype, void* const* dst,
                            const int32_t* dst_dtype, const int64_t* n, int count, float max_norm, float* norm_out,
                            void* workspace, int64_t workspace_bytes, void* stream) {
    MB_REQUIRE(count >= 0, "mb_grad_clip: count=%d < 0", count);
    MB_REQUIRE(norm_out, "mb_grad_clip: null norm_out");
    MB_REQUIRE(count == 0 || (src && src_dtype && n && (!dst || dst_dtype)), "mb_grad_clip: null pointer argument");
    MB_REQUIRE(max_norm >= 0.f, "mb_grad_clip: max_norm=%g", (double)max_norm);
    if (!workspace || workspace_bytes < mb_grad_clip_workspace(count))
        return fail(MB_ERR_WORKSPACE, "mb_grad_clip: workspace of %lld bytes, %lld are needed",
                    (long long)workspace_bytes, (long long)mb_grad_clip_workspace(count));
    bool in_place = dst != nullptr;
    for (int i = 0; i < count; ++i) {
        MB_REQUIRE(n[i] >= 0, "mb_grad_clip: tensor %d has %lld elements", i, (long long)n[i]);
        MB_REQUIRE(n[i] == 0 || (src[i] && (!dst || dst[i])), "mb_grad_clip: tensor %d has a null pointer", i);
        MB_REQUIRE(src_dtype[i] == MB_DTYPE_F32 || src_dtype[i] == MB_DTYPE_BF16, "mb_grad_clip: tensor %d: dtype=%d", i,
                   src_dtype[i]);
        if (dst) {
            MB_REQUIRE(dst_dtype[i] == MB_DTYPE_F32 || dst_dtype[i] == MB_DTYPE_BF16, "mb_grad_clip: tensor %d: dtype=%d",
                       i, dst_dtype[i]);
            in_place = in_place && (n[i] == 0 || (src[i] == dst[i] && src_dtype[i] == dst_dtype[i]));
        }
    }
    if (dst) {
        // no stretch may be written twice, nor written where another tensor is read: the
        // workgroups run in no order
        Stretch* s = new (std::nothrow) Stretch[2 * (size_t)count + 1];
        MB_REQUIRE(s, "mb_grad_clip: no host memory for %d tensors", count);
        int m = 0;
        for (int i = 0; i < count; ++i) {
            if (n[i] == 0) continue;
            const uintptr_t p = (uintptr_t)src[i], q = (uintptr_t)dst[i];
            const int64_t ps = src_dtype[i] == MB_DTYPE_F32 ? 4 : 2, qs = dst_dtype[i] == MB_DTYPE_F32 ? 4 : 2;
            s[m++] = {q, q + n[i] * qs, true};
            if (p != q || ps != qs) s[m++] = {p, p + n[i] * ps, false};
        }
        std::sort(s, s + m, [](const Stretch& a, const Stretch& b) { return a.from < b.from; });
        uintptr_t any = 0, written = 0;
        bool overlap = false;
        for (int i = 0; i < m; ++i) {
            overlap = overlap || s[i].from < (s[i].written ? any : written);
            any = std::max(any, s[i].to);
            if (s[i].written) written = std::max(written, s[i].to);
        }
        delete[] s;
        MB_REQUIRE(!overlap, "mb_grad_clip: tensors share memory that the call writes");
    }
    hipStream_t st = (hipStream_t)stream;
    int parts = 0;
    // pass 0: squares;  pass 1: scaling (or, with no dst, one workgroup that writes the norm)
    for (int pass = 0; pass < 2; ++pass) {
        int i = 0;
        bool norm_written = false;
        do {
            if (pass == 1 && !dst) i = count;
            ClipArgs a = {};
            int64_t chunks = 0;
            for (; i < count && a.count < kTensors; ++i) {
                if (n[i] == 0) continue;
                if (chunks + chunks_of(n[i]) > 0x7fffffff) break;
                const int t = a.count++;
                a.src[t] = src[i];
                a.dst[t] = dst ? dst[i] : nullptr;
                a.n[t] = n[i];
                a.first[t] = (int32_t)chunks;
                const bool sb = src_dtype[i] == MB_DTYPE_BF16, db = dst && dst_dtype[i] == MB_DTYPE_BF16;
                const bool vec = !((uintptr_t)src[i] & (sb ? 7 : 15)) && (!dst || !((uintptr_t)dst[i] & (db ? 7 : 15)));
                a.kind[t] = (uint8_t)((sb ? 1 : 0) | (db ? 2 : 0) | (vec ? 4 : 0));
                chunks += chunks_of(n[i]);
            }
            MB_REQUIRE(i >= count || a.count > 0, "mb_grad_clip: tensor %d has %lld elements, too many", i, (long long)n[i]);
            a.chunks = (int)chunks;
            const int blocks = (int)std::max<int64_t>(1, std::min<int64_t>(chunks, kClipBlocks));
            a.max_norm = max_norm;
            a.norm_out = norm_out;
            a.in_place = in_place;
            if (pass == 0) {
                if (a.count == 0) break;
                a.part = (double*)workspace + parts;
                parts += blocks;
                hipLaunchKernelGGL(grad_square_kernel, dim3(blocks), dim3(kClipThreads), 0, st, a);
            } else {
                if (a.count == 0 && norm_written) break;
                a.part = (double*)workspace;
                a.parts = parts;
                a.write_norm = !norm_written;
                norm_written = true;
                hipLaunchKernelGGL(grad_scale_kernel, dim3(blocks), dim3(kClipThreads), 0, st, a);
            }
        } while (i < count);
    }
    return check_launch("mb_grad_clip");
}
