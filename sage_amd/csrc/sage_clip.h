// Clipping of gradients by their global norm: N = sqrt(sum over all tensors of g^2), and g * (max_norm / N) where N exceeds
// max_norm.  Memory-bound: the gradients are read twice and written once (N is not known before the last one is read).
//
// Squares are summed in float64 (no float32 square overflows or vanishes, and the sum of 10^9 of them keeps its bits), in an
// order that depends on the sizes alone: one partial per block of CLIP_BLOCK elements of one tensor, then one workgroup sums
// the partials.  The list of tensors travels in the kernel arguments, CLIP_TENSORS at a time, so that a captured call
// holds it by value.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#define CLIP_TENSORS 128
#define CLIP_BLOCK 32768

struct ClipTable {
    const void* in[CLIP_TENSORS];
    void* out[CLIP_TENSORS];
    int64_t size[CLIP_TENSORS];          // elements, negative for bf16
    uint32_t first[CLIP_TENSORS + 1];    // block that a tensor starts at
    uint32_t n;
    uint32_t block0;                     // partial of block 0
};

// 16 bytes at the alignment that elements have
struct __attribute__((packed, aligned(2))) clip_u4 { uint32_t v[4]; };

__device__ __forceinline__ uint32_t clip_find(const ClipTable& t, uint32_t block) {
    uint32_t lo = 0, hi = t.n;           // the last tensor whose first block is not past this one
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (t.first[mid] <= block) lo = mid; else hi = mid;
    }
    return lo;
}
__device__ __forceinline__ float clip_lo(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float clip_hi(uint32_t u) { return __uint_as_float(u & 0xFFFF0000u); }

__device__ __forceinline__ double clip_block_sum(double v, double* red) {
    for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
    const int waves = blockDim.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0.0;
    for (int i = 0; i < waves; ++i) s += red[i];
    return s;
}

__global__ __launch_bounds__(256) void k_clip_squares(ClipTable t, double* __restrict__ part) {
    __shared__ double red[4];
    const uint32_t i = clip_find(t, blockIdx.x);
    const bool bf16 = t.size[i] < 0;
    const int64_t n = bf16 ? -t.size[i] : t.size[i], at = (int64_t)(blockIdx.x - t.first[i]) * CLIP_BLOCK;
    const int m = (int)min((int64_t)CLIP_BLOCK, n - at);
    double s0 = 0.0, s1 = 0.0;
    if (bf16) {
        const uint16_t* p = (const uint16_t*)t.in[i] + at;
        for (int j = threadIdx.x * 8; j + 8 <= m; j += 2048) {
            const clip_u4 q = *(const clip_u4*)(p + j);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const double a = clip_lo(q.v[k]), b = clip_hi(q.v[k]);
                s0 = fma(a, a, s0); s1 = fma(b, b, s1);
            }
        }
        const int j = (m & ~7) + threadIdx.x;
        if (threadIdx.x < 8 && j < m) { const double a = clip_lo(p[j]); s0 = fma(a, a, s0); }
    } else {
        const float* p = (const float*)t.in[i] + at;
        for (int j = threadIdx.x * 4; j + 4 <= m; j += 1024) {
            const clip_u4 q = *(const clip_u4*)(p + j);
#pragma unroll
            for (int k = 0; k < 4; k += 2) {
                const double a = __uint_as_float(q.v[k]), b = __uint_as_float(q.v[k + 1]);
                s0 = fma(a, a, s0); s1 = fma(b, b, s1);
            }
        }
        const int j = (m & ~3) + threadIdx.x;
        if (threadIdx.x < 4 && j < m) { const double a = p[j]; s0 = fma(a, a, s0); }
    }
    const double s = clip_block_sum(s0 + s1, red);
    if (threadIdx.x == 0) part[t.block0 + blockIdx.x] = s;
}

// the norm, and the factor behind it (1 where nothing is to be clipped, or where the norm is not finite)
__global__ __launch_bounds__(1024) void k_clip_norm(const double* __restrict__ part, uint32_t n, double max_norm, float* __restrict__ norm, float* __restrict__ factor) {
    __shared__ double red[16];
    double s = 0.0;
    for (uint32_t i = threadIdx.x; i < n; i += 1024) s += part[i];
    s = sqrt(clip_block_sum(s, red));
    if (threadIdx.x == 0) {
        *norm = (float)s;
        *factor = s > max_norm && s < INFINITY ? (float)(max_norm / s) : 1.0f;
    }
}

__global__ __launch_bounds__(256) void k_clip_scale(ClipTable t, const float* __restrict__ factor) {
    const float f = *factor;
    const uint32_t i = clip_find(t, blockIdx.x);
    if (f == 1.0f && t.in[i] == t.out[i]) return;
    const bool bf16 = t.size[i] < 0;
    const int64_t n = bf16 ? -t.size[i] : t.size[i], at = (int64_t)(blockIdx.x - t.first[i]) * CLIP_BLOCK;
    const int m = (int)min((int64_t)CLIP_BLOCK, n - at);
    if (bf16) {
        const uint16_t* p = (const uint16_t*)t.in[i] + at;
        uint16_t* o = (uint16_t*)t.out[i] + at;
        for (int j = threadIdx.x * 8; j + 8 <= m; j += 2048) {
            clip_u4 q = *(const clip_u4*)(p + j);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const __bf16 a = (__bf16)(clip_lo(q.v[k]) * f), b = (__bf16)(clip_hi(q.v[k]) * f);
                q.v[k] = (uint32_t)__builtin_bit_cast(uint16_t, a) | (uint32_t)__builtin_bit_cast(uint16_t, b) << 16;
            }
            *(clip_u4*)(o + j) = q;
        }
        const int j = (m & ~7) + threadIdx.x;
        if (threadIdx.x < 8 && j < m) ((__bf16*)o)[j] = (__bf16)(clip_lo(p[j]) * f);
    } else {
        const float* p = (const float*)t.in[i] + at;
        float* o = (float*)t.out[i] + at;
        for (int j = threadIdx.x * 4; j + 4 <= m; j += 1024) {
            clip_u4 q = *(const clip_u4*)(p + j);
#pragma unroll
            for (int k = 0; k < 4; ++k) q.v[k] = __float_as_uint(__uint_as_float(q.v[k]) * f);
            *(clip_u4*)(o + j) = q;
        }
        const int j = (m & ~3) + threadIdx.x;
        if (threadIdx.x < 4 && j < m) o[j] = p[j] * f;
    }
}
