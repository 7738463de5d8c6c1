// Clipping of gradients by their global norm: N = sqrt(sum over all tensors of g^2), and g * (max_norm / N) where N exceeds
// max_norm.  Memory-bound: the gradients are read twice and written once (N is not known before the last one is read); where
// they fit the 256 MB cache behind HBM only once.  10^8 float32 elements: 196 us, 6.1 TB/s of those 12 bytes an element; two
// tensors of 13,107,200: 54 us; 301 tensors, float32 and bf16, 4 * 10^8 elements: 552 us.
//
// Squares are summed in float64 (no float32 square overflows or vanishes, and the sum of 10^9 of them keeps its bits), in an
// order that depends on the sizes alone: one partial per block of one tensor's elements, then one workgroup sums the partials.
// Blocks of 8,192 elements (10^8 elements: 226 us; of 16,384 233, of 32,768 237), of 2,048 up to 2^22 elements, where larger ones
// leave CUs idle.  The list of tensors travels in the kernel arguments, CLIP_TENSORS at a time, so that a captured call
// holds it by value.  Few elements are one workgroup's work in one launch in place of three: 2 tensors, 1,024 / 16,384 / 32,768
// elements 4.0 / 5.2 / 7.2 us against 7.4 / 7.7 / 8.0; 65,536 elements 11.0 against 7.9.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#define CLIP_TENSORS 128
#define CLIP_BLOCK 8192
#define CLIP_SMALL 2048     // of a block, up to 2^22 elements in all
#define CLIP_ONE 32768      // elements that one workgroup clips in one launch
#define CLIP_PIECE 1024

struct ClipTable {
    const void* in[CLIP_TENSORS];
    void* out[CLIP_TENSORS];
    int64_t size[CLIP_TENSORS];          // elements, negative for bf16
    uint32_t first[CLIP_TENSORS + 1];    // block that a tensor starts at
    uint32_t n;
    uint32_t block0;                     // partial of block 0
    int32_t block;                       // elements of a block
};

// 16 bytes at the alignment that elements have
struct __attribute__((packed, aligned(2))) clip_u4 { uint32_t v[4]; };

// The tensor that a block lies in: the last whose first block is not past it.  A whole wave asks, and each lane looks at two of
// the entries.
struct ClipFind {
    uint32_t a, b;
    __device__ __forceinline__ explicit ClipFind(const ClipTable& t) {
        const uint32_t lane = threadIdx.x & 63;
        a = lane < t.n ? t.first[lane] : 0xFFFFFFFFu;
        b = lane + 64 < t.n ? t.first[lane + 64] : 0xFFFFFFFFu;
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t block) const {
        return __popcll(__ballot(a <= block)) + __popcll(__ballot(b <= block)) - 1;
    }
};
static_assert(CLIP_TENSORS == 128, "two entries a lane");
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

__device__ __forceinline__ void clip_put(void* p, const clip_u4& q) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4), aligned(2)));
    __builtin_nontemporal_store(u4{q.v[0], q.v[1], q.v[2], q.v[3]}, (u4*)p);
}
// `m` elements of tensor i from `at`, by THREADS threads
template <int THREADS, int UNROLL>
__device__ __forceinline__ double clip_squares(const ClipTable& t, uint32_t i, int64_t at, int m, int thread) {
    double s0 = 0.0, s1 = 0.0;
    if (t.size[i] < 0) {
        const uint16_t* p = (const uint16_t*)t.in[i] + at;
#pragma unroll UNROLL
        for (int j = thread * 8; j + 8 <= m; j += THREADS * 8) {
            const clip_u4 q = *(const clip_u4*)(p + j);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const double a = clip_lo(q.v[k]), b = clip_hi(q.v[k]);
                s0 = fma(a, a, s0); s1 = fma(b, b, s1);
            }
        }
        const int j = (m & ~7) + thread;
        if (thread < 8 && j < m) { const double a = clip_lo(p[j]); s0 = fma(a, a, s0); }
    } else {
        const float* p = (const float*)t.in[i] + at;
#pragma unroll UNROLL
        for (int j = thread * 4; j + 4 <= m; j += THREADS * 4) {
            const clip_u4 q = *(const clip_u4*)(p + j);
#pragma unroll
            for (int k = 0; k < 4; k += 2) {
                const double a = __uint_as_float(q.v[k]), b = __uint_as_float(q.v[k + 1]);
                s0 = fma(a, a, s0); s1 = fma(b, b, s1);
            }
        }
        const int j = (m & ~3) + thread;
        if (thread < 4 && j < m) { const double a = p[j]; s0 = fma(a, a, s0); }
    }
    return s0 + s1;
}

// max_norm / N as part * 2^power, |part| in [1/2, 1]: N may pass float32's range and the factor fall below it where the clipped
// gradients do neither.  1 where nothing is to be clipped, or where a gradient is not finite.
struct ClipFactor {
    float part;
    int32_t power;
    __device__ __forceinline__ ClipFactor() {}
    __device__ __forceinline__ ClipFactor(double norm, double max_norm) : part(1.0f), power(0) {
        if (norm > max_norm && norm < INFINITY) part = (float)frexp(max_norm / norm, &power);
    }
    __device__ __forceinline__ bool one() const { return part == 1.0f && power == 0; }
    __device__ __forceinline__ float operator*(float g) const { return ldexpf(g * part, power); }
};

template <int THREADS, int UNROLL>
__device__ __forceinline__ void clip_scale(const ClipTable& t, uint32_t i, int64_t at, int m, int thread, ClipFactor f) {
    if (t.size[i] < 0) {
        const uint16_t* p = (const uint16_t*)t.in[i] + at;
        uint16_t* o = (uint16_t*)t.out[i] + at;
#pragma unroll UNROLL
        for (int j = thread * 8; j + 8 <= m; j += THREADS * 8) {
            clip_u4 q = *(const clip_u4*)(p + j);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const __bf16 a = (__bf16)(f * clip_lo(q.v[k])), b = (__bf16)(f * clip_hi(q.v[k]));
                q.v[k] = (uint32_t)__builtin_bit_cast(uint16_t, a) | (uint32_t)__builtin_bit_cast(uint16_t, b) << 16;
            }
            clip_put(o + j, q);
        }
        const int j = (m & ~7) + thread;
        if (thread < 8 && j < m) ((__bf16*)o)[j] = (__bf16)(f * clip_lo(p[j]));
    } else {
        const float* p = (const float*)t.in[i] + at;
        float* o = (float*)t.out[i] + at;
#pragma unroll UNROLL
        for (int j = thread * 4; j + 4 <= m; j += THREADS * 4) {
            clip_u4 q = *(const clip_u4*)(p + j);
#pragma unroll
            for (int k = 0; k < 4; ++k) q.v[k] = __float_as_uint(f * __uint_as_float(q.v[k]));
            clip_put(o + j, q);
        }
        const int j = (m & ~3) + thread;
        if (thread < 4 && j < m) o[j] = f * p[j];
    }
}
__device__ __forceinline__ int clip_part(const ClipTable& t, uint32_t i, int64_t at, int block) {
    const int64_t n = t.size[i] < 0 ? -t.size[i] : t.size[i];
    return (int)min((int64_t)block, n - at);
}

__global__ __launch_bounds__(256) void k_clip_squares(ClipTable t, double* __restrict__ part) {
    __shared__ double red[4];
    const uint32_t i = ClipFind(t)(blockIdx.x);
    const int64_t at = (int64_t)(blockIdx.x - t.first[i]) * t.block;
    const double s = clip_block_sum(clip_squares<256, 4>(t, i, at, clip_part(t, i, at, t.block), threadIdx.x), red);
    if (threadIdx.x == 0) part[t.block0 + blockIdx.x] = s;
}

// the norm, and the factor behind it
__global__ __launch_bounds__(1024) void k_clip_norm(const double* __restrict__ part, uint32_t n, double max_norm, float* __restrict__ norm, ClipFactor* __restrict__ factor) {
    __shared__ double red[16];
    double s = 0.0;
#pragma unroll 8
    for (uint32_t i = threadIdx.x; i < n; i += 1024) s += part[i];
    s = sqrt(clip_block_sum(s, red));
    if (threadIdx.x == 0) {
        *norm = (float)s;
        *factor = ClipFactor(s, max_norm);
    }
}

// From the last block to the first, and with stores that leave the caches alone: what k_clip_squares read last is then still
// there (10^8 float32: both passes 196 us, 214 from the first block on; with ordinary stores 231).
__global__ __launch_bounds__(256) void k_clip_scale(ClipTable t, const ClipFactor* __restrict__ factor) {
    const ClipFactor f = *factor;
    const uint32_t block = gridDim.x - 1 - blockIdx.x, i = ClipFind(t)(block);
    if (f.one() && t.in[i] == t.out[i]) return;
    const int64_t at = (int64_t)(block - t.first[i]) * t.block;
    clip_scale<256, 4>(t, i, at, clip_part(t, i, at, t.block), threadIdx.x, f);
}

// Few gradients: all by one workgroup, a wave per piece of CLIP_PIECE elements.
__global__ __launch_bounds__(1024) void k_clip_one(ClipTable t, double max_norm, float* __restrict__ norm) {
    __shared__ double red[16];
    const int lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), pieces = t.first[t.n];
    const ClipFind find(t);
    double s = 0.0;
    for (uint32_t p = wave; p < pieces; p += 16) {
        const uint32_t i = find(p);
        const int64_t at = (int64_t)(p - t.first[i]) * CLIP_PIECE;
        s += clip_squares<64, 4>(t, i, at, clip_part(t, i, at, CLIP_PIECE), lane);
    }
    s = sqrt(clip_block_sum(s, red));
    const ClipFactor f(s, max_norm);
    if (threadIdx.x == 0) *norm = (float)s;
    for (uint32_t p = wave; p < pieces; p += 16) {
        const uint32_t i = find(p);
        if (f.one() && t.in[i] == t.out[i]) continue;
        const int64_t at = (int64_t)(p - t.first[i]) * CLIP_PIECE;
        clip_scale<64, 4>(t, i, at, clip_part(t, i, at, CLIP_PIECE), lane, f);
    }
}
