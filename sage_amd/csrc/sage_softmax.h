// Softmax over a whole vocabulary: log probabilities of given tokens with entropy and the most likely alternatives, and
// the gradient of both, without ever storing the [tokens][vocabulary] matrix of logits.
//
//   s_nv = x_n . w_v + b_v                 lse_n = log sum_v exp s_nv          p_nv = exp(s_nv - lse_n)
//   logprob_n = s_n,t(n) - lse_n           H_n = lse_n - sum_v p_nv s_nv
//   G_nv = g_n (1[v = t(n)] - p_nv) - h_n p_nv (log p_nv + H_n)     (g, h: the gradients of logprob and H)
//   dx = G w      dw = G^T x      db_v = sum_n G_nv
//
// Matrix layout.  A "stationary" operand (tokens in the forward pass and for dx, ids for dw) stays in a wave's registers, the
// other one "streams" past it 32 rows at a time, on v_mfma_f32_32x32x16 (M = 32) or, where a wave's registers hold no 32 columns
// (the widest rows, few tokens), v_mfma_f32_16x16x32 (M = 16).  The streaming rows are the matrix's rows and the stationary
// ones its columns: lane l then holds, of column l % M, the values j = 0 .. M / 2 - 1 of rows RS (j / 4) + 4 (l / M) + j % 4, so
// maxima and sums over the streaming axis need no lane to talk to another one until the end, and eight of the weights are, as
// they lie in the registers, an operand of the next product (the transposed fragments list their rows in that order).
// Vector instructions hide behind the 32x32 MFMA and hardly behind the 16x16 one (4 waves a SIMD, 16 fma and 3 exp
// beside 131,072 products' MFMAs: 64 ns against 82, the MFMAs alone 55 and 61).
//
// bf16 inputs are multiplied as they are (products of two bf16 are exact in float32).  float32 inputs are taken as the sum of
// two float16 (11 + 11 bits) and three of the four products are formed; what is left out is 2^-22 of |x||w|, the size of
// float32's own rounding in a sum of a few terms, and it costs 3 MFMAs where three bf16 parts cost 6 and the float32 MFMA 16
// (256 against 4,096 operations per clock and CU).  float16's narrow range is met by powers of two, exact in both
// directions: a row has one that brings its largest element to 2^13 (32 rows share one where they differ by no more than 2^8),
// and the weights of a column share one that follows their largest (both below).  Where the weights are read only once (few tokens), the three bf16 parts are formed on
// the way instead: they need no scale.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>

typedef __bf16 vs_bf8 __attribute__((ext_vector_type(8)));
typedef float vs_f4 __attribute__((ext_vector_type(4)));
typedef float vs_f8 __attribute__((ext_vector_type(8)));
typedef float vs_f16 __attribute__((ext_vector_type(16)));

template <int M> struct VsTile;
template <> struct VsTile<16> {
    using Acc = vs_f4;
    static constexpr int K = 32, NB = 2, RS = 16;      // summation slots, row tiles of 32 rows
};
template <> struct VsTile<32> {
    using Acc = vs_f16;
    static constexpr int K = 16, NB = 1, RS = 8;
};
template <int M> constexpr int VS_NJ = M / 2;          // values of a lane in 32 rows x M columns
template <int M> constexpr int VS_HALVES = M / 16;     // operands of the second product they make
template <int M> __device__ __forceinline__ int vs_row(int j, int lane) { return (j >> 2) * VsTile<M>::RS + (lane / M) * 4 + (j & 3); }

#define VS_LOG2E 1.4426950408889634f
#define VS_LN2 0.6931471805599453f
#define VS_CHUNK 8             // ids per stored maximum (the unit in which alternatives are looked for)
#define VS_BLOCK 256           // ids are dealt out in blocks of this many
// A chunk is eight of 32 ids that one lane sees, of a tile of either width: its maximum needs no other lane.  Chunk c: of block
// c / 32 the ids 32 (c % 8) .. + 31, of these rows 4 p .. and 16 + 4 p .. with p = c / 8 % 4.
__device__ __forceinline__ int vs_chunk_row(int c, int i) {      // the i-th of the 8 ids of a chunk
    return (c >> 5) * VS_BLOCK + (c & 7) * 32 + (i >> 2) * 16 + ((c >> 3) & 3) * 4 + (i & 3);
}
#define VS_NOTHING (-1.0e30f)  // reference of a row that has seen no finite logit yet; a bias this low masks its id
#define VS_MASKED (-3.0e30f)   // what a masked logit is raised to: p is 0 there, and p times the exponent too
#define VS_SLACK 4096.0f       // a lane's terms of 32 rows that sum to more than this move the running reference
#define VS_TMIN (-200.0f)      // 2^-200 is 0 in float32

struct VsSrc {                 // a row-major matrix of float32 or bf16
    const void* p;
    int64_t ld;                // elements from one row to the next
    int32_t rows, dim;
    int32_t is_bf16;
};

__device__ __forceinline__ float vs_load(const VsSrc& s, int64_t row, int d) {
    return s.is_bf16 ? __uint_as_float((uint32_t)((const uint16_t*)s.p)[row * s.ld + d] << 16) : ((const float*)s.p)[row * s.ld + d];
}

// max(a, b) that keeps a NaN (fmaxf would turn a NaN logit into a masked one, and takes an instruction more to do it)
__device__ __forceinline__ float vs_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// eight 16-bit elements of a fragment: bf16, or float16 where values are in two parts
typedef uint32_t vs_bits __attribute__((ext_vector_type(4)));
typedef _Float16 vs_h8 __attribute__((ext_vector_type(8)));

template <int PL, int M>
__device__ __forceinline__ typename VsTile<M>::Acc vs_mfma(vs_bits a, vs_bits b, typename VsTile<M>::Acc c) {
    const vs_h8 ah = __builtin_bit_cast(vs_h8, a), bh = __builtin_bit_cast(vs_h8, b);
    const vs_bf8 ab = __builtin_bit_cast(vs_bf8, a), bb = __builtin_bit_cast(vs_bf8, b);
    if constexpr (M == 32) return PL == 2 ? __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bh, c, 0, 0, 0) : __builtin_amdgcn_mfma_f32_32x32x16_bf16(ab, bb, c, 0, 0, 0);
    else return PL == 2 ? __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, bh, c, 0, 0, 0) : __builtin_amdgcn_mfma_f32_16x16x32_bf16(ab, bb, c, 0, 0, 0);
}

// c[r][t] += a[r] . b[t] for R x TB independent accumulators, both operands in PL parts (largest first): the products are the
// outer loop, small ones first, so that an accumulator is not needed again right after it was written.
template <int PL, int M, int R, int TB, class B>
__device__ __forceinline__ void vs_mfma_parts(const vs_bits (&a)[R][PL], const B& b, typename VsTile<M>::Acc (&c)[R][TB]) {
    constexpr int pa[6] = {1, 2, 0, 1, 0, 0}, pb[6] = {1, 0, 2, 0, 1, 0};
#pragma unroll
    for (int q = PL == 3 ? 0 : PL == 2 ? 3 : 5; q < 6; ++q)
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int t = 0; t < TB; ++t) c[r][t] = vs_mfma<PL, M>(a[r][pa[q]], b(t, pb[q]), c[r][t]);
}

// v as the sum of PL parts, each rounded to nearest: one bf16 (within 2^-9 |v|), two float16 (within 2^-23 |v| if |v| is between
// 2^-3 and 2^15), three bf16 (exact).  Two elements at a time.
template <int PL>
__device__ __forceinline__ void vs_split(vs_f8 v, vs_bits* out) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int p = 0; p < PL; ++p) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f2 pair = {v[2 * i], v[2 * i + 1]};
            if constexpr (PL == 2) {
                const h2 h = __builtin_convertvector(pair, h2);
                out[p][i] = __builtin_bit_cast(uint32_t, h);
                if (p + 1 < PL) { v[2 * i] -= (float)h[0]; v[2 * i + 1] -= (float)h[1]; }
            } else {
                const uint32_t u = __builtin_bit_cast(uint32_t, __builtin_convertvector(pair, b2));
                out[p][i] = u;
                if (p + 1 < PL) { v[2 * i] -= __uint_as_float(u << 16); v[2 * i + 1] -= __uint_as_float(u & 0xFFFF0000u); }
            }
        }
    }
}

// ---- fragments ----------------------------------------------------------------------------------------------------
// 2 KS fragments of either kind for 32 rows, each [PL][lane] of eight elements.  S fragments (M rows x K elements): lane l
// holds row l % M, elements 8 (l / M) .. .  T fragments (M elements x K rows): lane l holds element l % M and eight rows in the
// order that a lane has values in.  Rows past the end and elements past `dim` are zero.  A fragment is one
// coalesced 1 KiB load of a wave, whatever the caller's row length, stride and alignment are.  One workgroup packs 32 rows:
// a lane loads the eight elements that its place in an S fragment asks for; T fragments are read back through LDS.
// PL = 2: a row is multiplied by 2^e, e such that its largest finite element comes to just under 2^13, or that of the 32 rows, if no row
// is smaller by more than 2^VS_SPREAD: elements are then off by at most 2^-37 of that largest one, or 2^-29 of their own row's, a 32nd of a
// float32's step.  (One scale for 32 rows, whatever they hold, would take all bits of rows beside one 10^9 times larger.)  Bound by HBM:
// 131,072 x 300 bf16 for a forward pass, 79 MB read and 84 MB written, 37 us (4.4 TB/s); rows of 511 bf16, that start at any
// 2-byte boundary, 84 MB in all in 23 us (33 with unaligned loads in place of aligned words).

// eight elements from `d` on; zeros past the end of the row
template <int PL>
__device__ __forceinline__ vs_f8 vs_eight(const VsSrc& s, int64_t row, int d) {
    vs_f8 v;
    if (d + 8 <= s.dim) {
        if constexpr (PL == 1) {
            struct __attribute__((packed, aligned(2))) Raw { uint32_t v[4]; };
            const uint16_t* p = (const uint16_t*)s.p + row * s.ld + d;
            if (((s.ld & 1) || ((uintptr_t)s.p & 2)) && row > 0 && row + 1 < s.rows) {
                // rows at odd 2-byte boundaries: the five words that the eight elements lie in (between two other rows: in bounds)
                struct __attribute__((packed, aligned(4))) Words { uint32_t v[4]; };
                const uint32_t* q = (const uint32_t*)((uintptr_t)p & ~(uintptr_t)3);
                const Words a = *(const Words*)q;
                const uint32_t last = q[4], by = ((uint32_t)(uintptr_t)p & 2) * 8;
                Raw r;
#pragma unroll
                for (int i = 0; i < 4; ++i) r.v[i] = __builtin_amdgcn_alignbit(i < 3 ? a.v[i + 1] : last, a.v[i], by);
                v = __builtin_convertvector(__builtin_bit_cast(vs_bf8, r), vs_f8);
            } else v = __builtin_convertvector(__builtin_bit_cast(vs_bf8, *(const Raw*)p), vs_f8);
        } else {
            struct __attribute__((packed, aligned(4))) Raw { float v[8]; };
            v = __builtin_bit_cast(vs_f8, *(const Raw*)((const float*)s.p + row * s.ld + d));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = d + i < s.dim ? vs_load(s, row, d + i) : 0.0f;
    }
    return v;
}

// What goes with the fragments of 32 ids: their biases (0 where the caller gives none, -inf past the end: p = 0 there), then
// the exponent of their scale, their largest size, whether their scales differ, and by how much each row's exponent
// exceeds the common one (a byte each; 0 where they share it).  A mask of the type's lowest value becomes -inf too: next to it no logit
// keeps a bit, and float32 could not hold it in powers of two.  PL = 2 keeps the biases in powers of two.
#define VS_SPREAD 8
#define VS_INFO 44
#define VS_INFO_EXP 32
#define VS_INFO_WIDE 33
#define VS_INFO_DIFFER 34
#define VS_INFO_MORE 36
// What goes with those of 32 tokens in the gradient: lse in powers of two (L), A and B of G = p (A + B e), e = log2 p, for the ids
// that are not the target; the target, and its own G (gl until k_vs_target has formed it); the exponents as above.
#define VS_TOKEN 172
#define VS_TOKEN_A 32
#define VS_TOKEN_B 64
#define VS_TOKEN_GT 96
#define VS_TOKEN_TARGET 128
#define VS_TOKEN_EXP 160
#define VS_TOKEN_DIFFER 161
#define VS_TOKEN_MORE 164
__device__ __forceinline__ float vs_more(const float* more, int row) { return (float)((const uint8_t*)more)[row]; }

struct VsPack {
    VsSrc src;
    uint4 *S, *T;              // T: of a gradient, or null
    float* exps;               // PL = 2, of tokens in a forward pass: e of each row, its own whatever the others are; or null
    int32_t groups;            // of 32 rows
    // ids: their biases (`bias` or null)
    float* info;               // null: not of ids
    const float* bias;
    // tokens of a gradient
    float* tokens;             // null: not of those
    const float *lse, *entropy, *g, *h;
    const int64_t* targets;
    int32_t vocab;
};

// A token that has no part in the gradient, whatever its x, lse and entropy hold
__device__ __forceinline__ bool vs_idle(const VsPack& a, int64_t i) {
    const bool of_target = a.g && a.targets && a.targets[i] >= 0 && a.g[i] != 0.0f;
    return !of_target && !(a.h && a.h[i] != 0.0f);
}
// lse in powers of two; what p is to be multiplied by to make up for its rounding
__device__ __forceinline__ float vs_lse2(float l, float& fix) {
    const double exact = (double)l * 1.4426950408889634;
    const float l2 = (float)exact;
    fix = exp2f((float)((double)l2 - exact));
    return l2;
}
__device__ __forceinline__ void vs_put_token(const VsPack& a, int64_t i) {
    // rows past the end, idle ones and rows whose every id is masked: an lse that makes every p 0, whatever the bias is
    float l2 = -VS_NOTHING, A = 0.0f, B = 0.0f, gl = 0.0f;
    int32_t t = -1;
    if (i < a.src.rows && !vs_idle(a, i)) {
        const float l = a.lse[i];
        const int64_t tt = a.targets ? a.targets[i] : -1;
        const bool empty = l == -INFINITY;
        float fix = 1.0f;                         // p is short of 2^-(rounding of l2); A and B make up for it
        if (!empty) l2 = vs_lse2(l, fix);
        if (tt >= 0 && a.g) gl = a.g[i];
        if (tt >= a.vocab) gl = NAN;
        t = tt >= 0 && tt < a.vocab ? (int32_t)tt : -1;
        A = -gl;
        if (a.h && a.h[i] != 0.0f && !empty) { A -= a.h[i] * a.entropy[i]; B = -a.h[i] * VS_LN2; }
        A *= fix; B *= fix;
    }
    float* to = a.tokens + (i >> 5) * VS_TOKEN + (i & 31);
    to[0] = l2; to[VS_TOKEN_A] = A; to[VS_TOKEN_B] = B; to[VS_TOKEN_GT] = gl; to[VS_TOKEN_TARGET] = __int_as_float(t);
}

// Two matrices in one launch: the first workgroups pack `a`, the others `b`.
template <int KS, int PL, int M, bool FORWARD>
__global__ __launch_bounds__(256) void k_vs_pack(VsPack pa, VsPack pb) {
    const bool second = (int)blockIdx.x >= pa.groups;
    const VsPack& a = second ? pb : pa;
    const int64_t group = second ? (int64_t)blockIdx.x - pa.groups : blockIdx.x;
    constexpr int DP = KS * 32, LD = DP + 4, N = (KS + 1) / 2;      // fragments of a wave
    __shared__ float tile[FORWARD ? 1 : 32 * LD];      // (a forward pass has no use for T, and more workgroups at a time without it)
    __shared__ float wmax[4], rmax[4][32];
    constexpr int K = VsTile<M>::K, STEPS = DP / K;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane % M;
    auto row_of = [&](int f) { return f / STEPS * M + col; };
    auto element_of = [&](int f) { return f % STEPS * K + lane / M * 8; };
    const int64_t row0 = group * 32;
    bool there[32 / M];                        // rows past the end, of masked ids and of idle tokens are taken as 0, whatever they hold
#pragma unroll
    for (int r = 0; r < 32 / M; ++r) {
        const int64_t row = row0 + r * M + col;
        there[r] = row < a.src.rows && !(a.bias && a.bias[row] <= VS_NOTHING) && !(a.tokens && vs_idle(a, row));
    }
    vs_f8 v[N];
    float big = 0.0f, fin[32 / M];             // of all, and the largest finite size of each of this lane's rows
#pragma unroll
    for (int r = 0; r < 32 / M; ++r) fin[r] = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int f = i * 4 + wave;
        v[i] = vs_f8(0.0f);
        if (f < 2 * KS && there[f / STEPS ? 32 / M - 1 : 0] && element_of(f) < a.src.dim) v[i] = vs_eight<PL>(a.src, row0 + row_of(f), element_of(f));
        float most = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float q = fabsf(v[i][j]);
            big = fmaxf(big, q);
            most = fmaxf(most, q < INFINITY ? q : 0.0f);
        }
#pragma unroll
        for (int r = 0; r < 32 / M; ++r) fin[r] = fmaxf(fin[r], f / STEPS == r ? most : 0.0f);
    }
    for (int o = 1; o < 64; o <<= 1) big = fmaxf(big, __shfl_xor(big, o));
    if (lane == 0) wmax[wave] = big;
    if (PL == 2)
#pragma unroll
        for (int r = 0; r < 32 / M; ++r) {
            for (int o = M; o < 64; o <<= 1) fin[r] = fmaxf(fin[r], __shfl_xor(fin[r], o));
            if (lane < M) rmax[wave][r * M + col] = fin[r];
        }
    __syncthreads();
    big = fmaxf(fmaxf(wmax[0], wmax[1]), fmaxf(wmax[2], wmax[3]));
    int e = 0, more = 0, exps[32 / M];         // the common exponent, what row `lane` % 32 has beyond it, those of this lane's rows
    bool differ = false;
#pragma unroll
    for (int r = 0; r < 32 / M; ++r) exps[r] = 0;
    if (PL == 2) {
        const int i = lane & 31;
        const float own = fmaxf(fmaxf(rmax[0][i], rmax[1][i]), fmaxf(rmax[2][i], rmax[3][i]));
        float all = own;
        for (int o = 1; o < 32; o <<= 1) all = fmaxf(all, __shfl_xor(all, o));
        if (all > 0.0f) e = 13 - __builtin_amdgcn_frexp_expf(all);
        if (own > 0.0f) more = min(13 - __builtin_amdgcn_frexp_expf(own) - e, 255);
        differ = a.exps || __any(more > VS_SPREAD);
        if (!differ) more = 0;
#pragma unroll
        for (int r = 0; r < 32 / M; ++r) exps[r] = e + __shfl(more, r * M + col);
    }
    if (threadIdx.x == 0) {
        if (a.info) {
            a.info[group * VS_INFO + VS_INFO_WIDE] = big;
            a.info[group * VS_INFO + VS_INFO_EXP] = (float)e;
            a.info[group * VS_INFO + VS_INFO_DIFFER] = differ ? 1.0f : 0.0f;
        }
        if (a.tokens) {
            a.tokens[group * VS_TOKEN + VS_TOKEN_EXP] = (float)e;
            a.tokens[group * VS_TOKEN + VS_TOKEN_DIFFER] = differ ? 1.0f : 0.0f;
        }
    }
    if (threadIdx.x < 32) {
        const int64_t row = row0 + threadIdx.x;
        if (a.exps) a.exps[row] = (float)(e + more);
        if (a.info) ((uint8_t*)&a.info[group * VS_INFO + VS_INFO_MORE])[threadIdx.x] = (uint8_t)more;
        if (a.tokens) ((uint8_t*)&a.tokens[group * VS_TOKEN + VS_TOKEN_MORE])[threadIdx.x] = (uint8_t)more;
        if (a.info) {
            const float b = row >= a.src.rows ? -INFINITY : a.bias ? a.bias[row] : 0.0f;
            a.info[group * VS_INFO + threadIdx.x] = b <= VS_NOTHING ? -INFINITY : PL == 2 ? b * VS_LOG2E : b;
        }
        if (a.tokens) vs_put_token(a, row);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int f = i * 4 + wave;
        if (f >= 2 * KS) continue;
        if (PL == 2)
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = ldexpf(v[i][j], exps[f / STEPS ? 32 / M - 1 : 0]);
        if (!FORWARD && a.T) {
            float* to = tile + row_of(f) * LD + element_of(f);
            *(vs_f4*)to = vs_f4{v[i][0], v[i][1], v[i][2], v[i][3]};
            *(vs_f4*)(to + 4) = vs_f4{v[i][4], v[i][5], v[i][6], v[i][7]};
        }
        vs_bits part[PL];
        vs_split<PL>(v[i], part);
#pragma unroll
        for (int p = 0; p < PL; ++p) *(vs_bits*)&a.S[((group * 2 * KS + f) * PL + p) * 64 + lane] = part[p];
    }
    if (FORWARD || !a.T) return;
    __syncthreads();
    for (int f = wave; f < 2 * KS; f += 4) {
        vs_f8 q;
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j] = tile[vs_row<M>(f % VS_HALVES<M> * 8 + j, lane) * LD + f / VS_HALVES<M> * M + col];
        vs_bits part[PL];
        vs_split<PL>(q, part);
#pragma unroll
        for (int p = 0; p < PL; ++p) *(vs_bits*)&a.T[((group * 2 * KS + f) * PL + p) * 64 + lane] = part[p];
    }
}

// All are known before any is written back: without this the compiler takes new registers for what a rarely taken branch
// changes, and copies the old ones into them each time the branch is not taken.  The values come
// from vector instructions (the compiler sees to the waits that a matrix instruction's result needs before those read it).
template <class V>
__device__ __forceinline__ void vs_in_place(V& v) {
    constexpr int N = sizeof(V) / 4;
    float a[N];
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] = v[i];
    if constexpr (N == 4) asm volatile("" : "+v"(a[0]), "+v"(a[1]), "+v"(a[2]), "+v"(a[3]));
    else
        asm volatile("" : "+v"(a[0]), "+v"(a[1]), "+v"(a[2]), "+v"(a[3]), "+v"(a[4]), "+v"(a[5]), "+v"(a[6]), "+v"(a[7]), "+v"(a[8]), "+v"(a[9]),
                     "+v"(a[10]), "+v"(a[11]), "+v"(a[12]), "+v"(a[13]), "+v"(a[14]), "+v"(a[15]));
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = a[i];
}

// 2^n as a factor of log2(e), kept finite (logits beyond float32 are inf or 0 all the same)
__device__ __forceinline__ float vs_unit(float n) { return ldexpf(VS_LOG2E, (int)__builtin_amdgcn_fmed3f(n, -126.0f, 126.0f)); }

// ---- forward ------------------------------------------------------------------------------------------------------
struct VsFwd {
    const uint4 *xS, *wS;
    const float* info;         // [ids / 32][VS_INFO]
    const float* x_exp;        // PL = 2: [tokens]
    int32_t has_bias;          // the caller gave one: -inf may stand anywhere (else only past `vocab`)
    int32_t vocab;
    const int64_t* targets;    // of `rows` tokens, or null
    int32_t rows;
    int32_t n_tiles;           // token tiles of TB M rows
    int32_t splits;            // ranges of the vocabulary
    int32_t blocks;            // blocks of VS_BLOCK ids
    int32_t chunks;            // chunks of VS_CHUNK ids: 32 a block
    int64_t n_pad;             // row length of the partials
    float4* part;              // [splits][n_pad]: reference (in powers of two), sum of exps, sum of exp * exponent, sum of exps without the target's
    float* wide;               // [splits]: largest |weight|
    _Float16* chunk_max;       // [n_pad][chunks] or null: largest logits, -inf where all are masked
};

// Sums of a row, relative to 2^ref: s of exp, e of exp * exponent (the entropy's), R of exp over all ids but the target (1 - p_t, to its own
// last bits where p_t is near 1: the log probability is then log(1 - R / S)).  A softmax in one pass: the reference is
// moved to the running maximum only when a step's terms have outgrown it by VS_SLACK, a few times per row; the common step
// neither rescales nor looks for a maximum.  Eight terms are summed first, then up to VS_BLOCK / 4 of those, then these: sums of 262,144 terms keep
// their last bits.
struct VsStat {
    float ref, s, e, S, E, R;
    __device__ __forceinline__ void clear() { ref = VS_NOTHING; s = e = S = E = R = 0.0f; }
    __device__ __forceinline__ void flush() { S += s; E += e; s = e = 0.0f; }
    __device__ __forceinline__ void move(float now) {      // (a sum that vanishes takes its exponents with it: 0 * inf)
        const float d = ref - now, f = exp2f(d);
        e = f == 0.0f ? 0.0f : f * fmaf(d, s, e);
        E = f == 0.0f ? 0.0f : f * fmaf(d, S, E);
        s *= f; S *= f; R *= f;
        ref = now;
    }
    __device__ __forceinline__ void join(float r2, float s2, float e2, float R2) {     // S, E and R with another range's
        const float now = fmaxf(ref, r2);
        if (now > ref) move(now);
        const float d = r2 - now, f = exp2f(d);
        E += f == 0.0f ? 0.0f : f * fmaf(d, s2, e2);
        S += s2 != s2 ? s2 : f * s2;
        R += f * R2;
    }
};

template <int KS, int PL, int M>
using VsOperand = vs_bits[KS * 32 / VsTile<M>::K][PL];         // the fragments of M stationary rows
template <int M, int TB>
using VsLogits = typename VsTile<M>::Acc[VsTile<M>::NB][TB];
template <int M, int TB>
__device__ __forceinline__ float vs_value(const VsLogits<M, TB>& s, int t, int j) {
    constexpr int NI = VS_NJ<M> / VsTile<M>::NB;
    return s[j / NI][t][j % NI];
}
template <int M, int TB>
__device__ __forceinline__ void vs_set(VsLogits<M, TB>& s, int t, int j, float v) {
    constexpr int NI = VS_NJ<M> / VsTile<M>::NB;
    s[j / NI][t][j % NI] = v;
}

// 32 streaming rows against the stationary ones: s += w . x
template <int KS, int PL, int M, int TB>
__device__ __forceinline__ void vs_product(const uint4* w, const VsOperand<KS, PL, M> (&x)[TB], VsLogits<M, TB>& s) {
    constexpr int STEPS = KS * 32 / VsTile<M>::K, NB = VsTile<M>::NB;
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
        vs_bits wf[NB][PL];
#pragma unroll
        for (int rb = 0; rb < NB; ++rb)
#pragma unroll
            for (int p = 0; p < PL; ++p) wf[rb][p] = *(const vs_bits*)&w[((rb * STEPS + k) * PL + p) * 64];
        vs_mfma_parts<PL, M, NB, TB>(wf, [&](int t, int p) { return x[t][k][p]; }, s);
    }
}

template <int KS, int PL, int M, int TB>
__device__ __forceinline__ void vs_stationary(const uint4* S, int64_t tile, int lane, VsOperand<KS, PL, M> (&x)[TB]) {
    constexpr int STEPS = KS * 32 / VsTile<M>::K;
#pragma unroll
    for (int t = 0; t < TB; ++t)
#pragma unroll
        for (int k = 0; k < STEPS; ++k)
#pragma unroll
            for (int p = 0; p < PL; ++p) x[t][k][p] = *(const vs_bits*)&S[(((tile * TB + t) * STEPS + k) * PL + p) * 64 + lane];
}

template <int M, int TB>
struct VsRowsOfTile {
    static constexpr int NJ = VS_NJ<M>;
    static constexpr int C = NJ / VS_CHUNK;    // chunks of a lane in 32 ids
    VsStat st[TB];
    float top[TB][C], even[TB][C], wide;       // wide: the largest size of a weight
    uint32_t keep[TB][C][3];
    int target[TB];                            // -1: none
    __device__ __forceinline__ void clear(const VsFwd& a, int64_t row0, bool live) {     // of the tile's first row
#pragma unroll
        for (int t = 0; t < TB; ++t) {
            st[t].clear();
            const int64_t row = row0 + t * M + threadIdx.x % M;
            const int64_t v = live && a.targets && row < a.rows ? a.targets[row] : -1;
            target[t] = v >= 0 && v < a.vocab ? (int)v : -1;
        }
        wide = 0.0f;
    }
    // the logits of 32 ids, in powers of two after multiplication by unit[t]; TOP: their largest is kept
    template <bool TOP, bool SCALED, bool ONCE = false>
    __device__ __forceinline__ void add(int row0, const VsLogits<M, TB>& s, const float (&unit)[TB]) {
        float ls[TB], le[TB], lr[TB];
        bool here = false;
#pragma unroll
        for (int t = 0; t < TB; ++t) here |= (uint32_t)(target[t] - row0) < 32;
        // A logit of -inf has p = 0, and an exponent that 0 times is NaN: the second look, rarely taken, stops exponents where p is 0.
        // ONCE: so does the first (kernels bound by memory: 5 tokens x 229,376 ids of bf16 55.3 us, 57.3 with a second look).
        auto sums = [&](auto again) {
            float most = 0.0f;
#pragma unroll
            for (int t = 0; t < TB; ++t) {
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    float e = fmaf(vs_value<M, TB>(s, t, j), SCALED ? unit[t] : VS_LOG2E, -st[t].ref);
                    if (decltype(again)::value) e = vs_max(e, VS_TMIN);
                    const float p = __builtin_amdgcn_exp2f(e);
                    ls[t] = j ? ls[t] + p : p;
                    le[t] = j ? fmaf(p, e, le[t]) : p * e;
                }
                most = ONCE ? fmaxf(most, ls[t]) : vs_max(most, fmaf(le[t], 0.0f, ls[t]));
            }
            return most;
        };
        if (__any(!(sums(std::integral_constant<bool, ONCE>{}) <= VS_SLACK))) {
#pragma unroll
            for (int t = 0; t < TB; ++t) st[t].move(ls[t] > VS_SLACK ? largest(s, t) * (SCALED ? unit[t] : VS_LOG2E) : st[t].ref);
            sums(std::true_type{});
        }
#pragma unroll
        for (int t = 0; t < TB; ++t) lr[t] = ls[t];
        if (__any(here))                       // (rare: a token has one target)
#pragma unroll
            for (int t = 0; t < TB; ++t) {
                const int at = target[t] - row0 - vs_row<M>(0, threadIdx.x & 63);
                lr[t] = 0.0f;
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    const float p = __builtin_amdgcn_exp2f(fmaf(vs_value<M, TB>(s, t, j), SCALED ? unit[t] : VS_LOG2E, -st[t].ref));
                    lr[t] += at == vs_row<M>(j, 0) ? 0.0f : p;
                }
            }
#pragma unroll
        for (int t = 0; t < TB; ++t) {
            st[t].s += ls[t];
            st[t].e += le[t];
            st[t].R += lr[t];
            if (TOP)
#pragma unroll
                for (int c = 0; c < C; ++c) top[t][c] = SCALED ? of_chunk(s, t, c) * (unit[t] * VS_LN2) : of_chunk(s, t, c);
        }
    }
    static __device__ __forceinline__ float of_chunk(const VsLogits<M, TB>& s, int t, int c) {
        auto v = [&](int i) { return vs_value<M, TB>(s, t, C == 1 ? i : (i >> 2) * 8 + c * 4 + (i & 3)); };
        return vs_max(vs_max(vs_max(vs_max(vs_max(vs_max(vs_max(v(0), v(1)), v(2)), v(3)), v(4)), v(5)), v(6)), v(7));
    }
    static __device__ __forceinline__ float largest(const VsLogits<M, TB>& s, int t) {
        return C == 1 ? of_chunk(s, t, 0) : vs_max(of_chunk(s, t, 0), of_chunk(s, t, C - 1));
    }
    // Step h of a block (32 ids) is done: its largest logits are kept as float16 (-inf stands for masked ids alone) and those of
    // eight steps are stored together (WHOLE: the wave sees whole blocks), or of two.
    template <bool WHOLE>
    __device__ __forceinline__ void chunk(const VsFwd& a, int64_t tile, int block, int h, int lane, bool live) {
#pragma unroll
        for (int t = 0; t < TB; ++t)
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const float m = a.has_bias && top[t][c] < VS_NOTHING ? -INFINITY : top[t][c];
                if ((h & 1) == 0) { even[t][c] = m; continue; }
                const uint32_t two = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(even[t][c], m));     // (stays finite)
                _Float16* to = a.chunk_max + ((tile * TB + t) * M + lane % M) * a.chunks + block * 32 + (lane / M + c * 2) * 8;
                if (!WHOLE) { if (live) *(uint32_t*)(to + h - 1) = two; }
                else if (h == 1) keep[t][c][0] = two;
                else if (h == 3) keep[t][c][1] = two;
                else if (h == 5) keep[t][c][2] = two;
                else if (live) *(uint4*)to = make_uint4(keep[t][c][0], keep[t][c][1], keep[t][c][2], two);
            }
    }
    __device__ __forceinline__ void flush() {
#pragma unroll
        for (int t = 0; t < TB; ++t) st[t].flush();
    }
    __device__ __forceinline__ void join_lanes() {
#pragma unroll
        for (int t = 0; t < TB; ++t) {
            st[t].flush();
#pragma unroll
            for (int o = M; o <= 32; o <<= 1) {
                const float r2 = __shfl_xor(st[t].ref, o), s2 = __shfl_xor(st[t].S, o), e2 = __shfl_xor(st[t].E, o), R2 = __shfl_xor(st[t].R, o);
                st[t].join(r2, s2, e2, R2);
            }
        }
    }
    __device__ __forceinline__ void store(const VsFwd& a, int64_t tile, int split, int lane) {
        join_lanes();
#pragma unroll
        for (int t = 0; t < TB; ++t)
            if (lane < M) a.part[(int64_t)split * a.n_pad + (tile * TB + t) * M + lane] = make_float4(st[t].ref, st[t].S, st[t].E, st[t].R);
        if (tile == 0 && lane == 0) a.wide[split] = wide;
    }
};

// What the rows that a lane has logits of have beyond the common exponent, four bytes a word
template <int M>
__device__ __forceinline__ void vs_mores(const float* more, int lane, uint32_t (&to)[VS_NJ<M> / 4]) {
#pragma unroll
    for (int q = 0; q < VS_NJ<M> / 4; ++q) to[q] = ((const uint32_t*)more)[vs_row<M>(q * 4, lane) / 4];
}
template <int N>
__device__ __forceinline__ int vs_more_of(const uint32_t (&more)[N], int j) { return (int)(more[j >> 2] >> (j & 3) * 8 & 255); }

// Where the scales of the 32 streaming rows differ, their logits are brought to the common one.
template <int M, int TB>
__device__ __forceinline__ void vs_common(const uint32_t (&more)[VS_NJ<M> / 4], VsLogits<M, TB>& s) {
#pragma unroll
    for (int t = 0; t < TB; ++t) {
#pragma unroll
        for (int j = 0; j < VS_NJ<M>; ++j) vs_set<M, TB>(s, t, j, ldexpf(vs_value<M, TB>(s, t, j), -vs_more_of(more, j)));
#pragma unroll
        for (int b = 0; b < VsTile<M>::NB; ++b) vs_in_place(s[b][t]);
    }
}
__device__ __forceinline__ bool vs_differ(float flag) { return __builtin_amdgcn_readfirstlane(__float_as_int(flag)) != 0; }

// Adds the biases where the product did not start from them, and raises masked logits.
template <int M, int TB, bool SCALED>
__device__ __forceinline__ void vs_mask(VsLogits<M, TB>& s, float (&unit)[TB], const vs_f4 (&b)[VS_NJ<M> / 4]) {
#pragma unroll
    for (int t = 0; t < TB; ++t) {
#pragma unroll
        for (int j = 0; j < VS_NJ<M>; ++j) {
            float v = vs_value<M, TB>(s, t, j);
            if (SCALED) v = fmaf(v, unit[t], b[j >> 2][j & 3]);
            vs_set<M, TB>(s, t, j, vs_max(v, VS_MASKED));
        }
        if (SCALED) unit[t] = 1.0f;
    }
}

// What 32 rows' logits start from: their biases (`of`: by row), or 0 where the product is scaled
template <int PL, int M, int TB>
__device__ __forceinline__ void vs_begin(const float* of, int lane, VsLogits<M, TB>& s, vs_f4 (&b)[VS_NJ<M> / 4]) {
#pragma unroll
    for (int q = 0; q < VS_NJ<M> / 4; ++q) b[q] = *(const vs_f4*)&of[vs_row<M>(q * 4, lane)];
#pragma unroll
    for (int t = 0; t < TB; ++t)
#pragma unroll
        for (int j = 0; j < VS_NJ<M>; ++j) vs_set<M, TB>(s, t, j, PL == 1 ? b[j >> 2][j & 3] : 0.0f);
}

// 32 ids against a tile: their logits are formed and counted
template <int KS, int PL, int M, int TB, bool TOP>
__device__ __forceinline__ void vs_forward_step(const VsFwd& a, int row0, const uint4* w, const float* info, const VsOperand<KS, PL, M> (&x)[TB],
                                                const float (&x_exp)[TB], VsRowsOfTile<M, TB>& rows) {
    if (TOP) rows.wide = fmaxf(rows.wide, info[VS_INFO_WIDE]);
    VsLogits<M, TB> s;
    vs_f4 b[VS_NJ<M> / 4];
    float unit[TB];
    vs_begin<PL, M, TB>(info, threadIdx.x & 63, s, b);
    const float e = PL == 2 ? info[VS_INFO_EXP] : 0.0f;
#pragma unroll
    for (int t = 0; t < TB; ++t) unit[t] = PL == 2 ? vs_unit(-(e + x_exp[t])) : VS_LOG2E;
    vs_product<KS, PL, M, TB>(w, x, s);
    if (PL == 2)
        if (vs_differ(info[VS_INFO_DIFFER])) {
            uint32_t more[VS_NJ<M> / 4];
            vs_mores<M>(info + VS_INFO_MORE, threadIdx.x & 63, more);
            vs_common<M, TB>(more, s);
        }
    if (a.has_bias || row0 + 32 > a.vocab) vs_mask<M, TB, PL == 2>(s, unit, b);      // (the same in the whole grid)
    rows.template add<TOP, PL == 2>(row0, s, unit);
}

// Bound by the matrix units and the power they draw (the clock falls to 1.8 - 2.2 GHz under them), the exponentials beside
// them second.  8,192 tokens x 262,144 ids, D = 50 float32: 764 us (mean of 10, as all below), 0.82 * 10^12 operations of the MFMAs (three
// products, 64 elements for 50) at 1.08 * 10^15 a second, where a large bf16 matrix product of the library reaches 1.37 * 10^15; 4,096 x
// 65,536, D = 300 bf16: 175 us, 0.98 * 10^15.  The MFMAs are busy 55 % of a 1.95 GHz clock in both.
// Four waves, a tile each, share the streaming rows through LDS.  SR rows at a time are copied straight into LDS (they are
// packed in the order of the copy) while the SR before them are worked on: one barrier a step.
typedef const __attribute__((address_space(1))) void* vs_global_ptr;
typedef __attribute__((address_space(3))) void* vs_lds_ptr;
template <int N>               // 16-byte pieces, a multiple of 256
__device__ __forceinline__ void vs_stage(const uint4* from, uint4* to) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < N; i += 256)
        __builtin_amdgcn_global_load_lds((vs_global_ptr)(from + i + wave * 64 + lane), (vs_lds_ptr)(to + i + wave * 64), 16, 0, 0);
}
template <int N>               // floats, at most 256
__device__ __forceinline__ void vs_stage_floats(const float* from, float* to) {
    if (threadIdx.x < N) __builtin_amdgcn_global_load_lds((vs_global_ptr)(from + threadIdx.x), (vs_lds_ptr)(to + (threadIdx.x & ~63)), 4, 0, 0);
}
// This wave's copies into LDS have arrived: vmcnt 0, the other counters as they are.
__device__ __forceinline__ void vs_copies_done() { __builtin_amdgcn_s_waitcnt(0x0F70); }

// A stage: SR rows of fragments and what goes with them.  `to` and `from` are different stages, and the compiler has to know
// it (__restrict__ through an inlined function): else it waits for the copy under way before each read of LDS.
template <int KS, int PL, int M, int SR>
struct VsStage {
    static constexpr int N = SR * KS * PL * 4, INFO = SR / 32 * VS_INFO, SIZE = N + INFO / 4;
    static __device__ __forceinline__ void fetch(const uint4* w, const float* info, uint4* to) {
        vs_stage<N>(w, to);
        vs_stage_floats<INFO>(info, (float*)(to + N));
    }
    template <int TB, bool TOP>
    static __device__ __forceinline__ void step(const VsFwd& a, int base, bool more, const uint4* __restrict__ next, const float* __restrict__ next_info,
                                                uint4* __restrict__ to, const uint4* __restrict__ from, const VsOperand<KS, PL, M> (&x)[TB],
                                                const float (&x_exp)[TB], VsRowsOfTile<M, TB>& rows, int64_t tile, bool live) {
        const int lane = threadIdx.x & 63;
        vs_copies_done();                  // (a barrier alone does not wait for them)
        __syncthreads();                   // `from` has arrived, and nobody reads `to` any more
        if (more) fetch(next, next_info, to);
#pragma unroll 1
        for (int r = 0; r < SR; r += 32) {
            const int row0 = base + r;
            vs_forward_step<KS, PL, M, TB, TOP>(a, row0, from + r * KS * PL * 4 + lane, (const float*)(from + N) + r / 32 * VS_INFO, x, x_exp, rows);
            if (TOP) rows.template chunk<true>(a, tile, row0 / VS_BLOCK, (row0 >> 5) & 7, lane, live);
        }
        if (((base + SR) & (VS_BLOCK - 1)) == 0) rows.flush();
    }
};

// Waves of a SIMD that the registers are shared out for (D = 50, 4,096 x 65,536 bf16: four 90 us, three 97; 8,192 x 262,144 float32: three 765, two 805)
constexpr int vs_fwd_waves(int KS, int PL, bool TOP) { return KS > 2 ? 2 : PL == 2 ? 3 : TOP ? 2 : 4; }
template <int KS, int PL, int M, int TB, int SR, bool TOP>
__global__ __launch_bounds__(256, vs_fwd_waves(KS, PL, TOP)) void k_vs_forward(VsFwd a) {
    using Stage = VsStage<KS, PL, M, SR>;
    __shared__ uint4 buf0[Stage::SIZE], buf1[Stage::SIZE];
    const int lane = threadIdx.x & 63;
    const int split = blockIdx.x % a.splits;
    const int tile = (blockIdx.x / a.splits) * 4 + (threadIdx.x >> 6);
    const bool live = tile < a.n_tiles;
    const int row_begin = (int)((int64_t)a.blocks * split / a.splits) * VS_BLOCK, row_end = (int)((int64_t)a.blocks * (split + 1) / a.splits) * VS_BLOCK;
    VsOperand<KS, PL, M> x[TB];
    vs_stationary<KS, PL, M, TB>(a.xS, live ? tile : 0, lane, x);
    float x_exp[TB];
#pragma unroll
    for (int t = 0; t < TB; ++t) x_exp[t] = PL == 2 ? a.x_exp[((live ? tile : 0) * TB + t) * M + lane % M] : 0.0f;
    VsRowsOfTile<M, TB> rows;
    rows.clear(a, (int64_t)tile * TB * M, live);
    const uint4* w = a.wS + (int64_t)row_begin * KS * PL * 4;
    const float* info = a.info + row_begin / 32 * VS_INFO;
    Stage::fetch(w, info, buf0);
    for (int base = row_begin; base < row_end; base += 2 * SR) {
        w += SR * KS * PL * 4; info += Stage::INFO;
        Stage::template step<TB, TOP>(a, base, true, w, info, buf1, buf0, x, x_exp, rows, tile, live);
        w += SR * KS * PL * 4; info += Stage::INFO;
        Stage::template step<TB, TOP>(a, base + SR, base + 2 * SR < row_end, w, info, buf0, buf1, x, x_exp, rows, tile, live);
    }
    if (live) rows.store(a, tile, split, lane);
}

// The bias of one id: 0 where the caller gives none, -inf where it masks the id.
__device__ __forceinline__ float vs_bias_of(const float* bias, int64_t v) {
    const float b = bias ? bias[v] : 0.0f;
    return b <= VS_NOTHING ? -INFINITY : b;
}

// Few tokens: bound by the one reading of the weights, which are taken as they lie (no packing): a lane loads the eight
// elements of a row that its place in a fragment asks for, at whatever alignment they have.  The last piece of a row that is
// no whole number of pieces long is taken back from the row's end, with the elements before it weighted 0 in x: no read
// leaves the row (so there are eight elements at least).  A wave is a tile of 16 TB tokens against one range of the vocabulary; the
// four of a workgroup join theirs.  One token, 262,144 x 50 float32: 52 MB in 15.2 us (3.4 TB/s); five, 229,376 x 300 bf16: 138 MB in
// 32 us (4.3 TB/s; a copy of 4 GB reaches 4.8).
template <int PL> struct VsPiece;
template <> struct VsPiece<1> {            // of bf16: a fragment as it is
    vs_bf8 v;
    __device__ __forceinline__ void load(const VsSrc& s, int64_t row, int at) {
        struct __attribute__((packed, aligned(2))) Raw { uint32_t v[4]; };
        v = __builtin_bit_cast(vs_bf8, *(const Raw*)((const uint16_t*)s.p + row * s.ld + at));
    }
    __device__ __forceinline__ vs_f8 floats() const { return __builtin_convertvector(v, vs_f8); }
    __device__ __forceinline__ void parts(vs_bits (&out)[1]) const { out[0] = __builtin_bit_cast(vs_bits, v); }
    typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
    u16x8 most;                            // running largest size: the bits of a bf16 without its sign are ordered
    __device__ __forceinline__ void clear() { most = u16x8(0); }
    __device__ __forceinline__ void measure(const VsPiece& q) { most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x8, q.v) & u16x8(0x7FFF)); }
    __device__ __forceinline__ float largest() const {
        unsigned m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, (unsigned)most[i]);
        return __uint_as_float(m << 16);
    }
};
template <> struct VsPiece<3> {            // of float32
    vs_f8 v;
    __device__ __forceinline__ void load(const VsSrc& s, int64_t row, int at) {
        struct __attribute__((packed, aligned(4))) Raw { float v[4]; };
        const Raw r = *(const Raw*)((const float*)s.p + row * s.ld + at), q = *(const Raw*)((const float*)s.p + row * s.ld + at + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[i] = r.v[i]; v[i + 4] = q.v[i]; }
    }
    __device__ __forceinline__ vs_f8 floats() const { return v; }
    __device__ __forceinline__ void parts(vs_bits (&out)[3]) const { vs_split<3>(v, out); }
    __device__ __forceinline__ void clear() { v = vs_f8(0.0f); }
    __device__ __forceinline__ void measure(const VsPiece& q) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = fmaxf(v[i], fabsf(q.v[i]));
    }
    __device__ __forceinline__ float largest() const {
        float m = v[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) m = fmaxf(m, v[i]);
        return m;
    }
};

struct VsRaw {
    VsSrc x, w;
    const float* bias;         // as the caller gave it, or null
    VsFwd f;                   // chunks, blocks, n_pad, part, chunk_max; splits: workgroups of a tile
};
// (One wave a SIMD where two would spill: D = 300 float32, 16 tokens, 131,072 ids 39 us against 67; D = 512 bf16 35 against 51.)
template <int KS, int PL, int TB>
__global__ __launch_bounds__(256, KS * PL > 14 ? 1 : 2) void k_vs_forward_raw(VsRaw a) {
    const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    constexpr int KG = PL == 1 || KS <= 4 ? KS : KS == 8 ? 4 : KS == 10 ? 5 : 2;    // 32-element steps whose loads are under way together
    __shared__ float4 red[4][TB * 16];
    __shared__ float widest[4];
    const int tile = blockIdx.y;
    int at[KS];
    vs_bits x[TB][KS][PL];
#pragma unroll
    for (int k = 0; k < KS; ++k) {
        const int d = k * 32 + quad * 8;
        at[k] = min(d, a.w.dim - 8);
#pragma unroll
        for (int t = 0; t < TB; ++t) {
            const int row = (tile * TB + t) * 16 + col;
            VsPiece<PL> q;
            q.load(a.x, min(row, a.x.rows - 1), at[k]);
            vs_f8 v = q.floats();
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = row < a.x.rows && d < a.w.dim && at[k] + i >= d ? v[i] : 0.0f;
            vs_split<PL>(v, x[t][k]);
        }
    }
    VsRowsOfTile<16, TB> rows;
    rows.clear(a.f, (int64_t)tile * TB * 16, true);
    float wide = 0.0f;
    const float unscaled[TB] = {};
    const int units = gridDim.x * 4, unit = blockIdx.x * 4 + (threadIdx.x >> 6), pieces = a.f.blocks * 4;
    const int c0 = (int)((int64_t)pieces * unit / units), c1 = (int)((int64_t)pieces * (unit + 1) / units);
    for (int c = c0; c < c1; ++c) {
#pragma unroll 1
        for (int row0 = c * 64; row0 < (c + 1) * 64; row0 += 32) {
            // (loads first and together; the bias is added last, so that no wait for it stands before the products)
            VsPiece<PL> raw[2][KG], big[2];
            vs_f4 s[2][TB], b[2];
            float of_row[2] = {0.0f, 0.0f};
            big[0].clear(); big[1].clear();
#pragma unroll
            for (int rb = 0; rb < 2; ++rb)
#pragma unroll
                for (int t = 0; t < TB; ++t) s[rb][t] = vs_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int g = 0; g < KS; g += KG) {
#pragma unroll
                for (int k = 0; k < KG; ++k)
#pragma unroll
                    for (int rb = 0; rb < 2; ++rb)
                        if (g + k < KS) raw[rb][k].load(a.w, min(row0 + rb * 16 + col, a.w.rows - 1), at[g + k]);
                if (g + KG >= KS && a.bias) {
#pragma unroll
                    for (int rb = 0; rb < 2; ++rb) of_row[rb] = a.bias[min(row0 + rb * 16 + col, a.w.rows - 1)];
#pragma unroll
                    for (int j = 0; j < 8; ++j) b[j >> 2][j & 3] = a.bias[min(row0 + (j >> 2) * 16 + quad * 4 + (j & 3), a.w.rows - 1)];
                }
#pragma unroll
                for (int k = 0; k < KG; ++k)
                    if (g + k < KS) {
                        vs_bits wf[2][PL];
#pragma unroll
                        for (int rb = 0; rb < 2; ++rb) {
                            big[rb].measure(raw[rb][k]);
                            raw[rb][k].parts(wf[rb]);
                        }
                        vs_mfma_parts<PL, 16, 2, TB>(wf, [&](int t, int p) { return x[t][g + k][p]; }, s);
                    }
                if (KG < KS) __builtin_amdgcn_sched_barrier(0);     // (the loads of all groups at once would spill)
            }
            if (a.bias || row0 + 32 > a.w.rows) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float q = a.bias ? b[j >> 2][j & 3] : 0.0f;
                    const bool gone = q <= VS_NOTHING || row0 + (j >> 2) * 16 + quad * 4 + (j & 3) >= a.w.rows;
#pragma unroll
                    for (int t = 0; t < TB; ++t) s[j >> 2][t][j & 3] = gone ? VS_MASKED : s[j >> 2][t][j & 3] + q;
                }
            }
            if (a.f.chunk_max) {
#pragma unroll
                for (int rb = 0; rb < 2; ++rb) wide = fmaxf(wide, of_row[rb] <= VS_NOTHING ? 0.0f : big[rb].largest());
            }
            rows.template add<true, false, true>(row0, s, unscaled);
            if (a.f.chunk_max) rows.template chunk<false>(a.f, tile, row0 / VS_BLOCK, (row0 >> 5) & 7, lane, true);
        }
        if ((c & 3) == 3) rows.flush();
    }
    rows.join_lanes();
    for (int o = 1; o < 64; o <<= 1) wide = fmaxf(wide, __shfl_xor(wide, o));
#pragma unroll
    for (int t = 0; t < TB; ++t)
        if (quad == 0) red[threadIdx.x >> 6][t * 16 + col] = make_float4(rows.st[t].ref, rows.st[t].S, rows.st[t].E, rows.st[t].R);
    if (lane == 0) widest[threadIdx.x >> 6] = wide;
    __syncthreads();
    if (threadIdx.x < TB * 16) {
        VsStat st;
        st.clear();
        for (int i = 0; i < 4; ++i) { const float4 q = red[i][threadIdx.x]; st.join(q.x, q.y, q.z, q.w); }
        a.f.part[(int64_t)blockIdx.x * a.f.n_pad + tile * TB * 16 + threadIdx.x] = make_float4(st.ref, st.S, st.E, st.R);
        if (tile == 0 && threadIdx.x == 0) a.f.wide[blockIdx.x] = fmaxf(fmaxf(widest[0], widest[1]), fmaxf(widest[2], widest[3]));
    }
}

// Joins the ranges of a row, by WAVES waves, and takes the given token's log probability: its logit, summed in float64, less
// lse; where the others' sum is less than half of all log(1 - that share), since lse has the rounding of the logits it is made of.  Bound by latency: 4 us for 87 rows of 64 ranges,
// 8 us for 8,192 rows of a few.
struct VsJoin {
    VsSrc x, w;
    const float* bias;         // as the caller gave it, or null
    const int64_t* targets;    // or null
    const float4* part;
    const float* wide;         // null where alternatives are not asked for
    int32_t n, splits;
    int64_t n_pad;
    float *logprob, *entropy, *lse;
};
template <int WAVES>
struct VsJoined {
    VsStat st;
    float wide;                // the largest size of a weight
    double lse;
    float rest;                // the share of the ids that are not the target
    bool empty;                // nothing but -inf
    // over `n` lanes (a power of two): the largest reference first, then sums relative to it
    __device__ __forceinline__ void over(int n) {
        VsStat q;
        q.clear();
        q.ref = st.ref;
        for (int o = 1; o < n; o <<= 1) q.ref = fmaxf(q.ref, __shfl_xor(q.ref, o));
        q.join(st.ref, st.S, st.E, st.R);
        for (int o = 1; o < n; o <<= 1) {
            q.S += __shfl_xor(q.S, o);
            q.E += __shfl_xor(q.E, o);
            q.R += __shfl_xor(q.R, o);
            wide = fmaxf(wide, __shfl_xor(wide, o));
        }
        st = q;
    }
    static __device__ __forceinline__ bool alone(const VsJoin& a) { return WAVES == 1 || a.splits <= 64; }   // few ranges: the first wave joins them
    __device__ __forceinline__ void gather(const VsJoin& a, int64_t row, int tid, float4* red) {
        st.clear();
        wide = 0.0f;
        if (alone(a) && tid >= 64) return;
#pragma unroll 4
        for (int i = tid; i < a.splits; i += alone(a) ? 64 : 64 * WAVES) {
            const float4 q = a.part[(int64_t)i * a.n_pad + row];
            if (a.wide) wide = fmaxf(wide, a.wide[i]);
            st.join(q.x, q.y, q.z, q.w);
        }
        over(a.splits > 32 ? 64 : a.splits > 16 ? 32 : a.splits > 8 ? 16 : 8);
        if (WAVES > 1 && (tid & 63) == 0) {
            red[tid >> 6 << 1] = make_float4(st.ref, st.S, st.E, st.R);
            red[(tid >> 6 << 1) + 1].x = wide;
        }
    }
    // (with more than one wave all have to have gathered)
    __device__ __forceinline__ void finish(const VsJoin& a, int64_t row, int tid, const float4* red) {
        if constexpr (WAVES > 1) {
            const int i = alone(a) ? 0 : tid % WAVES * 2;
            const float4 q = red[i];
            st.clear();
            st.ref = q.x; st.S = q.y; st.E = q.z; st.R = q.w; wide = red[i + 1].x;
            if (!alone(a)) over(WAVES);
        }
        empty = st.S == 0.0f;
        rest = st.R / st.S;
        const float l = log2f(st.S);
        lse = empty ? -INFINITY : ((double)st.ref + (double)l) * 0.6931471805599453;
        if (tid != 0) return;
        a.lse[row] = (float)lse;
        if (a.entropy) {
            const float h = VS_LN2 * (l - st.E / st.S);
            a.entropy[row] = empty || h < 0.0f ? 0.0f : h;
        }
    }
};
// the given token's logit, in every lane of the wave that asks, without its bias; and what is made of it
__device__ __forceinline__ double vs_target_logit(const VsJoin& a, int64_t row, int64_t t, int lane) {
    double dot = 0.0;
    if (t >= 0 && t < a.w.rows) {
        float x[8], w[8];                  // (512 elements at most, all loads under way together)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int d = min(lane + i * 64, a.w.dim - 1);
            x[i] = vs_load(a.x, row, d); w[i] = vs_load(a.w, t, d);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) dot += lane + i * 64 < a.w.dim ? (double)x[i] * (double)w[i] : 0.0;
        for (int o = 1; o < 64; o <<= 1) dot += __shfl_xor(dot, o);
    }
    return dot;
}
__device__ __forceinline__ void vs_put_logprob(const VsJoin& a, int64_t row, int64_t t, double dot, double lse, float rest, bool empty) {
    float lp = 0.0f;
    if (t >= a.w.rows) lp = NAN;
    else if (t >= 0) {
        const float b = vs_bias_of(a.bias, t);
        lp = empty || b == -INFINITY ? -INFINITY : rest < 0.5f ? log1pf(-rest) : (float)(dot + (double)b - lse);
        if (lp > 0.0f) lp = 0.0f;
    }
    a.logprob[row] = lp;
}
template <int WAVES>
__global__ __launch_bounds__(256) void k_vs_join(VsJoin a) {
    __shared__ float4 red[8];
    const int64_t row = WAVES == 1 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
    if (row >= a.n) return;
    const int tid = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x;
    const bool last = tid >> 6 == WAVES - 1 && a.logprob;      // its wave takes the given token
    VsJoined<WAVES> j;
    j.gather(a, row, tid, red);
    const int64_t t = last ? a.targets[row] : -1;
    const double dot = vs_target_logit(a, row, t, tid & 63);
    if (WAVES > 1) __syncthreads();
    j.finish(a, row, tid, red);
    if (last && (tid & 63) == 0) vs_put_logprob(a, row, t, dot, j.lse, j.rest, j.empty);
}

// ---- alternatives -------------------------------------------------------------------------------------------------
// The k largest logits of a row, ties to the lower id, in the order of the logits as float64 sums them.  The forward pass
// left each chunk's largest float32 logit m, rounded towards 0 to float16; a float32 sum is within d = 4 (D + 16) 2^-24 (|m| + 2 |x|_1
// max |w|) of the true one (elements as two float16 of their row's scale add 2^-22 + 2^-29 + 2^-36 D of |x|_1 max |w|, less than a 16th of that),
// the rounding adds 2^-10 |m|.  At least k logits are no less than the k-th largest m - d, so only
// chunks with m + d at or above that can hold one of the k: a few more than k, of 8 ids each.  Their logits are formed again in
// float32, those that reach the bound once more in float64, and the best k of these few are ranked by counting.  A workgroup
// per row.
//
// The bound is taken over 256 groups of chunks (the k-th largest of the groups' largest m - d is a bound too, and rarely a
// lower one): one pass over the maxima, after which all threads look through what the few threads have seen whose best may be
// one.  Where too many chunks reach it (many equal logits, a zero vector), they are visited in ascending order, and once k
// logits are known a later one that cannot beat the k-th is skipped even when it ties.
//
// Bound by latency for a few rows (12.5 us for one row of 262,144 ids, k = 10), by the reading of the maxima for many: 8,192 rows of
// 262,144 ids 144 us (537 MB of maxima and 0.15 GB of rows looked at again); by those rows where they are wide and k is large: 1,021
// rows, D = 511, k = 32, 60 us for 0.28 GB.  Chunks of 8 as float16 take the bytes of chunks of 16 as float32 (which that case
// paid 140 us for).
#define VS_MAX_K 32
#define VS_CAND 1024
#define VS_LIST 256
struct VsTop {
    VsJoin join;               // the row's ranges are joined first
    const _Float16* chunk_max; // [rows][chunks]
    int32_t chunks, k;
    int32_t* ids;              // [n][k]
    float* logprobs;           // [n][k]
};

__device__ __forceinline__ bool vs_before(double v, int i, double w, int j) { return v > w || (v == w && i < j); }

// 16 bytes of a row at whatever alignment its elements have, as floats
template <bool BF16>
struct VsVec {
    static constexpr int E = BF16 ? 8 : 4;
    struct __attribute__((packed, aligned(2))) Raw { uint32_t v[4]; };
    float f[E];
    __device__ __forceinline__ void load(const void* base, int64_t element) {
        if constexpr (BF16) {
            const Raw r = *(const Raw*)((const uint16_t*)base + element);
#pragma unroll
            for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(r.v[i] << 16); f[2 * i + 1] = __uint_as_float(r.v[i] & 0xFFFF0000u); }
        } else {
            const Raw r = *(const Raw*)((const float*)base + element);
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(r.v[i]);
        }
    }
};

// sum over the 16 lanes of a DPP row, in every lane of it
__device__ __forceinline__ float vs_row_sum(float v) {
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xF, 0xF, true));    // quad_perm [1,0,3,2]
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xF, 0xF, true));    // quad_perm [2,3,0,1]
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xF, 0xF, true));   // row_half_mirror
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x140, 0xF, 0xF, true));   // row_mirror
    return v;
}

__device__ __forceinline__ double vs_row_sum(double v) {
    auto from = [&](auto ctrl) {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, decltype(ctrl)::value, 0xF, 0xF, true),
                       hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), decltype(ctrl)::value, 0xF, 0xF, true);
        return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
    };
    v += from(std::integral_constant<int, 0xB1>{});
    v += from(std::integral_constant<int, 0x4E>{});
    v += from(std::integral_constant<int, 0x141>{});
    v += from(std::integral_constant<int, 0x140>{});
    return v;
}

// x . row for R rows over 16 lanes, each its part (xs: x in LDS, and behind it, from xs[dim up to a whole piece], the last piece again as
// it is multiplied: a row that is no whole number of pieces long has it taken back from the row's end, with the elements
// before it weighted 0 -- no read leaves the row).
template <bool BF16, int R, class T>
__device__ __forceinline__ void vs_dots(const VsSrc& w, const int (&row)[R], const float* xs, int lane, T (&s)[R]) {
    constexpr int E = VsVec<BF16>::E;
#pragma unroll
    for (int r = 0; r < R; ++r) s[r] = 0;
    if (w.dim < E) {
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (lane < w.dim) s[r] = (T)xs[lane] * (T)vs_load(w, row[r], lane);
    } else {
        const int whole = w.dim / E * E;
        for (int d = lane * E; d < w.dim; d += 16 * E) {
            VsVec<BF16> v[R];
#pragma unroll
            for (int r = 0; r < R; ++r) v[r].load(w.p, row[r] * w.ld + min(d, w.dim - E));
            const float* x = xs + (d < whole ? d : whole + E);
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int i = 0; i < E; ++i) s[r] = fma((T)x[i], (T)v[r].f[i], s[r]);
        }
    }
}
// x into LDS in that form, by all threads
template <bool BF16>
__device__ __forceinline__ float vs_put_x(const VsSrc& x, int64_t row, float* xs, int tid, int threads) {      // -> this thread's sum of sizes
    constexpr int E = VsVec<BF16>::E;
    const int whole = x.dim / E * E;
    float l1 = 0.0f;
    for (int d = tid; d < x.dim; d += threads) {
        const float v = vs_load(x, row, d);
        xs[d] = v;
        l1 += fabsf(v);
    }
    if (x.dim > E && tid < E) xs[whole + E + tid] = x.dim - E + tid >= whole ? vs_load(x, row, x.dim - E + tid) : 0.0f;
    return l1;
}

template <bool BF16, int THREADS>
__global__ __launch_bounds__(THREADS, THREADS == 256 ? BF16 ? 5 : 7 : 4) void k_vs_top(VsTop a) {
    const VsSrc &x = a.join.x, &w = a.join.w;
    __shared__ __align__(16) float xs[512 + 16], best[256];
    __shared__ __align__(16) double cv[VS_CAND], cw[VS_MAX_K];
    __shared__ int ci[VS_CAND], cj[VS_MAX_K];
    __shared__ float red[THREADS / 64];
    __shared__ uint32_t found[4];
    __shared__ uint32_t list[VS_LIST];
    __shared__ uint16_t rows[VS_CAND];
    __shared__ int n_cand, n_rows, n_list;
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = tid & 15, quarter = lane >> 4;
    const _Float16* cm = a.chunk_max + row * a.chunks;
    typedef _Float16 h8 __attribute__((ext_vector_type(8)));
    VsJoined<THREADS / 64> joined;
    joined.gather(a.join, row, tid, (float4*)cv);
    // (few ranges are the first wave's: the others have the row ready by then)
    float l1 = 0.0f;
    if (wave) {
        l1 = vs_put_x<BF16>(x, row, xs, tid - 64, THREADS - 64);
        for (int o = 1; o < 64; o <<= 1) l1 += __shfl_xor(l1, o);
    }
    if (lane == 0) red[wave] = l1;
    if (tid == 0) n_cand = n_rows = n_list = 0;
    const int64_t target = a.join.logprob ? a.join.targets[row] : -1;
    float mine = -INFINITY;                 // this thread's largest
    if (a.chunks <= 256) {
        if (tid < a.chunks) mine = (float)cm[tid];
    } else {
        h8 most = h8(-(_Float16)INFINITY);
#pragma unroll 4
        for (int c = tid * 8; c < a.chunks; c += THREADS * 8) most = __builtin_elementwise_max(most, *(const h8*)&cm[c]);
#pragma unroll
        for (int i = 0; i < 8; ++i) mine = fmaxf(mine, (float)most[i]);
    }
    __syncthreads();
    joined.finish(a.join, row, tid, (float4*)cv);
    const double lse = joined.lse;
    auto given = [&]() {                    // by one wave
        const double dot = vs_target_logit(a.join, row, target, lane);
        if (lane == 0) vs_put_logprob(a.join, row, target, dot, lse, joined.rest, joined.empty);
    };
    if (lse != lse) {                       // no order among the logits
        if (tid < a.k) { a.ids[row * a.k + tid] = -1; a.logprobs[row * a.k + tid] = NAN; }
        if (wave == 1 && a.join.logprob) given();
        return;
    }
    l1 = 0.0f;
    for (int i = 0; i < THREADS / 64; ++i) l1 += red[i];
    const float eps = 4.0f * (float)(x.dim + 16) * 5.9604645e-8f;
    const float slack = eps * 2.0f * l1 * joined.wide;
    // a chunk's largest logit lies between these (d, and a step of float16; past its range there is one bound only)
    auto off = [&](float m) { return fmaf(eps + 0.0009765625f, fabsf(m), slack + 5.9604645e-8f); };
    auto above = [&](float m) { return m >= 65504.0f ? INFINITY : m + off(m); };
    auto below = [&](float m) { return m <= -65504.0f ? -INFINITY : fminf(m, 65504.0f) - off(fminf(m, 65504.0f)); };
    float low = below(mine);
    if (a.chunks <= 256) {
        if (tid < 256) best[tid] = low;
    } else {
        for (int o = 1; o < THREADS / 256; o <<= 1) low = fmaxf(low, __shfl_xor(low, o));
        if (tid % (THREADS / 256) == 0) best[tid / (THREADS / 256)] = low;
    }
    __syncthreads();
    if (wave == 1 && a.join.logprob) given();
    if (wave == 0) {
        // the k-th largest of the 256, two bits at a time, over the upper 20 of a key in the floats' order (a lower bound will do)
        uint32_t key[4];
        const float4 q = *(const float4*)&best[lane * 4];
        const float v[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t u = __float_as_uint(v[i]);
            key[i] = (u & 0x80000000u) ? ~u : u | 0x80000000u;
        }
        uint32_t at = 0;
        for (int bit = 30; bit >= 12; bit -= 2) {
            uint32_t next = at;
#pragma unroll
            for (uint32_t two = 1; two < 4; ++two) {
                int n = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) n += __popcll(__ballot(key[i] >= (at | two << bit)));
                if (n >= a.k) next = at | two << bit;
            }
            at = next;
        }
        if (lane == 0) red[0] = at <= 0x007FFFFFu ? -INFINITY : __uint_as_float((at & 0x80000000u) ? at & 0x7FFFFFFFu : ~at);
    }
    __syncthreads();
    const float bound = red[0];
    double least = -INFINITY;               // the k-th best so far once k are known: what comes later must beat it
    bool full = false;
    auto compact = [&]() {                  // keeps the best k of the candidates, in order
        __syncthreads();
        const int n = n_cand;
        for (int i = tid; i < n; i += THREADS) {
            int rank = 0;
#pragma unroll 4
            for (int j = 0; j < n; ++j) rank += vs_before(cv[j], ci[j], cv[i], ci[i]);
            if (rank < a.k) { cw[rank] = cv[i]; cj[rank] = ci[i]; }
        }
        __syncthreads();
        const int m = min(n, a.k);
        if (tid < m) { cv[tid] = cw[tid]; ci[tid] = cj[tid]; }
        if (tid == 0) n_cand = m;
        __syncthreads();
        if (m == a.k) { full = true; least = cv[m - 1]; }
    };
    // the ids of two chunks of the list (or one) that reach the bound, by a wave
    auto look = [&](int i, bool first, bool second, int base) {
        int v[4], u[4];
        float s[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            v[r] = vs_chunk_row((int)list[r >= 2 && second ? i + 1 : i], (r & 1) * 4 + quarter);
            u[r] = min(v[r], w.rows - 1);
        }
        vs_dots<BF16, 4, float>(w, u, xs, l16, s);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            s[r] = vs_row_sum(s[r]) + vs_bias_of(a.join.bias, u[r]);
            if (l16 == 0 && (r < 2 ? first : second) && v[r] == u[r] && s[r] > -INFINITY && fmaf(eps, fabsf(s[r]), s[r] + slack) >= bound) {
                const int at = atomicAdd(&n_rows, 1);
                if (at < VS_CAND) rows[at] = (uint16_t)((i - base + r / 2) * VS_CHUNK + (r & 1) * 4 + quarter);
            }
        }
    };
    int least_end = 0;                      // ids from here on had no part in `least`: equal ones come after it
    auto beaten = [&](double s, int v) { return full && (s < least || (s == least && v >= least_end)); };
    // the float64 logits of those ids, four of a wave at a time
    auto exact = [&](int n, int base) {
        for (int i0 = wave * 4; i0 < n; i0 += THREADS / 16) {
            const int i = min(i0 + quarter, n - 1), v[1] = {vs_chunk_row((int)list[base + rows[i] / VS_CHUNK], rows[i] % VS_CHUNK)};
            double s[1];
            vs_dots<BF16, 1, double>(w, v, xs, l16, s);
            s[0] = vs_row_sum(s[0]) + (double)vs_bias_of(a.join.bias, v[0]);
            if (l16 == 0 && i0 + quarter < n && !beaten(s[0], v[0])) {
                const int at = atomicAdd(&n_cand, 1);
                cv[at] = s[0]; ci[at] = v[0];
            }
        }
    };
    auto may = [&](int c, float m) {
        const float up = above(m);
        return m > -INFINITY && up >= bound && !beaten((double)up, (c >> 5) * VS_BLOCK);
    };
    // every chunk that may hold one of the k, usually a few more than k: the threads whose best may say so, and all of them look
    // through what these few have seen
    const bool may_be = mine > -INFINITY && above(mine) >= bound;
    if (a.chunks <= 256) {
        if (may_be && tid < a.chunks) list[atomicAdd(&n_list, 1)] = tid;
    } else {
        if (may_be) rows[atomicAdd(&n_rows, 1)] = (uint16_t)tid;
        __syncthreads();
        const uint32_t pieces = (uint32_t)(a.chunks + THREADS * 8 - 1) / (THREADS * 8);        // of 8 chunks, of a thread
        const uint32_t all = n_rows * pieces;
#pragma unroll 2
        for (uint32_t i = tid; i < all; i += THREADS) {
            const int c = ((int)(i % pieces) * THREADS + rows[i / pieces]) * 8;
            if (c >= a.chunks) continue;
            const h8 m = *(const h8*)&cm[c];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (m[j] > -(_Float16)INFINITY && above((float)m[j]) >= bound) {
                    const int at = atomicAdd(&n_list, 1);
                    if (at < VS_LIST) list[at] = c + j;
                }
        }
        __syncthreads();
        if (tid == 0) n_rows = 0;
    }
    __syncthreads();
    bool done = n_list <= VS_LIST;
    if (done) {                             // all their ids at once
        const int n = n_list;
        for (int i = wave * 2; i < n; i += THREADS / 32) look(i, true, i + 1 < n, 0);
        __syncthreads();
        done = n_rows <= VS_CAND;
        if (done) exact(n_rows, 0);
    }
    if (!done) {                            // many equal logits: block after block
        __syncthreads();
        for (int c0 = 0; c0 < a.chunks; c0 += 256) {
            const int c = c0 + tid;
            const bool want = tid < 256 && c < a.chunks && may(c, (float)cm[c]);
            const unsigned long long bal = __ballot(want);
            if (lane == 0 && wave < 4) found[wave] = __popcll(bal);
            __syncthreads();
            int before = 0;
            for (int i = 0; i < min(wave, 4); ++i) before += found[i];
            const int nl = found[0] + found[1] + found[2] + found[3];
            if (want) list[before + __popcll(bal & ((1ull << lane) - 1ull))] = c;
            __syncthreads();
            for (int i0 = 0; i0 < nl; i0 += 32) {
                if (tid == 0) n_rows = 0;
                __syncthreads();
                for (int i = i0 + wave * 2; i < min(i0 + 32, nl); i += THREADS / 32) {
                    const bool one = may(list[i], (float)cm[list[i]]), two = i + 1 < nl && may(list[i + 1], (float)cm[list[i + 1]]);
                    if (one || two) look(i, one, two, i0);
                }
                __syncthreads();
                exact(n_rows, i0);
                __syncthreads();
                const bool crowded = n_cand > VS_CAND - 256;
                if (crowded) { compact(); least_end = ((int)(list[min(i0 + 31, nl - 1)] >> 5) + 1) * VS_BLOCK; }
                __syncthreads();
            }
        }
    }
    compact();
    __syncthreads();
    if (tid < a.k) {
        const bool have = tid < n_cand;
        a.ids[row * a.k + tid] = have ? ci[tid] : -1;
        a.logprobs[row * a.k + tid] = have ? fminf((float)(cv[tid] - lse), 0.0f) : -INFINITY;
    }
}

// ---- backward -----------------------------------------------------------------------------------------------------
__device__ __forceinline__ void vs_store(void* p, int64_t at, float v, int bf16) {
    if (bf16) ((__bf16*)p)[at] = (__bf16)v;
    else ((float*)p)[at] = v;
}

// Either gradient forms the logits again: n V D products beside the n V D of its own sums, and neither is stored.  Bound by the
// matrix units' power (float32, three products each: 8,192 tokens x 262,144 ids, D = 50, dx 1.45 ms and dw 1.50 ms, 1.65 * 10^12 operations
// of the MFMAs each, 1.1 * 10^15 a second).  Wide rows leave registers for 16 columns of a wave and two or three waves of a
// SIMD, which wait for one another twice in 32 streaming rows: bf16, D = 300, 4,096 x 65,536, entropy gradient too, dx 380 us
// (0.90 * 10^15; MFMAs busy 51 % of a 1.8 GHz clock), dw 499 us (two waves a SIMD: 37 % of 1.9 GHz).  The LDS reads are not what it waits for:
// with the weights of four waves shared, each reading a quarter of the transposed fragments (29 KB for 40), dx took as long and
// dw 3 % longer.  What spills, in registers of a lane: float32 of 257 to 320 elements 47 to 70 (dx 1.31 ms, dw 1.39 ms at 4,096 x 65,536),
// bf16 above 320 21 in dw; in forward passes bf16 of up to 64 4, float32 of 257 to 320 with alternatives 6, and of the kernels that read the
// weights as they lie bf16 of 257 to 320 with two blocks 11, float32 above 320 67.
struct VsBwd {
    const uint4 *stayS;        // stationary rows (columns of the product)
    const uint4 *flowS, *flowT;// streaming rows, and transposed
    const float* info;         // of ids: [ids / 32][VS_INFO]
    const float* tokens;       // of tokens: [tokens / 32][VS_TOKEN]
    int32_t has_bias, want_db;
    int32_t vocab;
    int32_t n_tiles, splits, groups;   // groups of 32 streaming rows
    int64_t stay_pad;          // rows of a partial
    float* part;               // [splits][stay_pad][32 KS]; of tokens null where dx is not asked for
    float* bias_part;          // [splits][stay_pad]
    // of tokens: the sum of p over all ids but the target, [splits][stay_pad], and log2 p of the target, [stay_pad]
    float *rest, *target_e;
    // of ids, one range: the result itself
    void* out;                 // null: partials
    int64_t ldo;
    int32_t rows, dim;
    float* db;
};

// A wave: a tile of TB M stationary rows against one range of the streaming ones.  OF_IDS = false: the stationary rows
// are tokens, the result sum_v p' w_v with p' = p (A + B e), or p alone when there is no entropy gradient (A is then a
// factor of the whole row, applied at the end).  OF_IDS = true: the stationary rows are ids, the result sum_n G_nv x_n.
//
// The target's coefficient is g (1 - p_t): small where a token is predicted well, and nothing but rounding errors if it were left to
// g and g p_t, each rounded, to cancel.  So the sums over tokens leave the target out and find 1 - p_t as what the others
// add up to (k_vs_target, between the two gradients); dx gets the whole coefficient times w_t at the end, in float32, and dw takes it as
// the weight of that token and id.  In bf16 it is by far the largest of most tokens: dw adds what its rounding left over in the few
// steps in which one lies in the tile.
//
// bf16 inputs: the other weights are one bf16 each, as far off (2^-8) as an element of the result is when it is rounded to its own type;
// a result's error against 64 bits is that of its rounding alone where unlikely targets weigh most (0.0017 of its norm), up to 0.0021
// where well-predicted ones do.  Two parts for all of them would cost half as many products again: a step of 4,096 x 65,536, D = 300,
// 1,194 us in place of 1,006.
//
// Two float16 parts (PL = 2) of a weight: column t is kept multiplied by 2^sg[t], sg as large as the largest weight of the column
// so far allows (2^15 after the streaming rows' scale), and the sums with it.  It starts high and falls a few times.
template <int KS, int PL, int M, int TB, bool OF_IDS, bool ENTROPY, bool SUMS>
struct VsGrad {
    static constexpr float MOST = 15.0f, AIM = 13.0f;
    // Where a step's weights are formed again if a target is among them, and where its logits are changed before (4,096 x 65,536, both
    // gradients: D = 100 bf16 with entropy 350 us, 383 the other way; D = 100 float32 696, 753; D = 300 bf16 813, 824)
    static constexpr bool AGAIN = PL == 1 && KS <= 4;
    static constexpr int NJ = VS_NJ<M>, HALVES = VS_HALVES<M>, BLOCKS = SUMS ? KS * 32 / M : 0;     // SUMS = false: of tokens, without dx
    using Acc = typename VsTile<M>::Acc;
    using Weights = vs_bits[HALVES][PL];       // of one column, by streaming row
    VsOperand<KS, PL, M> y[TB];
    Acc acc[SUMS ? BLOCKS : 1][TB];
    float L[TB], A[TB], B[TB], db[TB], y_exp[TB], sg[TB], norm[TB], rest[TB];   // (of ids, L is the bias)
    int target[TB];
    int64_t stay0;

    __device__ __forceinline__ void start(const VsBwd& a, int64_t tile, int lane, bool live) {
        vs_stationary<KS, PL, M, TB>(a.stayS, tile, lane, y);
        stay0 = tile * TB * M;
#pragma unroll
        for (int t = 0; t < TB; ++t) {
            const int64_t r = stay0 + t * M + lane % M;
            db[t] = 0.0f; sg[t] = 300.0f; norm[t] = 0.0f; rest[t] = 0.0f;
            if constexpr (OF_IDS) {
                const float* of = a.info + (r >> 5) * VS_INFO;
                L[t] = of[r & 31];
                y_exp[t] = PL == 2 ? of[VS_INFO_EXP] + vs_more(of + VS_INFO_MORE, r & 31) : 0.0f;
            } else {
                const float* of = a.tokens + (r >> 5) * VS_TOKEN;
                L[t] = of[r & 31]; A[t] = of[VS_TOKEN_A + (r & 31)]; B[t] = of[VS_TOKEN_B + (r & 31)];
                y_exp[t] = PL == 2 ? of[VS_TOKEN_EXP] + vs_more(of + VS_TOKEN_MORE, r & 31) : 0.0f;
                target[t] = live ? __float_as_int(of[VS_TOKEN_TARGET + (r & 31)]) : -1;
                if (PL == 2 && ENTROPY) {      // |A + B e| brought below 1
                    const float size = fabsf(A[t]) + fabsf(B[t]) * 256.0f;
                    norm[t] = size > 0.0f && size < INFINITY ? (float)__builtin_amdgcn_frexp_expf(size) : 0.0f;
                    A[t] = ldexpf(A[t], -(int)norm[t]);
                    B[t] = ldexpf(B[t], -(int)norm[t]);
                }
            }
        }
#pragma unroll
        for (int d = 0; d < BLOCKS; ++d)
#pragma unroll
            for (int t = 0; t < TB; ++t) acc[d][t] = Acc(0.0f);
    }

    // column t gives up the powers of two that its lanes ask for (`ask` <= 0: none)
    __device__ __forceinline__ void lower(int t, float ask) {
        if (M == 16) ask = fmaxf(ask, __shfl_xor(ask, 16));
        ask = fmaxf(ask, __shfl_xor(ask, 32));
        if (!(ask > 0.0f)) ask = 0.0f;
        sg[t] -= ask;
#pragma unroll
        for (int d = 0; d < BLOCKS; ++d) {
            Acc v;
#pragma unroll
            for (int i = 0; i < M * M / 64; ++i) v[i] = ldexpf(acc[d][t][i], -(int)ask);
            vs_in_place(v);
            acc[d][t] = v;
        }
    }

    // Of tokens: targets among the 32 ids from row0 on are taken out of the sums.  Rare: a token has one.
    __device__ __forceinline__ bool any_target(int row0) const {
        bool here = false;
#pragma unroll
        for (int t = 0; t < TB; ++t) here |= (uint32_t)(target[t] - row0) < 32;
        return __any(here);
    }
    __device__ __forceinline__ void leave_targets(const VsBwd& a, int row0, const float (&unit)[TB], VsLogits<M, TB>& s) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int t = 0; t < TB; ++t) {
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const float v = vs_value<M, TB>(s, t, j);
                const bool it = target[t] == row0 + vs_row<M>(j, lane);
                if (it) a.target_e[stay0 + t * M + lane % M] = fmaf(v, unit[t], -L[t]);
                vs_set<M, TB>(s, t, j, it ? -INFINITY : v);
            }
            if (!AGAIN)
#pragma unroll
                for (int b = 0; b < VsTile<M>::NB; ++b) vs_in_place(s[b][t]);
        }
    }
    // Of ids: whether a target lies in the tile, of 32 tokens, and the weights of those tokens
    __device__ __forceinline__ bool targets_here(const float* of) const {
        return __any((uint32_t)(__float_as_int(of[VS_TOKEN_TARGET + (threadIdx.x & 31)]) - (int)stay0) < TB * M);
    }
    __device__ __forceinline__ void put_targets(const float* of, float (&G)[TB][NJ]) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int t = 0; t < TB; ++t)
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int at = vs_row<M>(j, lane);
                if (__float_as_int(of[VS_TOKEN_TARGET + at]) == (int)stay0 + t * M + lane % M) G[t][j] = of[VS_TOKEN_GT + at];
            }
    }

    // P: the weights of the 32 streaming rows from row0 on, in parts.  -> of ids: is a target among them?
    __device__ __forceinline__ bool weights(const VsBwd& a, int row0, const uint4* S, const float* of, Weights (&P)[TB]) {
        const int lane = threadIdx.x & 63;
        VsLogits<M, TB> s;
        vs_f4 b[NJ / 4];
        float unit[TB];
        const float f_exp = PL == 2 ? of[OF_IDS ? VS_TOKEN_EXP : VS_INFO_EXP] : 0.0f;
        if constexpr (OF_IDS) {
#pragma unroll
            for (int t = 0; t < TB; ++t)
#pragma unroll
                for (int j = 0; j < NJ; ++j) vs_set<M, TB>(s, t, j, PL == 1 ? L[t] : 0.0f);
        } else vs_begin<PL, M, TB>(of, lane, s, b);
#pragma unroll
        for (int t = 0; t < TB; ++t) unit[t] = PL == 2 ? vs_unit(-(f_exp + y_exp[t])) : VS_LOG2E;
        vs_product<KS, PL, M, TB>(S, y, s);
        uint32_t more[NJ / 4];
        const bool differ = PL == 2 && vs_differ(of[OF_IDS ? VS_TOKEN_DIFFER : VS_INFO_DIFFER]);
        if (differ) {
            vs_mores<M>(of + (OF_IDS ? VS_TOKEN_MORE : VS_INFO_MORE), lane, more);
            vs_common<M, TB>(more, s);
        }
        if (a.has_bias || (OF_IDS ? stay0 + TB * M > a.vocab : row0 + 32 > a.vocab)) {
            if constexpr (OF_IDS) {
#pragma unroll
                for (int t = 0; t < TB; ++t) {
#pragma unroll
                    for (int j = 0; j < NJ; ++j) {
                        float v = vs_value<M, TB>(s, t, j);
                        if (PL == 2) v = fmaf(v, unit[t], L[t]);
                        vs_set<M, TB>(s, t, j, vs_max(v, VS_MASKED));
                    }
                    if (PL == 2) unit[t] = 1.0f;
                }
            } else vs_mask<M, TB, PL == 2>(s, unit, b);
        }
        if constexpr (!OF_IDS && !AGAIN)
            if (any_target(row0)) leave_targets(a, row0, unit, s);
        if (PL == 2 && !OF_IDS && differ) {    // (as for ids, in the exponent)
#pragma unroll
            for (int t = 0; t < TB; ++t) {
#pragma unroll
                for (int j = 0; j < NJ; ++j) vs_set<M, TB>(s, t, j, fmaf(vs_value<M, TB>(s, t, j), unit[t], -(float)vs_more_of(more, j)));
                unit[t] = 1.0f;
#pragma unroll
                for (int b = 0; b < VsTile<M>::NB; ++b) vs_in_place(s[b][t]);
            }
        }
        float G[TB][NJ];
        float big[TB], ps[TB];                 // PL = 2: the power of two that a column's largest scaled weight is below; of tokens: the sum of p
        auto form = [&]() {
            vs_f4 rl[NJ / 4], ra[NJ / 4], rb[NJ / 4];
            if constexpr (OF_IDS) {
#pragma unroll
                for (int q = 0; q < NJ / 4; ++q) {
                    const float* at = of + vs_row<M>(q * 4, lane);
                    rl[q] = *(const vs_f4*)at;
                    ra[q] = *(const vs_f4*)(at + VS_TOKEN_A);
                    if (ENTROPY) rb[q] = *(const vs_f4*)(at + VS_TOKEN_B);
                }
            }
            float most = 0.0f;
#pragma unroll
            for (int t = 0; t < TB; ++t) {
                const float shift = PL == 2 ? sg[t] - f_exp : 0.0f;
                float m = 0.0f;
                ps[t] = 0.0f;
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    const float v = vs_value<M, TB>(s, t, j);
                    if constexpr (OF_IDS) {
                        float e = fmaf(v, PL == 2 ? unit[t] : VS_LOG2E, -rl[j >> 2][j & 3]);
                        const float p = __builtin_amdgcn_exp2f(e);
                        if (ENTROPY) e = vs_max(e, VS_TMIN);
                        G[t][j] = p * (ENTROPY ? fmaf(rb[j >> 2][j & 3], e, ra[j >> 2][j & 3]) : ra[j >> 2][j & 3]);
                    } else {
                        float e = fmaf(v, PL == 2 ? unit[t] : VS_LOG2E, shift - L[t]);
                        if (PL == 2) m = j ? fmaxf(m, e) : e;
                        G[t][j] = __builtin_amdgcn_exp2f(e);
                        ps[t] = j ? ps[t] + G[t][j] : G[t][j];
                        if (ENTROPY) {
                            e = vs_max(e, VS_TMIN);
                            G[t][j] *= fmaf(B[t], e, PL == 2 ? fmaf(-B[t], shift, A[t]) : A[t]);
                        }
                    }
                }
                if (!OF_IDS) { big[t] = m; most = fmaxf(most, m); }
            }
            return most;
        };
        float most = form();
        if constexpr (!OF_IDS && AGAIN)
            if (any_target(row0)) {
                leave_targets(a, row0, unit, s);
                form();
            }
        const bool of_target = OF_IDS && targets_here(of);
        if constexpr (OF_IDS) {
            if (of_target) put_targets(of, G);
            if (a.want_db)
#pragma unroll
                for (int t = 0; t < TB; ++t) {
                    float v = 0.0f;
#pragma unroll
                    for (int j = 0; j < NJ; j += 4) v += (G[t][j] + G[t][j + 1]) + (G[t][j + 2] + G[t][j + 3]);
                    db[t] += v;
                }
            if (PL == 2) {
#pragma unroll
                for (int t = 0; t < TB; ++t) {
                    float m = 0.0f;
#pragma unroll
                    for (int j = 0; j < NJ; ++j) m = fmaxf(m, fabsf(G[t][j]));
                    big[t] = m > 0.0f ? (float)__builtin_amdgcn_frexp_expf(m) + (sg[t] - f_exp) : 0.0f;
                }
                if (differ)                    // weights of rows with a smaller scale of their own are as much larger, for their products
#pragma unroll
                    for (int t = 0; t < TB; ++t) {
                        float m = -1000.0f;
#pragma unroll
                        for (int j = 0; j < NJ; ++j) m = fmaxf(m, G[t][j] != 0.0f ? (float)(__builtin_amdgcn_frexp_expf(G[t][j]) - vs_more_of(more, j)) : m);
                        big[t] = m + (sg[t] - f_exp);
                    }
#pragma unroll
                for (int t = 0; t < TB; ++t) most = fmaxf(most, big[t]);
            }
        }
        if (PL == 2)
            if (__any(most > MOST)) {
#pragma unroll
                for (int t = 0; t < TB; ++t) lower(t, ceilf(big[t] - AIM));
                if (!OF_IDS) form();           // (there the scale is in the exponent already)
            }
        int by[TB];
#pragma unroll
        for (int t = 0; t < TB; ++t) {
            by[t] = PL == 2 ? (int)(sg[t] - f_exp) : 0;
            if (!OF_IDS) ps[t] = PL == 2 ? ldexpf(ps[t], -by[t]) : ps[t];
        }
        if (differ)
#pragma unroll
            for (int t = 0; t < TB; ++t) {
                if (OF_IDS) {
#pragma unroll
                    for (int j = 0; j < NJ; ++j) G[t][j] = ldexpf(G[t][j], by[t] - vs_more_of(more, j));
                    by[t] = 0;
                } else {                       // p is 2^(e + more - by) there, with the e that G was formed of
                    ps[t] = 0.0f;
#pragma unroll
                    for (int j = 0; j < NJ; ++j) {
                        const float e = fmaf(vs_value<M, TB>(s, t, j), unit[t], (float)by[t] - L[t]), q = __builtin_amdgcn_exp2f(e);
                        ps[t] += ldexpf(q, vs_more_of(more, j) - by[t]);
                        if (ENTROPY) G[t][j] = q * fmaf(B[t], vs_max(e + (float)vs_more_of(more, j), VS_TMIN), fmaf(-B[t], (float)by[t], A[t]));
                    }
                }
            }
#pragma unroll
        for (int t = 0; t < TB; ++t) {
            if (!OF_IDS) rest[t] += ps[t];
#pragma unroll
            for (int u = 0; u < HALVES; ++u) {
                vs_f8 v;
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = PL == 2 && OF_IDS ? ldexpf(G[t][u * 8 + j], by[t]) : G[t][u * 8 + j];
                vs_split<PL>(v, P[t][u]);
            }
        }
        return of_target;
    }

    __device__ __forceinline__ void products(const uint4* T, const Weights (&P)[TB]) {
        constexpr int R = BLOCKS % 2 ? 1 : 2;      // blocks at once: their accumulators are independent
#pragma unroll
        for (int d = 0; d < BLOCKS; d += R)
#pragma unroll
            for (int u = 0; u < HALVES; ++u) {
                vs_bits f[R][PL];
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int p = 0; p < PL; ++p) f[r][p] = *(const vs_bits*)&T[(((d + r) * HALVES + u) * PL + p) * 64];
                vs_mfma_parts<PL, M, R, TB>(f, [&](int t, int p) { return P[t][u][p]; }, *(Acc(*)[R][TB]) & acc[d]);
            }
    }

    // Of ids, bf16: what the rounding of the targets' weights left over.  Rare: a token has one target.
    __device__ __forceinline__ void left_over(const uint4* T, const float* of) {
        const int lane = threadIdx.x & 63;
#pragma unroll 1
        for (int q = 0; q < TB * HALVES; ++q) {
            const int t = q / HALVES, u = q % HALVES;
            vs_f8 G;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int at = vs_row<M>(u * 8 + j, lane);
                G[j] = __float_as_int(of[VS_TOKEN_TARGET + at]) == (int)stay0 + t * M + lane % M ? of[VS_TOKEN_GT + at] : 0.0f;
            }
            vs_bits part[2];
            vs_split<1>(G, &part[0]);
            vs_split<1>(G - __builtin_convertvector(__builtin_bit_cast(vs_bf8, part[0]), vs_f8), &part[1]);
#pragma unroll
            for (int v = 0; v < TB; ++v)       // (registers have no index)
                if (v == t)
#pragma unroll
                    for (int d = 0; d < BLOCKS; ++d) {
                        Acc c = vs_mfma<PL, M>(*(const vs_bits*)&T[(d * HALVES + u) * 64], part[1], acc[d][v]);
#pragma unroll
                        for (int i = 0; i < M * M / 64; ++i) c[i] += 0.0f;     // (a vector instruction between, for its waits)
                        vs_in_place(c);
                        acc[d][v] = c;
                    }
        }
    }

    __device__ __forceinline__ void store(const VsBwd& a, int split, int lane) {
#pragma unroll
        for (int t = 0; t < TB; ++t) {
            const int64_t r = stay0 + t * M + lane % M;
            const bool final = OF_IDS && a.out;
            if (final && r >= a.rows) continue;
            if constexpr (!OF_IDS) {
                float v = rest[t];
                if (M == 16) v += __shfl_xor(v, 16);
                v += __shfl_xor(v, 32);
                if (lane < M) a.rest[(int64_t)split * a.stay_pad + r] = v;
                if (!a.part) continue;
            }
            float* out = a.part + ((int64_t)split * a.stay_pad + r) * (KS * 32);
#pragma unroll
            for (int d = 0; d < BLOCKS; ++d)
#pragma unroll
                for (int q = 0; q < M * M / 256; ++q) {
                    vs_f4 v;
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = PL == 2 ? ldexpf(acc[d][t][q * 4 + i], (int)(norm[t] - sg[t])) : acc[d][t][q * 4 + i];
                    const int e = d * M + q * 8 + lane / M * 4;
                    if (!final) *(vs_f4*)&out[e] = v;
                    else
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (e + i < a.dim) vs_store(a.out, r * a.ldo + e + i, v[i], PL == 1);
                }
            if (OF_IDS && a.want_db) {
                float v = db[t];
                if (M == 16) v += __shfl_xor(v, 16);
                v += __shfl_xor(v, 32);
                if (lane < M) *(final ? &a.db[r] : &a.bias_part[(int64_t)split * a.stay_pad + r]) = v;
            }
        }
    }
};

// Without dx the sums over tokens are not formed: by a branch, or, where their registers leave the compiler no room to
// keep them in place across one, by a kernel of its own.
constexpr bool vs_bwd_wide(int ks, int tb) { return ks * tb > 10; }

// The stages in LDS.  TURNS = false: SR rows with both their fragments at a time, two stages (one worked on, one under way).
// TURNS = true (wide rows): 32 rows, their S and their T fragments by turns, each under way while the other is worked on.
template <int KS, int PL, int M, int TB, int SR, bool OF_IDS, bool ENTROPY, bool SUMS>
struct VsGradStage {
    using Grad = VsGrad<KS, PL, M, TB, OF_IDS, ENTROPY, SUMS>;
    static __device__ __forceinline__ bool sums(const VsBwd& a) { return SUMS && (OF_IDS || vs_bwd_wide(KS, TB) || a.part); }
    static constexpr int HALF = SR * KS * PL * 4, INFO = (OF_IDS ? VS_TOKEN : VS_INFO), INFOS = SR / 32 * INFO;
    static constexpr int SIZE = 2 * HALF + (INFOS + 3) / 4;
    static __device__ __forceinline__ void fetch(const uint4* S, const uint4* T, const float* info, uint4* to) {
        vs_stage<HALF>(S, to);
        vs_stage<HALF>(T, to + HALF);
#pragma unroll
        for (int i = 0; i < SR / 32; ++i) vs_stage_floats<INFO>(info + i * INFO, (float*)(to + 2 * HALF) + i * INFO);
    }
    static __device__ __forceinline__ void step(const VsBwd& a, int base, bool more, const uint4* __restrict__ S, const uint4* __restrict__ T,
                                                const float* __restrict__ info, uint4* __restrict__ to, const uint4* __restrict__ from,
                                                Grad& g) {
        const int lane = threadIdx.x & 63;
        vs_copies_done();
        __syncthreads();
        if (more) fetch(S, T, info, to);
#pragma unroll 1
        for (int r = 0; r < SR; r += 32) {
            typename Grad::Weights P[TB];
            const float* of = (const float*)(from + 2 * HALF) + r / 32 * INFO;
            const bool of_target = g.weights(a, base + r, from + r * KS * PL * 4 + lane, of, P);
            if (sums(a)) g.products(from + HALF + r * KS * PL * 4 + lane, P);
            if (PL == 1 && of_target) g.left_over(from + HALF + r * KS * PL * 4 + lane, of);
        }
    }
    // by turns: each half with its own copy of what goes with it
    static constexpr int TURN = HALF + (INFO + 3) / 4;
    static __device__ __forceinline__ void fetch_half(const uint4* half, const float* info, uint4* to) {
        vs_stage<HALF>(half, to);
        vs_stage_floats<INFO>(info, (float*)(to + HALF));
    }
    static __device__ __forceinline__ bool turn_s(const VsBwd& a, int base, const uint4* __restrict__ T, const float* __restrict__ info, uint4* __restrict__ to,
                                                  const uint4* __restrict__ from, Grad& g, typename Grad::Weights (&P)[TB]) {
        vs_copies_done();
        __syncthreads();
        fetch_half(T, info, to);
        return g.weights(a, base, from + (threadIdx.x & 63), (const float*)(from + HALF), P);
    }
    static __device__ __forceinline__ void turn_t(const VsBwd& a, bool more, const uint4* __restrict__ S, const float* __restrict__ info, uint4* __restrict__ to,
                                                  const uint4* __restrict__ from, Grad& g, const typename Grad::Weights (&P)[TB], bool of_target) {
        vs_copies_done();
        __syncthreads();
        if (more) fetch_half(S, info, to);
        if (sums(a)) g.products(from + (threadIdx.x & 63), P);
        if (PL == 1 && of_target) g.left_over(from + (threadIdx.x & 63), (const float*)(from + HALF));
    }
};

// Waves of a SIMD that the registers are shared out for: as many as need no scratch, and one more where the compiler finds room.
constexpr int vs_bwd_waves(int KS, int PL, int M, int TB, bool OF_IDS) {
    return PL == 1 && !OF_IDS && KS >= 10 ? (KS == 10 ? 3 : 2) : TB * M * KS * (4 * PL + 8) > 170 * 16 ? 1 : 2;
}

template <int KS, int PL, int M, int TB, int SR, bool TURNS, bool OF_IDS, bool ENTROPY, bool SUMS>
__global__ __launch_bounds__(256, vs_bwd_waves(KS, PL, M, TB, OF_IDS)) void k_vs_backward(VsBwd a) {
    using Stage = VsGradStage<KS, PL, M, TB, SR, OF_IDS, ENTROPY, SUMS>;
    constexpr int SIZE = TURNS ? Stage::TURN : Stage::SIZE;
    __shared__ uint4 buf0[SIZE], buf1[SIZE];
    constexpr int PIECE = KS * PL * 4;         // 16-byte pieces of a row's fragments
    const int lane = threadIdx.x & 63;
    const int split = blockIdx.x % a.splits;
    const int tile = (blockIdx.x / a.splits) * 4 + (threadIdx.x >> 6);
    const bool live = tile < a.n_tiles;
    typename Stage::Grad g;
    g.start(a, live ? tile : 0, lane, live);
    const float* info = OF_IDS ? a.tokens : a.info;
    if constexpr (TURNS) {
        const int row_begin = (int)((int64_t)a.groups * split / a.splits) * 32, row_end = (int)((int64_t)a.groups * (split + 1) / a.splits) * 32;
        const uint4 *S = a.flowS + (int64_t)row_begin * PIECE, *T = a.flowT + (int64_t)row_begin * PIECE;
        info += (int64_t)row_begin / 32 * Stage::INFO;
        Stage::fetch_half(S, info, buf0);
        for (int base = row_begin; base < row_end; base += 32) {
            typename Stage::Grad::Weights P[TB];
            const bool of_target = Stage::turn_s(a, base, T, info, buf1, buf0, g, P);
            S += 32 * PIECE; T += 32 * PIECE; info += Stage::INFO;
            Stage::turn_t(a, base + 32 < row_end, S, info, buf0, buf1, g, P, of_target);
        }
    } else {
        const int units = a.groups / (SR / 32);
        const int row_begin = (int)((int64_t)units * split / a.splits) * SR, row_end = (int)((int64_t)units * (split + 1) / a.splits) * SR;
        const uint4 *S = a.flowS + (int64_t)row_begin * PIECE, *T = a.flowT + (int64_t)row_begin * PIECE;
        info += (int64_t)row_begin / 32 * Stage::INFO;
        Stage::fetch(S, T, info, buf0);
        for (int base = row_begin; base < row_end; base += 2 * SR) {
            S += SR * PIECE; T += SR * PIECE; info += Stage::INFOS;
            Stage::step(a, base, base + SR < row_end, S, T, info, buf1, buf0, g);
            if (base + SR >= row_end) break;
            S += SR * PIECE; T += SR * PIECE; info += Stage::INFOS;
            Stage::step(a, base + SR, base + 2 * SR < row_end, S, T, info, buf0, buf1, g);
        }
    }
    if (live) g.store(a, split, lane);
}

// A token's coefficient of its target, G_t = g (1 - p_t) - h p_t (log p_t + H), from what the sums over tokens left (5 us for
// 4,096 tokens): where p_t is above a half, 1 - p_t is what the other ids add up to, else it is formed from p_t, which is smaller.
__global__ __launch_bounds__(256) void k_vs_target(VsPack a, const float* __restrict__ rest, const float* __restrict__ target_e, int32_t splits, int64_t pad) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= a.src.rows) return;
    float* of = a.tokens + (i >> 5) * VS_TOKEN + (i & 31);
    if (__float_as_int(of[VS_TOKEN_TARGET]) < 0) return;       // (gl stays: 0, or NaN for a target past the vocabulary)
    float r = 0.0f, fix = 1.0f;
#pragma unroll 8
    for (int s = 0; s < splits; ++s) r += rest[(int64_t)s * pad + i];
    const float l = a.lse[i], e = target_e[i];
    const bool empty = l == -INFINITY;
    if (!empty) vs_lse2(l, fix);
    r *= fix;
    float p = exp2f(e) * fix;
    const bool near = p > 0.5f;
    if (near) p = 1.0f - r;
    float G = of[VS_TOKEN_GT] * (near ? r : 1.0f - p);
    if (a.h && a.h[i] != 0.0f && !empty && p > 0.0f) G -= a.h[i] * p * ((near ? log1pf(-r) : e * VS_LN2) + a.entropy[i]);
    of[VS_TOKEN_GT] = G;
}

// Sums the partials of a row in a fixed order (eight loads under way: 17 us for 4,096 x 320 of 8 ranges; 4 us for 129 x 64) and writes it: dx = A sum p w + G_t w_t (without an entropy gradient; with
// one the partials hold p (A + B e) already), dw as it is, db beside it.
struct VsSum {
    const float* part;
    const float* bias_part;
    int32_t rows, dim, dp, splits;
    int64_t pad;
    const float* tokens;       // of tokens; null for dw
    int32_t has_entropy;
    VsSrc w;
    void* out;
    int64_t ldo;
    int32_t out_bf16;
    float* db;
};
// Two results in one launch: the first `first` workgroups sum pa, the others pb.
__global__ __launch_bounds__(256) void k_vs_sum(VsSum pa, VsSum pb, uint32_t first) {
    const VsSum& a = blockIdx.x < first ? pa : pb;
    const int64_t i = (int64_t)(blockIdx.x < first ? blockIdx.x : blockIdx.x - first) * 256 + threadIdx.x;
    if (a.db && i < a.rows) {
        float v = 0.0f;
#pragma unroll 8
        for (int s = 0; s < a.splits; ++s) v += a.bias_part[(int64_t)s * a.pad + i];
        a.db[i] = v;
    }
    if (i >= (int64_t)a.rows * a.dim) return;
    const int64_t r = i / a.dim;
    const int d = (int)(i % a.dim);
    float v = 0.0f;
#pragma unroll 8
    for (int s = 0; s < a.splits; ++s) v += a.part[((int64_t)s * a.pad + r) * a.dp + d];
    if (a.tokens) {
        const float* of = a.tokens + (r >> 5) * VS_TOKEN + (r & 31);
        if (!a.has_entropy) v *= of[VS_TOKEN_A];
        const int32_t t = __float_as_int(of[VS_TOKEN_TARGET]);
        const float G = of[VS_TOKEN_GT];
        if (t >= 0) v = fmaf(G, vs_load(a.w, t, d), v);
        else if (G != G) v = G;
    }
    vs_store(a.out, r * a.ldo + d, v, a.out_bf16);
}

// no tokens: dw = 0, db = 0
__global__ __launch_bounds__(256) void k_vs_zero(void* out, int64_t ldo, int32_t rows, int32_t dim, int32_t out_bf16, float* db) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (db && i < rows) db[i] = 0.0f;
    if (i < (int64_t)rows * dim) vs_store(out, i / dim * ldo + i % dim, 0.0f, out_bf16);
}
