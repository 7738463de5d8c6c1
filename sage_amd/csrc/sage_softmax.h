// Softmax over a whole vocabulary: log probabilities of given tokens with entropy and the most likely alternatives, and
// the gradient of both, without ever storing the [tokens][vocabulary] matrix of logits.
//
//   s_nv = x_n . w_v + b_v                 lse_n = log sum_v exp s_nv          p_nv = exp(s_nv - lse_n)
//   logprob_n = s_n,t(n) - lse_n           H_n = lse_n - sum_v p_nv s_nv
//   G_nv = g_n (1[v = t(n)] - p_nv) - h_n p_nv (log p_nv + H_n)     (g, h: the gradients of logprob and H)
//   dx = G w      dw = G^T x      db_v = sum_n G_nv
//
// Matrix layout.  Every product runs on v_mfma_f32_16x16x32_bf16.  A "stationary" operand (tokens in the forward pass and
// for dx, ids for dw) stays in a wave's registers, the other one "streams" past it 32 rows at a time.  The product is taken
// with the streaming rows as matrix rows and the stationary ones as columns: lane l then holds, of column l % 16, the
// rows 4 (l / 16) .. + 3, so maxima and sums over the streaming axis need no lane to talk to another one until the end,
// and the eight weights of two 16-row tiles are, as they lie in the registers, the second operand of the next product
// (its 32 summation slots are the 32 streaming rows in the order 16 (j / 4) + 4 (l / 16) + j % 4; the transposed
// fragments are laid out in that order).
//
// bf16 inputs are multiplied as they are (products of two bf16 are exact in float32).  float32 inputs are taken as the sum
// of three bf16 (8 + 8 + 8 bits: exact), and six of the nine products are formed -- the other three are below 2^-24 of
// |x||w| --, which costs 6 bf16 MFMAs where the float32 MFMA costs 16 (256 against 4,096 operations per clock and CU).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

typedef __bf16 vs_bf8 __attribute__((ext_vector_type(8)));
typedef float vs_f4 __attribute__((ext_vector_type(4)));
typedef float vs_f8 __attribute__((ext_vector_type(8)));

#define VS_LOG2E 1.4426950408889634f
#define VS_LN2 0.6931471805599453f
#define VS_CHUNK 16            // ids per stored maximum (the unit in which alternatives are looked for)
#define VS_BLOCK 256           // ids are dealt out in blocks of this many
// A chunk is what one lane of a fragment sees of 64 ids: 4 (of each of four 16-row tiles), so its maximum needs no other
// lane.  Chunk c: of block c / 16 the lane quarter c / 4 % 4 of the 64 ids c % 4; a lane stores its four of a block at once.
__device__ __forceinline__ int vs_chunk_row(int c, int i) {      // the i-th of the 16 ids of a chunk
    return (c >> 4) * VS_BLOCK + (c & 3) * 64 + (i >> 2) * 16 + ((c >> 2) & 3) * 4 + (i & 3);
}
#define VS_NOTHING (-1.0e30f)  // reference of a row that has seen no finite logit yet; a bias this low masks its id
#define VS_SLACK 20.0f         // the running reference lags the maximum by at most this (in powers of two)
#define VS_TMIN (-200.0f)      // 2^-200 is 0 in float32: what a logit of -inf is raised to, so that 0 * log p is 0

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

__device__ __forceinline__ vs_f4 vs_mfma(vs_bf8 a, vs_bf8 b, vs_f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// c[r][t] += a[r] . b[t] for R x TB independent accumulators, both operands in PL parts (largest first): the parts are the
// outer loop, small products first, so that an accumulator is not needed again right after it was written.
template <int PL, int R, int TB, class B>
__device__ __forceinline__ void vs_mfma_parts(const vs_bf8 (&a)[R][PL], const B& b, vs_f4 (&c)[R][TB]) {
    constexpr int pa[6] = {1, 2, 0, 1, 0, 0}, pb[6] = {1, 0, 2, 0, 1, 0};
#pragma unroll
    for (int q = PL == 3 ? 0 : 5; q < 6; ++q)
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int t = 0; t < TB; ++t) c[r][t] = vs_mfma(a[r][pa[q]], b(t, pb[q]), c[r][t]);
}

// v as the sum of PL bf16 (each rounding to nearest; exact for PL = 3, within 2^-9 |v| for PL = 1), two at a time
template <int PL>
__device__ __forceinline__ void vs_split(vs_f8 v, vs_bf8* out) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int p = 0; p < PL; ++p) {
        u4 bits;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f2 pair = {v[2 * i], v[2 * i + 1]};
            bits[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(pair, b2));
            if (p + 1 < PL) {
                v[2 * i] -= __uint_as_float(bits[i] << 16);
                v[2 * i + 1] -= __uint_as_float(bits[i] & 0xFFFF0000u);
            }
        }
        out[p] = __builtin_bit_cast(vs_bf8, bits);
    }
}

// ---- fragments ----------------------------------------------------------------------------------------------------
// S fragments (16 rows x 32 elements): [row / 16][KS][PL][lane] of 8 bf16, lane l holding row l % 16, elements 8 (l / 16)..
// T fragments (16 elements x 32 rows): [row / 32][2 KS][PL][lane], lane l holding element l % 16 and the rows in the order
// 16 (j / 4) + 4 (l / 16) + j % 4.  Rows past the end and elements past `dim` are zero.  One workgroup packs 32 rows.
// A fragment is one coalesced 1 KiB load of a wave, whatever the caller's row length, stride and alignment are.
template <int KS, int PL>
__global__ __launch_bounds__(256) void k_vs_pack(VsSrc src, uint4* __restrict__ S, uint4* __restrict__ T, float* __restrict__ group_max) {
    constexpr int DP = KS * 32, LD = DP + 4;
    __shared__ float tile[32 * LD];
    __shared__ float wmax[4];
    const int64_t row0 = (int64_t)blockIdx.x * 32;
    float big = 0.0f;
    for (int i = threadIdx.x; i < 32 * DP; i += 256) {
        const int r = i / DP, d = i % DP;
        const float v = (row0 + r < src.rows && d < src.dim) ? vs_load(src, row0 + r, d) : 0.0f;
        tile[r * LD + d] = v;
        big = fmaxf(big, fabsf(v));
    }
    for (int o = 32; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor(big, o));
    if ((threadIdx.x & 63) == 0) wmax[threadIdx.x >> 6] = big;
    __syncthreads();
    if (group_max && threadIdx.x == 0) group_max[blockIdx.x] = fmaxf(fmaxf(wmax[0], wmax[1]), fmaxf(wmax[2], wmax[3]));
    for (int i = threadIdx.x; i < 2 * KS * 64; i += 256) {
        const int lane = i & 63, f = i >> 6, rb = f / KS, ks = f % KS;
        const float* at = tile + (rb * 16 + (lane & 15)) * LD + ks * 32 + (lane >> 4) * 8;
        vs_f8 v;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = at[j];
        vs_bf8 part[PL];
        vs_split<PL>(v, part);
#pragma unroll
        for (int p = 0; p < PL; ++p)
            *(vs_bf8*)&S[((((int64_t)blockIdx.x * 2 + rb) * KS + ks) * PL + p) * 64 + lane] = part[p];
    }
    if (!T) return;
    for (int i = threadIdx.x; i < 2 * KS * 64; i += 256) {
        const int lane = i & 63, db = i >> 6;
        vs_f8 v;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = tile[((j >> 2) * 16 + (lane >> 4) * 4 + (j & 3)) * LD + db * 16 + (lane & 15)];
        vs_bf8 part[PL];
        vs_split<PL>(v, part);
#pragma unroll
        for (int p = 0; p < PL; ++p) *(vs_bf8*)&T[(((int64_t)blockIdx.x * 2 * KS + db) * PL + p) * 64 + lane] = part[p];
    }
}

// The bias of every id, padded to whole chunks: 0 where the caller gives none, -inf past the end (p = 0 there).  A mask of
// the type's lowest value becomes -inf too: next to it no logit keeps a bit, and float32 could not hold it in powers of two.
__global__ __launch_bounds__(256) void k_vs_bias(const float* __restrict__ bias, int32_t vocab, int32_t padded, float* __restrict__ out) {
    const int v = blockIdx.x * 256 + threadIdx.x;
    if (v < padded) out[v] = v >= vocab ? -INFINITY : !bias ? 0.0f : bias[v] <= VS_NOTHING ? -INFINITY : bias[v];
}

// ---- forward ------------------------------------------------------------------------------------------------------
struct VsFwd {
    const uint4 *xS, *wS;
    const float* bias;         // [padded vocabulary]
    int32_t has_bias;          // the caller gave one: -inf may stand anywhere (else only past `vocab`)
    int32_t vocab;
    int32_t n_tiles;           // token tiles of 16 TB rows
    int32_t splits;            // ranges of the vocabulary
    int32_t blocks;            // blocks of VS_BLOCK ids
    int32_t chunks;            // chunks of VS_CHUNK ids: 16 a block
    int64_t n_pad;             // row length of the partials
    float4* part;              // [splits][n_pad]: reference (in powers of two), sum of exps, sum of exp * exponent
    float* chunk_max;          // [n_pad][chunks] or null
};

// Sums of a row, relative to 2^ref: s of exp, e of exp * exponent (the entropy's).  A softmax in one pass: the reference
// follows the running maximum in steps of at least 2^VS_SLACK, so it moves a few times per row and the common step has no
// rescaling.  Eight terms are summed first, then up to VS_BLOCK / 4 of those, then these: sums of 262,144 terms keep
// their last bits.
struct VsStat {
    float ref, s, e, S, E;
    __device__ __forceinline__ void clear() { ref = VS_NOTHING; s = e = S = E = 0.0f; }
    __device__ __forceinline__ void flush() { S += s; E += e; s = e = 0.0f; }
    __device__ __forceinline__ void move(float now) {      // (a sum that vanishes takes its exponents with it: 0 * inf)
        const float d = ref - now, f = exp2f(d);
        e = f == 0.0f ? 0.0f : f * fmaf(d, s, e);
        E = f == 0.0f ? 0.0f : f * fmaf(d, S, E);
        s *= f; S *= f;
        ref = now;
    }
    __device__ __forceinline__ void join(float r2, float s2, float e2) {     // S and E with another range's
        const float now = fmaxf(ref, r2);
        if (now > ref) move(now);
        const float d = r2 - now, f = exp2f(d);
        E += f == 0.0f ? 0.0f : f * fmaf(d, s2, e2);
        S += s2 != s2 ? s2 : f * s2;
    }
};

// 32 streaming rows against the stationary ones: s[rb][t] += w . x
template <int KS, int PL, int TB>
__device__ __forceinline__ void vs_product(const uint4* w, const vs_bf8 (&x)[TB][KS][PL], vs_f4 (&s)[2][TB]) {
#pragma unroll
    for (int k = 0; k < KS; ++k) {
        vs_bf8 wf[2][PL];
#pragma unroll
        for (int rb = 0; rb < 2; ++rb)
#pragma unroll
            for (int p = 0; p < PL; ++p) wf[rb][p] = *(const vs_bf8*)&w[((rb * KS + k) * PL + p) * 64];
        vs_mfma_parts<PL, 2, TB>(wf, [&](int t, int p) { return x[t][k][p]; }, s);
    }
}

template <int KS, int PL, int TB>
__device__ __forceinline__ void vs_stationary(const uint4* S, int64_t tile, int lane, vs_bf8 (&x)[TB][KS][PL]) {
#pragma unroll
    for (int t = 0; t < TB; ++t)
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int p = 0; p < PL; ++p) x[t][k][p] = *(const vs_bf8*)&S[(((tile * TB + t) * KS + k) * PL + p) * 64 + lane];
}

template <int TB>
struct VsRowsOfTile {
    VsStat st[TB];
    float top[TB];
    vs_f4 keep[TB];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int t = 0; t < TB; ++t) { st[t].clear(); top[t] = -INFINITY; }
    }
    // the logits of 32 ids; MASKED: some may be -inf
    template <bool MASKED>
    __device__ __forceinline__ void add(const vs_f4 (&s)[2][TB]) {
#pragma unroll
        for (int t = 0; t < TB; ++t) {
            float mx = vs_max(vs_max(vs_max(s[0][t][0], s[0][t][1]), s[0][t][2]), vs_max(vs_max(s[0][t][3], s[1][t][0]), s[1][t][1]));
            mx = vs_max(vs_max(mx, s[1][t][2]), s[1][t][3]);
            top[t] = vs_max(top[t], mx);
            mx *= VS_LOG2E;
            const bool up = mx > st[t].ref + VS_SLACK;
            if (__any(up)) st[t].move(up ? mx : st[t].ref);
            float ls, le;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float e = fmaf(s[j >> 2][t][j & 3], VS_LOG2E, -st[t].ref);
                if (MASKED) e = vs_max(e, VS_TMIN);
                const float p = __builtin_amdgcn_exp2f(e);
                ls = j ? ls + p : p;
                le = j ? fmaf(p, e, le) : p * e;
            }
            st[t].s += ls;
            st[t].e += le;
        }
    }
    // 64 ids are done, the h-th of their block: their largest logits are stored with those of the rest of the block, sixteen
    // bytes a lane (WHOLE: the wave sees whole blocks), or at once
    template <bool WHOLE>
    __device__ __forceinline__ void chunk(const VsFwd& a, int64_t tile, int block, int h, int lane, bool live) {
        if (a.chunk_max) {
#pragma unroll
            for (int t = 0; t < TB; ++t) {
                float* to = a.chunk_max + ((tile * TB + t) * 16 + (lane & 15)) * a.chunks + block * 16 + (lane >> 4) * 4;
                if (WHOLE) {
                    if (h == 0) keep[t][0] = top[t];
                    else if (h == 1) keep[t][1] = top[t];
                    else if (h == 2) keep[t][2] = top[t];
                    else if (live) *(vs_f4*)to = vs_f4{keep[t][0], keep[t][1], keep[t][2], top[t]};
                } else if (live) to[h] = top[t];
                top[t] = -INFINITY;
            }
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
            for (int o = 16; o <= 32; o <<= 1) {
                const float r2 = __shfl_xor(st[t].ref, o), s2 = __shfl_xor(st[t].S, o), e2 = __shfl_xor(st[t].E, o);
                st[t].join(r2, s2, e2);
            }
        }
    }
    __device__ __forceinline__ void store(const VsFwd& a, int64_t tile, int split, int lane) {
        join_lanes();
#pragma unroll
        for (int t = 0; t < TB; ++t) {
            if (lane < 16) a.part[(int64_t)split * a.n_pad + (tile * TB + t) * 16 + lane] = make_float4(st[t].ref, st[t].S, st[t].E, 0.0f);
        }
    }
};

template <int TB>
__device__ __forceinline__ void vs_bias_init(const float* bias, int lane, vs_f4 (&s)[2][TB]) {
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) {
        const vs_f4 b = *(const vs_f4*)&bias[rb * 16 + (lane >> 4) * 4];
#pragma unroll
        for (int t = 0; t < TB; ++t) s[rb][t] = b;
    }
}

// The widest float32 rows (a stage would not fit LDS twice): a wave is a tile of 16 TB tokens against one range of the
// vocabulary and reads its fragments itself.
template <int KS, int PL, int TB>
__global__ __launch_bounds__(256, 2) void k_vs_forward(VsFwd a) {
    const int lane = threadIdx.x & 63;
    const int unit = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (unit >= a.n_tiles * a.splits) return;
    const int tile = unit % a.n_tiles, split = unit / a.n_tiles;
    const int b0 = (int)((int64_t)a.blocks * split / a.splits), b1 = (int)((int64_t)a.blocks * (split + 1) / a.splits);
    vs_bf8 x[TB][KS][PL];
    vs_stationary<KS, PL, TB>(a.xS, tile, lane, x);
    VsRowsOfTile<TB> rows;
    rows.clear();
    for (int b = b0; b < b1; ++b) {
        for (int h = 0; h < 4; ++h) {
#pragma unroll 1
            for (int row0 = b * VS_BLOCK + h * 64; row0 < b * VS_BLOCK + (h + 1) * 64; row0 += 32) {
                vs_f4 s[2][TB];
                vs_bias_init<TB>(a.bias + row0, lane, s);
                vs_product<KS, PL, TB>(a.wS + (int64_t)row0 / 16 * KS * PL * 64 + lane, x, s);
                if (a.has_bias || row0 + 32 > a.vocab) rows.template add<true>(s);      // the same in the whole grid
                else rows.template add<false>(s);
            }
            rows.template chunk<true>(a, tile, b, h, lane, true);
        }
        rows.flush();
    }
    rows.store(a, tile, split, lane);
}

// Many tokens: four waves, a tile each, share the streaming rows through LDS.  SR rows at a time are copied straight into
// LDS (they are packed in the order of the copy) while the SR before them are worked on: one barrier a step.
typedef const __attribute__((address_space(1))) void* vs_global_ptr;
typedef __attribute__((address_space(3))) void* vs_lds_ptr;
template <int N>               // 16-byte pieces, a multiple of 256
__device__ __forceinline__ void vs_stage(const uint4* from, uint4* to) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < N; i += 256)
        __builtin_amdgcn_global_load_lds((vs_global_ptr)(from + i + wave * 64 + lane), (vs_lds_ptr)(to + i + wave * 64), 16, 0, 0);
}

// This wave's copies into LDS have arrived: vmcnt 0, the other counters as they are.
__device__ __forceinline__ void vs_copies_done() { __builtin_amdgcn_s_waitcnt(0x0F70); }

// A stage: SR rows of fragments and their SR biases.  `to` and `from` are different stages, and the compiler has to know it
// (__restrict__ through an inlined function): else it waits for the copy under way before each read of LDS.
template <int KS, int PL, int SR>
struct VsStage {
    static constexpr int N = SR * KS * PL * 4, SIZE = N + SR / 4;
    static __device__ __forceinline__ void fetch(const uint4* w, const float* bias, uint4* to) {
        vs_stage<N>(w, to);
        if (threadIdx.x < SR)
            __builtin_amdgcn_global_load_lds((vs_global_ptr)(bias + threadIdx.x), (vs_lds_ptr)(to + N + (threadIdx.x & ~63) / 4), 4, 0, 0);
    }
    template <int TB>
    static __device__ __forceinline__ void step(const VsFwd& a, int base, bool more, const uint4* __restrict__ next, const float* __restrict__ next_bias,
                                                uint4* __restrict__ to, const uint4* __restrict__ from, const vs_bf8 (&x)[TB][KS][PL], VsRowsOfTile<TB>& rows, int64_t tile, bool live) {
        const int lane = threadIdx.x & 63;
        vs_copies_done();                  // (a barrier alone does not wait for them)
        __syncthreads();                   // `from` has arrived, and nobody reads `to` any more
        if (more) fetch(next, next_bias, to);
#pragma unroll 1
        for (int r = 0; r < SR; r += 32) {
            const int row0 = base + r;
            vs_f4 s[2][TB];
            vs_bias_init<TB>((const float*)(from + N) + r, lane, s);
            vs_product<KS, PL, TB>(from + r * KS * PL * 4 + lane, x, s);
            if (a.has_bias || row0 + 32 > a.vocab) rows.template add<true>(s);
            else rows.template add<false>(s);
            if (row0 & 32) rows.template chunk<true>(a, tile, row0 / VS_BLOCK, (row0 >> 6) & 3, lane, live);
        }
        if (((base + SR) & (VS_BLOCK - 1)) == 0) rows.flush();
    }
};

template <int KS, int PL, int TB, int SR>
__global__ __launch_bounds__(256, 2) void k_vs_forward_staged(VsFwd a) {
    using Stage = VsStage<KS, PL, SR>;
    __shared__ uint4 buf0[Stage::SIZE], buf1[Stage::SIZE];
    const int lane = threadIdx.x & 63;
    const int split = blockIdx.x % a.splits;
    const int tile = (blockIdx.x / a.splits) * 4 + (threadIdx.x >> 6);
    const bool live = tile < a.n_tiles;
    const int row_begin = (int)((int64_t)a.blocks * split / a.splits) * VS_BLOCK, row_end = (int)((int64_t)a.blocks * (split + 1) / a.splits) * VS_BLOCK;
    vs_bf8 x[TB][KS][PL];
    vs_stationary<KS, PL, TB>(a.xS, live ? tile : 0, lane, x);
    VsRowsOfTile<TB> rows;
    rows.clear();
    const uint4* w = a.wS + (int64_t)row_begin * KS * PL * 4;
    const float* bias = a.bias + row_begin;
    Stage::fetch(w, bias, buf0);
    for (int base = row_begin; base < row_end; base += 2 * SR) {
        w += SR * KS * PL * 4; bias += SR;
        Stage::template step<TB>(a, base, true, w, bias, buf1, buf0, x, rows, tile, live);
        w += SR * KS * PL * 4; bias += SR;
        Stage::template step<TB>(a, base + SR, base + 2 * SR < row_end, w, bias, buf0, buf1, x, rows, tile, live);
    }
    if (live) rows.store(a, tile, split, lane);
}

// The bias of one id: 0 where the caller gives none, -inf where it masks the id.
__device__ __forceinline__ float vs_bias_of(const float* bias, int64_t v) {
    const float b = bias ? bias[v] : 0.0f;
    return b <= VS_NOTHING ? -INFINITY : b;
}

// sum over the 16 lanes of a DPP row, in every lane of it
__device__ __forceinline__ float vs_row_sum(float v) {
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xF, 0xF, true));    // quad_perm [1,0,3,2]
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xF, 0xF, true));    // quad_perm [2,3,0,1]
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xF, 0xF, true));   // row_half_mirror
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x140, 0xF, 0xF, true));   // row_mirror
    return v;
}

// Few tokens: bound by the one reading of the weights, which are taken as they lie (no packing): a lane loads the eight
// elements of a row that its place in a fragment asks for, at whatever alignment they have.  The last piece of a row that is
// no whole number of pieces long is taken back from the row's end, with the elements before it weighted 0 in x: no read
// leaves the row (so there are eight elements at least).  A wave is a tile of 16 TB tokens against one range of the vocabulary; the four of a workgroup join theirs.
template <int PL> struct VsPiece;
template <> struct VsPiece<1> {            // of bf16: a fragment as it is
    vs_bf8 v;
    __device__ __forceinline__ void load(const VsSrc& s, int64_t row, int at) {
        struct __attribute__((packed, aligned(2))) Raw { uint32_t v[4]; };
        v = __builtin_bit_cast(vs_bf8, *(const Raw*)((const uint16_t*)s.p + row * s.ld + at));
    }
    __device__ __forceinline__ vs_f8 floats() const { return __builtin_convertvector(v, vs_f8); }
    __device__ __forceinline__ void parts(vs_bf8 (&out)[1]) const { out[0] = v; }
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
    __device__ __forceinline__ void parts(vs_bf8 (&out)[3]) const { vs_split<3>(v, out); }
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
    float* group_max;          // [ids / 32] or null
    VsFwd f;                   // chunks, blocks, n_pad, part, chunk_max; splits: workgroups of a tile
};
template <int KS, int PL, int TB>
__global__ __launch_bounds__(256, KS * PL > 30 ? 1 : 2) void k_vs_forward_raw(VsRaw a) {
    const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    constexpr int KG = PL == 1 ? (KS < 16 ? KS : 8) : KS <= 4 ? KS : 2;    // 32-element steps whose loads are under way together
    __shared__ float4 red[4][TB * 16];
    const int tile = blockIdx.y;
    int at[KS];
    vs_bf8 x[TB][KS][PL];
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
    VsRowsOfTile<TB> rows;
    rows.clear();
    const int units = gridDim.x * 4, unit = blockIdx.x * 4 + (threadIdx.x >> 6), pieces = a.f.blocks * 4;
    const int c0 = (int)((int64_t)pieces * unit / units), c1 = (int)((int64_t)pieces * (unit + 1) / units);
    for (int c = c0; c < c1; ++c) {
#pragma unroll 1
        for (int row0 = c * 64; row0 < (c + 1) * 64; row0 += 32) {
            // (loads first and together; the bias is added last, so that no wait for it stands before the products)
            VsPiece<PL> raw[2][KG], big;
            vs_f4 s[2][TB], b[2];
            big.clear();
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
                    for (int j = 0; j < 8; ++j) b[j >> 2][j & 3] = a.bias[min(row0 + (j >> 2) * 16 + quad * 4 + (j & 3), a.w.rows - 1)];
                }
#pragma unroll
                for (int k = 0; k < KG; ++k)
                    if (g + k < KS) {
                        vs_bf8 wf[2][PL];
#pragma unroll
                        for (int rb = 0; rb < 2; ++rb) {
                            big.measure(raw[rb][k]);
                            raw[rb][k].parts(wf[rb]);
                        }
                        vs_mfma_parts<PL, 2, TB>(wf, [&](int t, int p) { return x[t][g + k][p]; }, s);
                    }
                if (KG < KS) __builtin_amdgcn_sched_barrier(0);     // (the loads of all groups at once would spill)
            }
            if (a.bias || row0 + 32 > a.w.rows) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float q = a.bias ? b[j >> 2][j & 3] : 0.0f;
                    const bool gone = q <= VS_NOTHING || row0 + (j >> 2) * 16 + quad * 4 + (j & 3) >= a.w.rows;
#pragma unroll
                    for (int t = 0; t < TB; ++t) s[j >> 2][t][j & 3] = gone ? -INFINITY : s[j >> 2][t][j & 3] + q;
                }
            }
            if (a.group_max) {
                float m = big.largest();
                for (int o = 1; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
                if (lane == 0 && tile == 0) a.group_max[row0 / 32] = m;
            }
            if (a.bias || row0 + 32 > a.w.rows) rows.template add<true>(s);
            else rows.template add<false>(s);
        }
        rows.template chunk<false>(a.f, tile, c >> 2, c & 3, lane, true);
        if ((c & 3) == 3) rows.flush();
    }
    rows.join_lanes();
#pragma unroll
    for (int t = 0; t < TB; ++t)
        if (quad == 0) red[threadIdx.x >> 6][t * 16 + col] = make_float4(rows.st[t].ref, rows.st[t].S, rows.st[t].E, 0.0f);
    __syncthreads();
    if (threadIdx.x < TB * 16) {
        VsStat st;
        st.clear();
        for (int i = 0; i < 4; ++i) { const float4 q = red[i][threadIdx.x]; st.join(q.x, q.y, q.z); }
        a.f.part[(int64_t)blockIdx.x * a.f.n_pad + tile * TB * 16 + threadIdx.x] = make_float4(st.ref, st.S, st.E, 0.0f);
    }
}

// Joins the ranges of a row and takes the given token's log probability.  The token's own logit is summed in float64 (its
// rounding would otherwise show where the probability is near 1).  WAVES waves work on a row; returns its lse to them all.
struct VsJoin {
    VsSrc x, w;
    const float* bias;         // as the caller gave it, or null
    const int64_t* targets;    // or null
    const float4* part;
    int32_t n, splits;
    int64_t n_pad;
    float *logprob, *entropy, *lse;
};
template <int WAVES>
__device__ __forceinline__ float vs_join_row(const VsJoin& a, int64_t row, int tid, float4* red, double* dred) {
    const int lane = tid & 63, wave = tid >> 6;
    VsStat st;
    st.clear();
    for (int i = tid; i < a.splits; i += 64 * WAVES) {
        const float4 q = a.part[(int64_t)i * a.n_pad + row];
        st.join(q.x, q.y, q.z);
    }
    const int64_t t = a.targets ? a.targets[row] : -1;
    double dot = 0.0;
    if (t >= 0 && t < a.w.rows)
        for (int d = tid; d < a.w.dim; d += 64 * WAVES) dot += (double)vs_load(a.x, row, d) * (double)vs_load(a.w, t, d);
    for (int o = 1; o < 64; o <<= 1) {
        const float r2 = __shfl_xor(st.ref, o), s2 = __shfl_xor(st.S, o), e2 = __shfl_xor(st.E, o);
        st.join(r2, s2, e2);
        dot += __shfl_xor(dot, o);
    }
    if constexpr (WAVES > 1) {
        if (lane == 0) { red[wave] = make_float4(st.ref, st.S, st.E, 0.0f); dred[wave] = dot; }
        __syncthreads();
        st.clear();
        dot = 0.0;
        for (int i = 0; i < WAVES; ++i) { st.join(red[i].x, red[i].y, red[i].z); dot += dred[i]; }
    }
    const bool empty = st.S == 0.0f;                // nothing but -inf
    const double lse = empty ? -INFINITY : ((double)st.ref + (double)log2f(st.S)) * 0.6931471805599453;
    if (tid == 0) {
        a.lse[row] = (float)lse;
        if (a.entropy) {
            const float h = VS_LN2 * (log2f(st.S) - st.E / st.S);
            a.entropy[row] = empty || h < 0.0f ? 0.0f : h;
        }
        if (a.logprob) {
            float lp = 0.0f;
            if (t >= a.w.rows) lp = NAN;
            else if (t >= 0) {
                lp = empty ? -INFINITY : (float)(dot + (double)vs_bias_of(a.bias, t) - lse);
                if (lp > 0.0f) lp = 0.0f;
            }
            a.logprob[row] = lp;
        }
    }
    return (float)lse;
}
template <int WAVES>
__global__ __launch_bounds__(256) void k_vs_join(VsJoin a) {
    __shared__ float4 red[4];
    __shared__ double dred[4];
    const int64_t row = WAVES == 1 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
    if (row >= a.n) return;
    (void)vs_join_row<WAVES>(a, row, WAVES == 1 ? threadIdx.x & 63 : threadIdx.x, red, dred);
}

// ---- alternatives -------------------------------------------------------------------------------------------------
// The k largest logits of a row, ties to the lower id, in the order of the logits as float64 sums them.  The forward pass
// left each chunk's largest float32 logit m; a float32 sum is within d = 4 (D + 16) 2^-24 (|m| + 2 |x|_1 max |w|) of the true
// one.  At least k logits are no less than the k-th largest m - d, so only chunks with m + d at or above that can hold one
// of the k: a few more than k, of 16 ids each.  Their logits are formed again in float32, those that reach the bound once more in float64,
// and the best k of these few are ranked by counting.  A workgroup per row.
//
// The bound is taken over 256 groups of chunks (the k-th largest of the groups' largest m - d is a bound too, and rarely a
// lower one): one pass over the maxima.  Where too many chunks reach it (many equal logits, a zero vector), they are visited
// in ascending order, and once k logits are known a later one that cannot beat the k-th is skipped even when it ties.
#define VS_MAX_K 32
#define VS_CAND 1024
#define VS_LIST 256
struct VsTop {
    VsJoin join;               // the row's ranges are joined first
    const float* chunk_max;    // [rows][chunks]
    const float* group_max;    // [8 blocks] largest |w| of 32 ids
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

// x . row over 16 lanes (xs: x in LDS); the result is in all of them.  The last piece of a row that is no whole number of
// pieces long is taken back from the row's end, with the elements before it weighted 0 -- no read leaves the row.
template <bool BF16>
__device__ __forceinline__ float vs_dot16(const VsSrc& w, int64_t row, const float* xs, int l16) {
    constexpr int E = VsVec<BF16>::E;
    float s = 0.0f;
    if (w.dim < E) {
        if (l16 < w.dim) s = xs[l16] * vs_load(w, row, l16);
    } else {
        for (int d = l16 * E; d < w.dim; d += 16 * E) {
            const int at = min(d, w.dim - E);
            VsVec<BF16> v;
            v.load(w.p, row * w.ld + at);
#pragma unroll
            for (int i = 0; i < E; ++i) s = at + i >= d ? fmaf(xs[at + i], v.f[i], s) : s;
        }
    }
    return vs_row_sum(s);
}

template <bool BF16, int THREADS>
__global__ __launch_bounds__(THREADS) void k_vs_top(VsTop a) {
    const VsSrc &x = a.join.x, &w = a.join.w;
    __shared__ float xs[512];
    __shared__ float best[256];
    __shared__ double cv[VS_CAND], cw[VS_MAX_K];
    __shared__ int ci[VS_CAND], cj[VS_MAX_K];
    __shared__ float red[THREADS / 64];
    __shared__ uint32_t found[4];
    __shared__ uint16_t list[VS_LIST], rows[VS_CAND];
    __shared__ int n_cand, n_rows, n_list;
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = tid & 15, quarter = lane >> 4;
    const float* cm = a.chunk_max + row * a.chunks;
    const float lse = vs_join_row<THREADS / 64>(a.join, row, tid, (float4*)cv, cw);
    __syncthreads();
    if (lse != lse) {                       // no order among the logits
        if (tid < a.k) { a.ids[row * a.k + tid] = -1; a.logprobs[row * a.k + tid] = NAN; }
        return;
    }
    float l1 = 0.0f;
    for (int d = tid; d < x.dim; d += THREADS) { const float v = vs_load(x, row, d); xs[d] = v; l1 += fabsf(v); }
    for (int o = 1; o < 64; o <<= 1) l1 += __shfl_xor(l1, o);
    if (lane == 0) red[wave] = l1;
    if (tid == 0) n_cand = n_rows = n_list = 0;
    __syncthreads();
    l1 = 0.0f;
    for (int i = 0; i < THREADS / 64; ++i) l1 += red[i];
    __syncthreads();
    const float eps = 4.0f * (float)(x.dim + 16) * 5.9604645e-8f;
    auto widest = [&](int block) {          // eps 2 |x|_1 max |w| of the block
        const float4 p = *(const float4*)&a.group_max[block * 8], q = *(const float4*)&a.group_max[block * 8 + 4];
        return eps * 2.0f * l1 * fmaxf(fmaxf(fmaxf(p.x, p.y), fmaxf(p.z, p.w)), fmaxf(fmaxf(q.x, q.y), fmaxf(q.z, q.w)));
    };
    auto off = [&](int c, float m) { return fmaf(eps, fabsf(m), widest(c >> 4)); };
    float low = -INFINITY;
    if (a.chunks <= 256) {
        if (tid < a.chunks && cm[tid] > -INFINITY) low = cm[tid] - off(tid, cm[tid]);
    } else
#pragma unroll 2
    for (int c = tid * 4; c < a.chunks; c += THREADS * 4) {
        const float4 m = *(const float4*)&cm[c];
        const float g = widest(c >> 4);
        // (m - d is increasing in m; of -inf it is -inf)
        const float top = fmaxf(fmaxf(m.x, m.y), fmaxf(m.z, m.w));
        low = fmaxf(low, top - fmaf(eps, fabsf(top), g));
    }
    if (a.chunks <= 256) {
        if (tid < 256) best[tid] = low;
    } else {
        for (int o = 1; o < THREADS / 256; o <<= 1) low = fmaxf(low, __shfl_xor(low, o));
        if (tid % (THREADS / 256) == 0) best[tid / (THREADS / 256)] = low;
    }
    __syncthreads();
    {                                       // the k-th largest of the 256: the largest value with at least k not below it
        float t = -INFINITY;
        if (tid < 256) {
            const float mine = best[tid];
            int above = 0;
            for (int j = 0; j < 256; j += 4) {
                const float4 q = *(const float4*)&best[j];
                above += (q.x >= mine) + (q.y >= mine) + (q.z >= mine) + (q.w >= mine);
            }
            t = above >= a.k ? mine : -INFINITY;
            for (int o = 1; o < 64; o <<= 1) t = fmaxf(t, __shfl_xor(t, o));
            if (lane == 0) red[wave] = t;
        }
    }
    __syncthreads();
    const float bound = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    double least = -INFINITY;               // the k-th best so far once k are known: what comes later must beat it
    bool full = false;
    auto compact = [&]() {                  // keeps the best k of the candidates, in order
        __syncthreads();
        const int n = n_cand;
        for (int i = tid; i < n; i += THREADS) {
            int rank = 0;
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
    // the ids of a chunk that reach the bound, four at a time; the float64 logit of an id
    auto look = [&](int c, int i0, int i1, int tag) {
        const float d = off(c, cm[c]);
#pragma unroll 4
        for (int i = i0; i < i1; i += 4) {
            const int v = vs_chunk_row(c, i + quarter), u = min(v, w.rows - 1);
            const float s = vs_dot16<BF16>(w, u, xs, l16) + vs_bias_of(a.join.bias, u);
            if (l16 == 0 && v == u && s > -INFINITY && s + d >= bound) {
                const int at = atomicAdd(&n_rows, 1);
                if (at < VS_CAND) rows[at] = (uint16_t)(tag * VS_CHUNK + i + quarter);
            }
        }
    };
    int least_end = 0;                      // ids from here on had no part in `least`: equal ones come after it
    auto beaten = [&](double s, int v) { return full && (s < least || (s == least && v >= least_end)); };
    auto exact = [&](int v) {
        double s = 0.0;
        for (int q = lane; q < w.dim; q += 64) s = fma((double)xs[q], (double)vs_load(w, v, q), s);
        for (int o = 1; o < 64; o <<= 1) s += __shfl_xor(s, o);
        s += (double)vs_bias_of(a.join.bias, v);
        if (lane == 0 && !beaten(s, v)) {
            const int at = atomicAdd(&n_cand, 1);
            cv[at] = s; ci[at] = v;
        }
    };
    auto may = [&](int c, float m) {
        const float up = m + off(c, m);
        return m > -INFINITY && up >= bound && !beaten((double)up, (c >> 4) * VS_BLOCK);
    };
    // every chunk that may hold one of the k: usually a few more than k
#pragma unroll 2
    for (int c = tid * 4; c < a.chunks; c += THREADS * 4) {
        const float4 m = *(const float4*)&cm[c];
        const float g = widest(c >> 4);
        const float v[4] = {m.x, m.y, m.z, m.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (v[i] > -INFINITY && v[i] + fmaf(eps, fabsf(v[i]), g) >= bound) {
                const int at = atomicAdd(&n_list, 1);
                if (at < VS_LIST) list[at] = (uint16_t)(c + i);
            }
    }
    __syncthreads();
    bool done = n_list <= VS_LIST;
    if (done) {                             // all their ids at once, a chunk for each wave
        const int n = n_list;
        for (int i = wave; i < n; i += THREADS / 64) look(list[i], 0, VS_CHUNK, i);
        __syncthreads();
        done = n_rows <= VS_CAND;
        if (done) {
            const int nr = n_rows;
            for (int i = wave; i < nr; i += THREADS / 64) exact(vs_chunk_row(list[rows[i] / VS_CHUNK], rows[i] % VS_CHUNK));
        }
    }
    if (!done) {                            // many equal logits: block after block
        __syncthreads();
        for (int c0 = 0; c0 < a.chunks; c0 += 256) {
            const int c = c0 + tid;
            const bool want = tid < 256 && c < a.chunks && may(c, cm[c]);
            const unsigned long long bal = __ballot(want);
            if (lane == 0 && wave < 4) found[wave] = __popcll(bal);
            __syncthreads();
            int before = 0;
            for (int i = 0; i < min(wave, 4); ++i) before += found[i];
            const int nl = found[0] + found[1] + found[2] + found[3];
            if (want) list[before + __popcll(bal & ((1ull << lane) - 1ull))] = (uint16_t)c;
            __syncthreads();
            for (int i0 = 0; i0 < nl; i0 += 16) {
                if (tid == 0) n_rows = 0;
                __syncthreads();
                for (int i = i0 + wave; i < min(i0 + 16, nl); i += THREADS / 64)
                    if (may(list[i], cm[list[i]])) look(list[i], 0, VS_CHUNK, i - i0);
                __syncthreads();
                const int nr = n_rows;
                for (int i = wave; i < nr; i += THREADS / 64) exact(vs_chunk_row(list[i0 + rows[i] / VS_CHUNK], rows[i] % VS_CHUNK));
                __syncthreads();
                const bool crowded = n_cand > VS_CAND - 256;
                if (crowded) { compact(); least_end = ((list[min(i0 + 15, nl - 1)] >> 4) + 1) * VS_BLOCK; }
                __syncthreads();
            }
        }
    }
    compact();
    __syncthreads();
    if (tid < a.k) {
        const bool have = tid < n_cand;
        a.ids[row * a.k + tid] = have ? ci[tid] : -1;
        a.logprobs[row * a.k + tid] = have ? fminf((float)(cv[tid] - (double)lse), 0.0f) : -INFINITY;
    }
}

// ---- backward -----------------------------------------------------------------------------------------------------
// What the gradient kernels read of a row: lse in powers of two, and G = p (A + B e) + gl [v = target], e = log2 p.
struct VsRow {
    float* lse2;               // [n_pad]
    float* A;
    float* B;
    float* gl;
    int32_t* target;
};
__global__ __launch_bounds__(256) void k_vs_rows(const float* __restrict__ lse, const float* __restrict__ entropy, const int64_t* __restrict__ targets,
                                                 const float* __restrict__ g, const float* __restrict__ h, int32_t n, int64_t n_pad, int32_t vocab, VsRow r) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n_pad) return;
    // rows past the end and rows whose every id is masked: an lse that makes every p 0, whatever the bias is
    float l2 = -VS_NOTHING, A = 0.0f, B = 0.0f, gl = 0.0f;
    int32_t t = -1;
    if (i < n) {
        const float l = lse[i];
        const int64_t tt = targets ? targets[i] : -1;
        const bool empty = l == -INFINITY;
        float fix = 1.0f;                         // p is short of 2^-(rounding of l2); A and B make up for it
        if (!empty) {
            const double exact = (double)l * 1.4426950408889634;
            l2 = (float)exact;
            fix = exp2f((float)((double)l2 - exact));
        }
        if (tt >= 0 && g) gl = g[i];
        if (tt >= vocab) gl = NAN;
        t = tt >= 0 && tt < vocab ? (int32_t)tt : -1;
        A = -gl;
        if (h && !empty) { A -= h[i] * entropy[i]; B = -h[i] * VS_LN2; }
        A *= fix; B *= fix;
    }
    r.lse2[i] = l2; r.A[i] = A; r.B[i] = B; r.gl[i] = gl; r.target[i] = t;
}

struct VsBwd {
    const uint4 *stayS;        // stationary rows (columns of the product)
    const uint4 *flowS, *flowT;// streaming rows, and transposed
    const float* bias;         // padded, by id
    int32_t has_bias, has_entropy;
    int32_t vocab;
    VsRow row;                 // by token
    int32_t n_tiles, splits, groups;   // groups of 32 streaming rows
    int64_t stay_pad;          // rows of a partial
    float* part;               // [splits][stay_pad][32 KS]
    float* bias_part;          // [splits][stay_pad] (OF_IDS with a bias gradient)
};

// One wave: a tile of 16 TB stationary rows against one range of the streaming ones.  OF_IDS = false: the stationary rows
// are tokens, the result sum_v p' w_v with p' = p (A + B e), or p alone when there is no entropy gradient (A is then a
// factor of the whole row, applied at the end); the target's own term is added at the end too, so that the largest
// coefficient is never rounded to bf16.  OF_IDS = true: the stationary rows are ids, the result sum_n G_nv x_n; the few
// steps in which a token's target lies in the tile add the rounded-off part of G in a second product.
template <int KS, int PL, int TB, bool OF_IDS>
__global__ __launch_bounds__(256) void k_vs_backward(VsBwd a) {
    constexpr int DP = KS * 32;
    const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    const int unit = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (unit >= a.n_tiles * a.splits) return;
    const int tile = unit % a.n_tiles, split = unit / a.n_tiles;
    const int g0 = (int)((int64_t)a.groups * split / a.splits), g1 = (int)((int64_t)a.groups * (split + 1) / a.splits);
    const int64_t stay0 = (int64_t)tile * TB * 16;
    vs_bf8 y[TB][KS][PL];
    vs_stationary<KS, PL, TB>(a.stayS, tile, lane, y);
    float lse2[TB], A[TB], B[TB], b0[TB], db[TB];
#pragma unroll
    for (int t = 0; t < TB; ++t) {
        const int64_t r = stay0 + t * 16 + col;
        if constexpr (OF_IDS) { b0[t] = a.bias[r]; db[t] = 0.0f; }
        else { lse2[t] = a.row.lse2[r]; A[t] = a.row.A[r]; B[t] = a.row.B[r]; }
    }
    vs_f4 acc[2 * KS][TB];
#pragma unroll
    for (int d = 0; d < 2 * KS; ++d)
#pragma unroll
        for (int t = 0; t < TB; ++t) acc[d][t] = vs_f4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int g = g0; g < g1; ++g) {
        const int row0 = g * 32;
        vs_f4 s[2][TB];
        const bool biased = a.has_bias || (OF_IDS ? stay0 + TB * 16 > a.vocab : row0 + 32 > a.vocab);
#pragma unroll
        for (int rb = 0; rb < 2; ++rb) {
            vs_f4 b = {0.0f, 0.0f, 0.0f, 0.0f};
            if (!OF_IDS && biased) b = *(const vs_f4*)&a.bias[row0 + rb * 16 + quad * 4];
#pragma unroll
            for (int t = 0; t < TB; ++t) {
                if constexpr (OF_IDS) s[rb][t] = vs_f4{b0[t], b0[t], b0[t], b0[t]};
                else s[rb][t] = b;
            }
        }
        vs_product<KS, PL, TB>(a.flowS + (int64_t)g * 2 * KS * PL * 64 + lane, y, s);
        vs_f4 L[2], rA[2], rB[2];
        bool hit = false;
        if constexpr (OF_IDS) {
#pragma unroll
            for (int rb = 0; rb < 2; ++rb) {
                L[rb] = *(const vs_f4*)&a.row.lse2[row0 + rb * 16 + quad * 4];
                rA[rb] = *(const vs_f4*)&a.row.A[row0 + rb * 16 + quad * 4];
                if (a.has_entropy) rB[rb] = *(const vs_f4*)&a.row.B[row0 + rb * 16 + quad * 4];
            }
            const int64_t t = a.row.target[row0 + (lane & 31)];
            hit = __any(t >= stay0 && t < stay0 + TB * 16);
        }
        vs_bf8 P[TB][PL], R[TB];
#pragma unroll
        for (int t = 0; t < TB; ++t) {
            vs_f8 G;
#pragma unroll
            for (int rb = 0; rb < 2; ++rb)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float e = fmaf(s[rb][t][i], VS_LOG2E, OF_IDS ? -L[rb][i] : -lse2[t]);
                    if (biased) e = vs_max(e, VS_TMIN);
                    float q = __builtin_amdgcn_exp2f(e);
                    if constexpr (OF_IDS) q *= a.has_entropy ? fmaf(rB[rb][i], e, rA[rb][i]) : rA[rb][i];
                    else if (a.has_entropy) q *= fmaf(B[t], e, A[t]);
                    G[rb * 4 + i] = q;
                }
            if constexpr (OF_IDS) {
                if (hit) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int at = row0 + (j >> 2) * 16 + quad * 4 + (j & 3);
                        if (a.row.target[at] == (int32_t)(stay0 + t * 16 + col)) G[j] += a.row.gl[at];
                    }
                }
                if (a.bias_part)
#pragma unroll
                    for (int j = 0; j < 8; ++j) db[t] += G[j];
            }
            vs_split<PL>(G, P[t]);
            if (OF_IDS && PL == 1) R[t] = __builtin_convertvector(G - __builtin_convertvector(P[t][0], vs_f8), vs_bf8);
        }
        const uint4* ft = a.flowT + (int64_t)g * 2 * KS * PL * 64 + lane;
#pragma unroll
        for (int d = 0; d < 2 * KS; d += 2) {
            vs_bf8 wf[2][PL];
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int p = 0; p < PL; ++p) wf[r][p] = *(const vs_bf8*)&ft[((d + r) * PL + p) * 64];
            vs_mfma_parts<PL, 2, TB>(wf, [&](int t, int p) { return P[t][p]; }, *(vs_f4(*)[2][TB]) & acc[d]);
        }
        if (OF_IDS && PL == 1 && hit) {
#pragma unroll
            for (int d = 0; d < 2 * KS; ++d) {
                const vs_bf8 wf = *(const vs_bf8*)&ft[d * 64];
#pragma unroll
                for (int t = 0; t < TB; ++t) acc[d][t] = vs_mfma(wf, R[t], acc[d][t]);
            }
        }
    }
#pragma unroll
    for (int t = 0; t < TB; ++t) {
        const int64_t r = stay0 + t * 16 + col;
        float* out = a.part + ((int64_t)split * a.stay_pad + r) * DP;
#pragma unroll
        for (int d = 0; d < 2 * KS; ++d) *(vs_f4*)&out[d * 16 + quad * 4] = acc[d][t];
        if constexpr (OF_IDS) {
            if (a.bias_part) {
                float v = db[t] + __shfl_xor(db[t], 16);
                v += __shfl_xor(v, 32);
                if (quad == 0) a.bias_part[(int64_t)split * a.stay_pad + r] = v;
            }
        }
    }
}

// Sums the partials of a row in a fixed order and writes it: dx = A sum p w + gl w_t (without an entropy gradient; with
// one the partials hold p (A + B e) already), dw as it is, db beside it.
struct VsSum {
    const float* part;
    const float* bias_part;
    int32_t rows, dim, dp, splits;
    int64_t pad;
    VsRow row;                 // of tokens: null pointers for dw
    int32_t has_entropy;
    VsSrc w;
    void* out;
    int64_t ldo;
    int32_t out_bf16;
    float* db;
};
__device__ __forceinline__ void vs_store(void* p, int64_t at, float v, int bf16) {
    if (bf16) ((__bf16*)p)[at] = (__bf16)v;
    else ((float*)p)[at] = v;
}
__global__ __launch_bounds__(256) void k_vs_sum(VsSum a) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (a.db && i < a.rows) {
        float v = 0.0f;
        for (int s = 0; s < a.splits; ++s) v += a.bias_part[(int64_t)s * a.pad + i];
        a.db[i] = v;
    }
    if (i >= (int64_t)a.rows * a.dim) return;
    const int64_t r = i / a.dim;
    const int d = (int)(i % a.dim);
    float v = 0.0f;
    for (int s = 0; s < a.splits; ++s) v += a.part[((int64_t)s * a.pad + r) * a.dp + d];
    if (a.row.A) {
        if (!a.has_entropy) v *= a.row.A[r];
        const int32_t t = a.row.target[r];
        if (t >= 0) v = fmaf(a.row.gl[r], vs_load(a.w, t, d), v);
        else if (a.row.gl[r] != a.row.gl[r]) v = a.row.gl[r];
    }
    vs_store(a.out, r * a.ldo + d, v, a.out_bf16);
}

// no tokens: dw = 0, db = 0
__global__ __launch_bounds__(256) void k_vs_zero(void* out, int64_t ldo, int32_t rows, int32_t dim, int32_t out_bf16, float* db) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (db && i < rows) db[i] = 0.0f;
    if (i < (int64_t)rows * dim) vs_store(out, i / dim * ldo + i % dim, 0.0f, out_bf16);
}
