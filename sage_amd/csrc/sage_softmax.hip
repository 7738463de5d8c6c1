// Host side of the vocabulary softmax and of gradient clipping (include/sage_hip.h).  gfx950 (MI355X) only.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdio>
#include <utility>
#include <vector>

#include "sage_internal.h"
#include "sage_softmax.h"
#include "sage_clip.h"

namespace {

constexpr int64_t VS_PAD = 128;                 // rows are padded to this (ids to VS_BLOCK)
constexpr int64_t VS_ROWS_MAX = 16384;          // tokens of one pass of the forward kernels (their chunks' maxima: 1 GB for 262,144 ids)
constexpr int64_t VS_RAW = 512;                 // at most this many tokens read the weights as they lie
constexpr size_t VS_ALIGN = 256;

inline int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }
inline uint32_t cdiv(int64_t a, int64_t b) { return (uint32_t)((a + b - 1) / b); }

// Makes the context's device current for a call and puts the caller's back.
struct OnDevice {
    int before = -1;
    bool ok = false;
    explicit OnDevice(int device) {
        if (hipGetDevice(&before) != hipSuccess) before = -1;
        ok = before == device || hipSetDevice(device) == hipSuccess;
        if (before == device) before = -1;
    }
    ~OnDevice() { if (before >= 0) (void)hipSetDevice(before); }
};

struct Arena {                                   // offsets first (base null), pointers later
    char* base = nullptr;
    int64_t used = 0;
    template <class T> T* take(int64_t n) {
        T* p = base ? reinterpret_cast<T*>(base + used) : nullptr;
        used += up(n * (int64_t)sizeof(T), VS_ALIGN);
        return p;
    }
};

int launched(sage_ctx* c, const char* what) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return SAGE_OK;
    char msg[256];
    std::snprintf(msg, sizeof msg, "%s: %s", what, hipGetErrorString(e));
    return sage_ctx_fail(c, SAGE_E_HIP, msg);
}

// 32-element steps of the padded row width: the instantiations there are
int vs_steps(int dim) {
    const int opts[] = {2, 4, 8, 10, 16};
    for (int o : opts) if (dim <= o * 32) return o;
    return 0;
}

// How each width runs.  ks: 32-element steps of the padded row; pl: parts of a packed element (1 bf16, 2 float32).
// Columns of a tile (the matrix instruction's) and tiles of a wave, as measured for each width (ks = 2, 4, 8, 10, 16 at
// D = 50, 100, 200, 300, 500, 4,096 tokens x 65,536 ids, D = 50 twice that both ways; us, the choice taken first, then the others of 16 and 32
// columns, one and two tiles, fastest first; without an entropy gradient, dw with its launches):
//   forward   32x2 32x2 16x2 32x2 32x1   float32   436 [460 461 518]   189 [198 205 234]   337 [358 399 700]     474 [508 552 781]     820 [953 1144 1388]
//             32x2 32x2 32x2 32x2 16x2   bf16      281 [288 309 334]   106 [105 108 120]   148 [158 164 198]     177 [182 193 217]     269 [286 337 613]
//   with alternatives the registers of the largest logits decide too
//             16x2 32x2 16x2 32x2 32x1   float32   548 [551 585 610]   238 [248 256 287]   410 [429 472 1027]    588 [648 669 908]     1063 [1213 1515 2118]
//             32x2 32x2 32x2 16x2 16x2   bf16      448 [407 426 441]   161 [156 159 171]   217 [231 232 272]     266 [274 295 408]     372 [390 440 988]
//   dx        16x2 16x2 16x1 16x2 16x1   float32   743 [727 768 828]   363 [377 418 477]   758 [911 1310 3436]   1310 [1686 2945 ..]  2677 [4810 7132 ..]
//             16x2 16x2 16x1 16x1 16x1   bf16      308 [311 326 358]   150 [160 168 202]   299 [311 359 447]     393 [1575 2526 ..]   620 [2428 2790 ..]
//   dw        16x2 16x2 16x1 16x2 16x1   float32   759 [740 801 853]   342 [370 423 508]   763 [923 954 3506]    1385 [1553 1768 ..]  2561 [4876 7436 ..]
//             16x2 16x2 16x1 16x1 16x2   bf16      311 [328 367 377]   134 [163 186 534]   359 [370 387 434]     392 [485 494 1834]    684 [744 935 5282]
// (The gradients take 16 columns throughout: 32 gain 2 % at the narrowest width alone, and wider ones than that spill their sums.)
constexpr int vs_fwd_tile(int ks, int pl, bool top) {
    if (pl == 1 ? ks == 10 : ks == 2) return top ? 16 : 32;
    return pl == 1 ? (ks <= 8 ? 32 : 16) : ks == 8 ? 16 : 32;
}
constexpr int vs_fwd_blocks(int ks, int pl) { return pl == 2 && ks == 16 ? 1 : 2; }
constexpr int vs_bwd_tile(int, int) { return 16; }
constexpr int vs_bwd_blocks(int ks, int pl, bool of_ids) { return ks <= 4 || (pl == 2 && ks == 10) || (pl == 1 && ks == 16 && of_ids) ? 2 : 1; }
// streaming rows of a stage: two stages of 16 to 64 KiB
constexpr int vs_fwd_rows(int ks, int pl) { return ks * pl <= 2 ? 128 : ks * pl <= 8 ? 64 : 32; }
constexpr int vs_bwd_rows(int, int) { return 32; }
constexpr bool vs_bwd_turns(int ks, int) { return ks >= 8; }
// 16-token blocks of a wave that reads the weights as they lie (the three bf16 parts of float32 are formed there)
constexpr int vs_raw_parts(int pl) { return pl == 1 ? 1 : 3; }
constexpr int vs_raw_most(int ks, int pl) { return ks * vs_raw_parts(pl) <= 10 ? 2 : 1; }

#define VS_BY_WIDTH(ks, pl, F)                                                        \
    do {                                                                              \
        if ((pl) == 1) {                                                              \
            switch (ks) {                                                             \
            case 2: { F(2, 1); break; }                                               \
            case 4: { F(4, 1); break; }                                               \
            case 8: { F(8, 1); break; }                                               \
            case 10: { F(10, 1); break; }                                             \
            default: { F(16, 1); break; }                                             \
            }                                                                         \
        } else {                                                                      \
            switch (ks) {                                                             \
            case 2: { F(2, 2); break; }                                               \
            case 4: { F(4, 2); break; }                                               \
            case 8: { F(8, 2); break; }                                               \
            case 10: { F(10, 2); break; }                                             \
            default: { F(16, 2); break; }                                             \
            }                                                                         \
        }                                                                             \
    } while (0)

struct Shape {
    int64_t n, vocab, vp;        // tokens, ids, padded ids
    int dim, ks, pl, k, cus;
};

template <int KS, int PL, bool TOP> constexpr auto vs_fwd_kernel = &k_vs_forward<KS, PL, vs_fwd_tile(KS, PL, TOP), vs_fwd_blocks(KS, PL), vs_fwd_rows(KS, PL), TOP>;
template <int KS, int PL, bool OF_IDS, bool ENTROPY, bool SUMS = true>
constexpr auto vs_bwd_kernel = &k_vs_backward<KS, PL, vs_bwd_tile(KS, PL), vs_bwd_blocks(KS, PL, OF_IDS), vs_bwd_rows(KS, PL), vs_bwd_turns(KS, PL), OF_IDS, ENTROPY, SUMS>;

// workgroups of a kernel that a CU holds at once (the same on every gfx950)
template <auto KERNEL>
int per_cu() {
    static std::atomic<int> cached{0};
    int n = cached.load(std::memory_order_relaxed);
    if (!n) {
        if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, KERNEL, 256, 0) != hipSuccess || n < 1) n = 1;
        cached.store(n, std::memory_order_relaxed);
    }
    return n;
}

// Into how many ranges the streaming axis (of `units` pieces) is cut, for `groups` workgroups along the other: the number that
// ends soonest if the chip works `resident` workgroups off at a time, each as long as its pieces and `cost` more to start
// and end (the loading of its stationary rows; for the gradients the writing and adding of its sums too).  No cost at all
// and three times as much measure within 2 % of these (6 shapes, 129 x 1,200 to 8,192 x 65,536).
int vs_splits(int64_t resident, int64_t groups, int64_t units, double cost) {
    const int64_t most = std::min(units, std::max<int64_t>(1, 4 * resident / groups));
    int64_t best = 1;
    double least = 1e300;
    for (int64_t s = 1; s <= most; ++s) {
        const double t = (double)((groups * s + resident - 1) / resident) * ((double)((units + s - 1) / s) + cost);
        if (t < least) { least = t; best = s; }
    }
    return (int)best;
}

// Token blocks (of 16) of a wave that reads the weights as they lie, one, or two where registers allow and tokens are there;
// 0: the weights are packed first.  Packing costs a launch and a pass over the weights, reading them as they lie one such pass per
// tile: worth it for 2 tiles (3 of two blocks), and for more where the vocabulary is short.  Measured, us, as they lie / packed:
//   D = 50 float32, 262,144 ids   64 tokens 39 / 57   128: 67 / 57      16,384 ids   256: 14 / 22   384: 18 / 22    32,768   512: 35 / 25
//   D = 300 bf16, 131,072 ids     64: 46 / 65   128: 74 / 65            8,192 ids    256: 15 / 28                  32,768   256: 32 / 34
//   D = 300 float32, 131,072 ids  32: 75 / 128   64: 139 / 138          8,192 ids    128: 19 / 45
//   D = 512 bf16, 131,072 ids     32: 71 / 80   64: 127 / 81            1,200 ids    512: 20 / 27                  32,768   96: 51 / 36
int vs_raw_blocks(const Shape& s) {
    if (s.n > VS_RAW || s.dim < 8) return 0;
    int most = 1;
#define VS_F(KS, PL) most = vs_raw_most(KS, PL)
    VS_BY_WIDTH(s.ks, s.pl, VS_F);
#undef VS_F
    const int64_t tiles = cdiv(s.n, most * 16);
    if ((tiles - most - 1) * s.vp * (s.ks + 8) > (1 << 20)) return 0;
    return s.n <= 16 ? 1 : most;
}

struct FwdPlan {
    int64_t rows, n_pad, tiles, chunks;
    int splits;
    int raw;                    // 16-token blocks of a tile of k_vs_forward_raw (0: the weights are packed)
    uint4 *xS, *wS;
    float *info, *x_exp, *wide;
    _Float16* chunk_max;
    float4* part;
    int64_t bytes;
};
FwdPlan plan_fwd(const Shape& s, void* ws) {
    FwdPlan p{};
    Arena a{(char*)ws};
    const int64_t blocks = s.vp / VS_BLOCK, frag = (int64_t)s.ks * s.pl * 64;          // uint4 of a 16-row block
    p.chunks = s.vp / VS_CHUNK;
    p.raw = vs_raw_blocks(s);
    if (p.raw) {
        p.rows = s.n;
        p.tiles = cdiv(s.n, p.raw * 16);
        p.n_pad = p.tiles * p.raw * 16;
        p.splits = (int)std::min<int64_t>(blocks, s.cus * 4);     // a wave has 64 ids at least
    } else {
        p.rows = std::min(s.n, VS_ROWS_MAX);
        p.n_pad = up(p.rows, VS_PAD);
        int64_t resident = s.cus;
#define VS_F(KS, PL)                                                                        \
    p.tiles = cdiv(p.rows, vs_fwd_blocks(KS, PL) * vs_fwd_tile(KS, PL, s.k > 0));           \
    resident *= s.k > 0 ? per_cu<vs_fwd_kernel<KS, PL, true>>() : per_cu<vs_fwd_kernel<KS, PL, false>>()
        VS_BY_WIDTH(s.ks, s.pl, VS_F);
#undef VS_F
        p.splits = vs_splits(resident, cdiv(p.tiles, 4), blocks, 1.0);
        p.wS = a.take<uint4>(s.vp / 16 * frag);
        p.xS = a.take<uint4>(p.n_pad / 16 * frag);
        p.info = a.take<float>(s.vp / 32 * VS_INFO);
        p.x_exp = a.take<float>(p.n_pad);
    }
    p.part = a.take<float4>(p.splits * p.n_pad);
    p.wide = a.take<float>(p.splits);
    p.chunk_max = a.take<_Float16>(s.k ? p.n_pad * p.chunks : 0);
    p.bytes = a.used;
    return p;
}

struct BwdPlan {
    int64_t np, tiles_x, tiles_w;
    int splits_x, splits_w;
    uint4 *xS, *xT, *wS, *wT;
    float *info, *tokens, *part_x, *part_w, *bias_part, *rest, *target_e;
    int64_t bytes;
};
// (one plan, with and without an entropy gradient)
BwdPlan plan_bwd(const Shape& s, void* ws) {
    BwdPlan p{};
    Arena a{(char*)ws};
    p.np = up(s.n, VS_PAD);
    int64_t units_w = 1, units_x = 1, resident_x = s.cus, resident_w = s.cus;
#define VS_F(KS, PL)                                                                            \
    p.tiles_x = cdiv(s.n, vs_bwd_blocks(KS, PL, false) * vs_bwd_tile(KS, PL)); p.tiles_w = cdiv(s.vocab, vs_bwd_blocks(KS, PL, true) * vs_bwd_tile(KS, PL)); \
    units_x = s.vp / vs_bwd_rows(KS, PL); units_w = p.np / vs_bwd_rows(KS, PL);                 \
    resident_x *= std::min(per_cu<vs_bwd_kernel<KS, PL, false, false>>(), per_cu<vs_bwd_kernel<KS, PL, false, true>>());        \
    resident_w *= std::min(per_cu<vs_bwd_kernel<KS, PL, true, false>>(), per_cu<vs_bwd_kernel<KS, PL, true, true>>())
    VS_BY_WIDTH(s.ks, s.pl, VS_F);
#undef VS_F
    p.splits_x = vs_splits(resident_x, cdiv(p.tiles_x, 4), units_x, 8.0);
    p.splits_w = vs_splits(resident_w, cdiv(p.tiles_w, 4), units_w, 8.0);
    const int64_t frag = (int64_t)s.ks * s.pl * 64;
    p.wS = a.take<uint4>(s.vp / 16 * frag);
    p.wT = a.take<uint4>(s.vp / 16 * frag);
    p.xS = a.take<uint4>(p.np / 16 * frag);
    p.xT = a.take<uint4>(p.np / 16 * frag);
    p.info = a.take<float>(s.vp / 32 * VS_INFO);
    p.tokens = a.take<float>(p.np / 32 * VS_TOKEN);
    p.part_x = a.take<float>(p.splits_x * p.np * s.ks * 32);
    p.part_w = a.take<float>(p.splits_w > 1 ? p.splits_w * s.vp * s.ks * 32 : 0);
    p.bias_part = a.take<float>(p.splits_w > 1 ? p.splits_w * s.vp : 0);
    p.rest = a.take<float>(p.splits_x * p.np);
    p.target_e = a.take<float>(p.np);
    p.bytes = a.used;
    return p;
}

int vs_shape(sage_ctx* c, int32_t dtype, int64_t n, int64_t vocab, int32_t dim, int32_t k, Shape* s) {
    if (dtype != SAGE_F32 && dtype != SAGE_BF16) return sage_ctx_fail(c, SAGE_E_ARG, "dtype must be SAGE_F32 or SAGE_BF16");
    if (n < 0 || vocab < 1 || dim < 1) return sage_ctx_fail(c, SAGE_E_ARG, "need n >= 0, vocab >= 1 and dim >= 1");
    if (k < 0 || k > VS_MAX_K) return sage_ctx_fail(c, SAGE_E_LIMIT, "at most 32 alternatives");
    if (dim > 512) return sage_ctx_fail(c, SAGE_E_LIMIT, "embedding dimension above 512 is not supported");
    if (vocab > (1 << 20)) return sage_ctx_fail(c, SAGE_E_LIMIT, "a vocabulary of more than 2^20 ids is not supported");
    if (n > (1 << 22)) return sage_ctx_fail(c, SAGE_E_LIMIT, "more than 2^22 tokens in one call are not supported");
    *s = Shape{n, vocab, up(vocab, VS_BLOCK), dim, vs_steps(dim), dtype == SAGE_BF16 ? 1 : 2, k, sage_ctx_compute_units(c)};
    return SAGE_OK;
}

int check_matrix(sage_ctx* c, const char* what, const void* p, int64_t ld, int32_t dim, int32_t dtype) {
    char msg[128];
    const int size = dtype == SAGE_BF16 ? 2 : 4;
    if (!p) std::snprintf(msg, sizeof msg, "%s is null", what);
    else if (ld < dim) std::snprintf(msg, sizeof msg, "%s: rows overlap (stride %lld, dimension %d)", what, (long long)ld, (int)dim);
    else if ((uintptr_t)p % size) std::snprintf(msg, sizeof msg, "%s is not aligned to its elements", what);
    else return SAGE_OK;
    return sage_ctx_fail(c, SAGE_E_ARG, msg);
}

int check_workspace(sage_ctx* c, const void* p, int64_t have, int64_t need) {
    char msg[128];
    if (!p || (uintptr_t)p % VS_ALIGN) std::snprintf(msg, sizeof msg, "the workspace must be aligned to 256 bytes");
    else if (have < need) std::snprintf(msg, sizeof msg, "the workspace holds %lld bytes, %lld are needed", (long long)have, (long long)need);
    else return SAGE_OK;
    return sage_ctx_fail(c, SAGE_E_ARG, msg);
}

template <bool FORWARD, bool TOP = false>
void pack(const Shape& s, const VsPack& a, const VsPack& b, hipStream_t st) {
#define VS_F(KS, PL) k_vs_pack<KS, PL, FORWARD ? vs_fwd_tile(KS, PL, TOP) : vs_bwd_tile(KS, PL), FORWARD><<<(uint32_t)(a.groups + b.groups), 256, 0, st>>>(a, b)
    VS_BY_WIDTH(s.ks, s.pl, VS_F);
#undef VS_F
}
VsPack pack_of(const VsSrc& src, uint4* S, uint4* T, int64_t padded) {
    VsPack p{};
    p.src = src; p.S = S; p.T = T; p.groups = (int32_t)(padded / 32);
    return p;
}

VsSrc rows_from(const VsSrc& m, int64_t row, int64_t rows) {
    VsSrc r = m;
    r.p = (const char*)m.p + row * m.ld * (m.is_bf16 ? 2 : 4);
    r.rows = (int32_t)rows;
    return r;
}

}  // namespace

extern "C" {

int64_t sage_token_logprobs_workspace(sage_ctx* c, int32_t dtype, int64_t n, int64_t vocab, int32_t dim, int32_t alternatives) {
    if (!c) return SAGE_E_ARG;
    Shape s;
    const int rc = vs_shape(c, dtype, n, vocab, dim, alternatives, &s);
    if (rc) return rc;
    return n ? plan_fwd(s, nullptr).bytes : 0;
}

int sage_token_logprobs_device(sage_ctx* c, int32_t dtype, int64_t n, int64_t vocab, int32_t dim, const void* d_x, int64_t ldx,
                               const void* d_weight, int64_t ldw, const float* d_bias, const int64_t* d_targets, int32_t alternatives,
                               float* d_logprob, float* d_entropy, float* d_lse, int32_t* d_alt_ids, float* d_alt_logprobs,
                               void* d_workspace, int64_t workspace_bytes, void* stream) {
    if (!c) return SAGE_E_ARG;
    Shape s;
    int rc = vs_shape(c, dtype, n, vocab, dim, alternatives, &s);
    if (rc) return rc;
    if (!d_lse && n) return sage_ctx_fail(c, SAGE_E_ARG, "d_lse is null");
    if (alternatives && n && (!d_alt_ids || !d_alt_logprobs)) return sage_ctx_fail(c, SAGE_E_ARG, "alternatives need d_alt_ids and d_alt_logprobs");
    if (d_logprob && n && !d_targets) return sage_ctx_fail(c, SAGE_E_ARG, "d_logprob needs d_targets");
    if (n && (rc = check_matrix(c, "d_x", d_x, ldx, dim, dtype))) return rc;
    if ((rc = check_matrix(c, "d_weight", d_weight, ldw, dim, dtype))) return rc;
    if (n == 0) return SAGE_OK;
    const FwdPlan p = plan_fwd(s, d_workspace);
    if ((rc = check_workspace(c, d_workspace, workspace_bytes, p.bytes))) return rc;
    OnDevice dev(sage_ctx_device(c));
    if (!dev.ok) return sage_ctx_fail(c, SAGE_E_HIP, "the context's device cannot be made current");
    const hipStream_t st = (hipStream_t)stream;
    const VsSrc w{d_weight, ldw, (int32_t)vocab, dim, dtype == SAGE_BF16}, x{d_x, ldx, (int32_t)n, dim, dtype == SAGE_BF16};
    VsPack of_w = pack_of(w, p.wS, nullptr, s.vp);
    of_w.info = p.info; of_w.bias = d_bias;
    for (int64_t r0 = 0; r0 < n; r0 += p.rows) {
        const int64_t rows = std::min(p.rows, n - r0);
        const VsSrc xr = rows_from(x, r0, rows);
        const int64_t* targets = d_targets ? d_targets + r0 : nullptr;
        const VsFwd f{p.xS, p.wS, p.info, p.x_exp, d_bias != nullptr, (int32_t)vocab, targets, (int32_t)rows, (int32_t)p.tiles, p.splits, (int32_t)(s.vp / VS_BLOCK), (int32_t)p.chunks,
                      p.n_pad, p.part, p.wide, alternatives ? p.chunk_max : nullptr};
        if (p.raw) {
            const VsRaw q{xr, w, d_bias, f};
            const dim3 grid(p.splits, (uint32_t)p.tiles);
#define VS_F(KS, PL)                                                                                                            \
    if constexpr (vs_raw_most(KS, PL) > 1)                                                                                      \
        if (p.raw > 1) { k_vs_forward_raw<KS, vs_raw_parts(PL), vs_raw_most(KS, PL)><<<grid, 256, 0, st>>>(q); break; }         \
    k_vs_forward_raw<KS, vs_raw_parts(PL), 1><<<grid, 256, 0, st>>>(q)
            VS_BY_WIDTH(s.ks, s.pl, VS_F);
#undef VS_F
        } else {
            if (r0) of_w.groups = 0;               // packed with the first rows
            VsPack of_x = pack_of(xr, p.xS, nullptr, p.n_pad);
            of_x.exps = p.x_exp;
            if (alternatives) pack<true, true>(s, of_w, of_x, st); else pack<true, false>(s, of_w, of_x, st);
            const uint32_t grid = cdiv(p.tiles, 4) * p.splits;
#define VS_F(KS, PL) if (alternatives) vs_fwd_kernel<KS, PL, true><<<grid, 256, 0, st>>>(f); else vs_fwd_kernel<KS, PL, false><<<grid, 256, 0, st>>>(f)
            VS_BY_WIDTH(s.ks, s.pl, VS_F);
#undef VS_F
        }
        const VsJoin j{xr, w, d_bias, targets, p.part, alternatives ? p.wide : nullptr, (int32_t)rows, p.splits, p.n_pad,
                       d_logprob ? d_logprob + r0 : nullptr, d_entropy ? d_entropy + r0 : nullptr, d_lse + r0};
        if (alternatives) {
            const VsTop t{j, p.chunk_max, (int32_t)p.chunks, alternatives, d_alt_ids + r0 * alternatives, d_alt_logprobs + r0 * alternatives};
            // a row alone on a CU is bound by latency: sixteen waves share its chain of loads (262,144 ids, D = 50, with the forward
            // kernel: one row 26.7 us, 28.7 by four waves; 256 rows 75 and 76; 320 rows 96 and 88)
            const bool wide = rows <= s.cus;
            if (dtype == SAGE_BF16) { if (wide) k_vs_top<true, 1024><<<(uint32_t)rows, 1024, 0, st>>>(t); else k_vs_top<true, 256><<<(uint32_t)rows, 256, 0, st>>>(t); }
            else { if (wide) k_vs_top<false, 1024><<<(uint32_t)rows, 1024, 0, st>>>(t); else k_vs_top<false, 256><<<(uint32_t)rows, 256, 0, st>>>(t); }
        // few rows, or many ranges: four waves share a row's ranges, or one joins them while another takes the target's logit (with the
        // forward kernel: one token, 1,024 ranges 19.1 us, 23.1 by one wave; 87 tokens, 64 ranges 10.7 and 11.7; 8,192 of a few 221 and 217)
        } else if (rows <= s.cus || p.splits > 64) k_vs_join<4><<<(uint32_t)rows, 256, 0, st>>>(j);
        else k_vs_join<1><<<cdiv(rows, 4), 256, 0, st>>>(j);
    }
    return launched(c, "sage_token_logprobs_device");
}

int64_t sage_token_logprobs_backward_workspace(sage_ctx* c, int32_t dtype, int64_t n, int64_t vocab, int32_t dim) {
    if (!c) return SAGE_E_ARG;
    Shape s;
    const int rc = vs_shape(c, dtype, n, vocab, dim, 0, &s);
    if (rc) return rc;
    return n ? plan_bwd(s, nullptr).bytes : 0;
}

int sage_token_logprobs_backward_device(sage_ctx* c, int32_t dtype, int64_t n, int64_t vocab, int32_t dim, const void* d_x, int64_t ldx,
                                        const void* d_weight, int64_t ldw, const float* d_bias, const int64_t* d_targets,
                                        const float* d_lse, const float* d_entropy, const float* d_grad_logprob, const float* d_grad_entropy,
                                        void* d_dx, int64_t lddx, void* d_dweight, int64_t lddw, float* d_dbias, void* d_workspace,
                                        int64_t workspace_bytes, void* stream) {
    if (!c) return SAGE_E_ARG;
    Shape s;
    int rc = vs_shape(c, dtype, n, vocab, dim, 0, &s);
    if (rc) return rc;
    if (n && !d_lse) return sage_ctx_fail(c, SAGE_E_ARG, "d_lse is null");
    if (n && !d_grad_logprob && !d_grad_entropy) return sage_ctx_fail(c, SAGE_E_ARG, "no gradient is given");
    if (n && d_grad_logprob && !d_targets) return sage_ctx_fail(c, SAGE_E_ARG, "d_grad_logprob needs d_targets");
    if (n && d_grad_entropy && !d_entropy) return sage_ctx_fail(c, SAGE_E_ARG, "d_grad_entropy needs d_entropy");
    if (!d_dx && !d_dweight && !d_dbias) return sage_ctx_fail(c, SAGE_E_ARG, "no result is asked for");
    if (d_dbias && !d_dweight) return sage_ctx_fail(c, SAGE_E_ARG, "d_dbias comes with d_dweight");
    if (n && (rc = check_matrix(c, "d_x", d_x, ldx, dim, dtype))) return rc;
    if ((rc = check_matrix(c, "d_weight", d_weight, ldw, dim, dtype))) return rc;
    if (n && d_dx && (rc = check_matrix(c, "d_dx", d_dx, lddx, dim, dtype))) return rc;
    if (d_dweight && (rc = check_matrix(c, "d_dweight", d_dweight, lddw, dim, dtype))) return rc;
    OnDevice dev(sage_ctx_device(c));
    if (!dev.ok) return sage_ctx_fail(c, SAGE_E_HIP, "the context's device cannot be made current");
    const hipStream_t st = (hipStream_t)stream;
    const int bf16 = dtype == SAGE_BF16;
    if (n == 0) {
        if (d_dweight) k_vs_zero<<<cdiv(vocab * dim, 256), 256, 0, st>>>(d_dweight, lddw, (int32_t)vocab, dim, bf16, d_dbias);
        return launched(c, "sage_token_logprobs_backward_device");
    }
    const BwdPlan p = plan_bwd(s, d_workspace);
    if ((rc = check_workspace(c, d_workspace, workspace_bytes, p.bytes))) return rc;
    const VsSrc w{d_weight, ldw, (int32_t)vocab, dim, bf16}, x{d_x, ldx, (int32_t)n, dim, bf16};
    VsPack of_w = pack_of(w, p.wS, d_dx ? p.wT : nullptr, s.vp);
    of_w.info = p.info; of_w.bias = d_bias;
    VsPack of_x = pack_of(x, p.xS, d_dweight ? p.xT : nullptr, p.np);
    of_x.tokens = p.tokens; of_x.lse = d_lse; of_x.entropy = d_entropy; of_x.g = d_grad_logprob; of_x.h = d_grad_entropy; of_x.targets = d_targets;
    of_x.vocab = (int32_t)vocab;
    pack<false>(s, of_w, of_x, st);
    const bool entropy = d_grad_entropy != nullptr;
    VsBwd b{};
    b.info = p.info; b.tokens = p.tokens; b.has_bias = d_bias != nullptr; b.vocab = (int32_t)vocab;
    VsSum sum_x{}, sum_w{};
    uint32_t groups_x = 0, groups_w = 0;
    {                                                            // over tokens first: dw takes from it what the targets' own weights are
        b.stayS = p.xS; b.flowS = p.wS; b.flowT = d_dx ? p.wT : p.wS;            // (without dx the second half of a stage is not looked at)
        b.n_tiles = (int32_t)p.tiles_x; b.splits = p.splits_x; b.groups = (int32_t)(s.vp / 32); b.stay_pad = p.np;
        b.part = d_dx ? p.part_x : nullptr; b.rest = p.rest; b.target_e = p.target_e;
        const uint32_t grid = cdiv(p.tiles_x, 4) * p.splits_x;
#define VS_F(KS, PL)                                                                            \
    if constexpr (vs_bwd_wide(KS, vs_bwd_blocks(KS, PL, false)))                                \
        if (!d_dx) { vs_bwd_kernel<KS, PL, false, false, false><<<grid, 256, 0, st>>>(b); break; } \
    if (entropy) vs_bwd_kernel<KS, PL, false, true><<<grid, 256, 0, st>>>(b); else vs_bwd_kernel<KS, PL, false, false><<<grid, 256, 0, st>>>(b)
        VS_BY_WIDTH(s.ks, s.pl, VS_F);
#undef VS_F
        if (d_targets) k_vs_target<<<cdiv(n, 256), 256, 0, st>>>(of_x, p.rest, p.target_e, p.splits_x, p.np);
    }
    if (d_dx) {
        sum_x = VsSum{p.part_x, nullptr, (int32_t)n, dim, s.ks * 32, p.splits_x, p.np, p.tokens, entropy, w, d_dx, lddx, bf16, nullptr};
        groups_x = cdiv(n * dim, 256);
    }
    if (d_dweight) {
        b.stayS = p.wS; b.flowS = p.xS; b.flowT = p.xT;
        b.n_tiles = (int32_t)p.tiles_w; b.splits = p.splits_w; b.groups = (int32_t)(p.np / 32); b.stay_pad = s.vp;
        b.want_db = d_dbias != nullptr; b.bias_part = p.bias_part; b.part = p.part_w;
        if (p.splits_w == 1) { b.out = d_dweight; b.ldo = lddw; b.rows = (int32_t)vocab; b.dim = dim; b.db = d_dbias; }
        const uint32_t grid = cdiv(p.tiles_w, 4) * p.splits_w;
#define VS_F(KS, PL) if (entropy) vs_bwd_kernel<KS, PL, true, true><<<grid, 256, 0, st>>>(b); else vs_bwd_kernel<KS, PL, true, false><<<grid, 256, 0, st>>>(b)
        VS_BY_WIDTH(s.ks, s.pl, VS_F);
#undef VS_F
        if (p.splits_w > 1) {
            sum_w = VsSum{p.part_w, p.bias_part, (int32_t)vocab, dim, s.ks * 32, p.splits_w, s.vp, nullptr, 0, w, d_dweight, lddw, bf16, d_dbias};
            groups_w = cdiv(vocab * dim, 256);
        }
    }
    if (groups_x + groups_w) k_vs_sum<<<groups_x + groups_w, 256, 0, st>>>(sum_x, sum_w, groups_x);
    return launched(c, "sage_token_logprobs_backward_device");
}

static int64_t clip_block(int64_t elements) { return elements <= (1 << 22) ? CLIP_SMALL : CLIP_BLOCK; }

static int64_t clip_table(ClipTable& t, int64_t n_tensors, const void* const* d_grads, void* const* d_out, const int64_t* sizes,
                          const int32_t* dtypes, int64_t block, int64_t i) {
    t.n = 0; t.first[0] = 0; t.block = (int32_t)block;
    for (; i < n_tensors && t.n < CLIP_TENSORS; ++i) {
        if (sizes[i] == 0) continue;
        t.in[t.n] = d_grads[i]; t.out[t.n] = d_out[i];
        t.size[t.n] = dtypes[i] == SAGE_BF16 ? -sizes[i] : sizes[i];
        t.first[t.n + 1] = t.first[t.n] + cdiv(sizes[i], block);
        ++t.n;
    }
    return i;
}

int64_t sage_clip_grad_norm_workspace(sage_ctx* c, int64_t n_tensors, const int64_t* sizes) {
    if (!c) return SAGE_E_ARG;
    if (n_tensors < 0 || (n_tensors && !sizes)) return sage_ctx_fail(c, SAGE_E_ARG, "need n_tensors >= 0 and their sizes");
    int64_t blocks = 0, elements = 0;
    for (int64_t i = 0; i < n_tensors; ++i) {
        if (sizes[i] < 0) return sage_ctx_fail(c, SAGE_E_ARG, "a tensor has a negative size");
        if (sizes[i] > (int64_t)1 << 44 || (elements += sizes[i]) > (int64_t)1 << 44) return sage_ctx_fail(c, SAGE_E_LIMIT, "more than 2^44 elements are not supported");
    }
    const int64_t block = clip_block(elements);
    for (int64_t i = 0; i < n_tensors; ++i) blocks += (sizes[i] + block - 1) / block;
    if (blocks > 1 << 30) return sage_ctx_fail(c, SAGE_E_LIMIT, "more than 2^30 tensors and blocks of tensors are not supported");
    return up(blocks * 8, VS_ALIGN) + (int64_t)VS_ALIGN;
}

int sage_clip_grad_norm_device(sage_ctx* c, int64_t n_tensors, const void* const* d_grads, void* const* d_out, const int64_t* sizes,
                               const int32_t* dtypes, double max_norm, float* d_norm, void* d_workspace, int64_t workspace_bytes,
                               void* stream) {
    if (!c) return SAGE_E_ARG;
    const int64_t need = sage_clip_grad_norm_workspace(c, n_tensors, sizes);
    if (need < 0) return (int)need;
    if (!d_norm) return sage_ctx_fail(c, SAGE_E_ARG, "d_norm is null");
    if (!(max_norm >= 0.0) || std::isinf(max_norm)) return sage_ctx_fail(c, SAGE_E_ARG, "max_norm must be finite and not negative");
    if (n_tensors && (!d_grads || !d_out || !dtypes)) return sage_ctx_fail(c, SAGE_E_ARG, "need the tensors' addresses and types");
    int rc;
    if ((rc = check_workspace(c, d_workspace, workspace_bytes, need))) return rc;
    try {
        std::vector<std::pair<uintptr_t, int64_t>> written;      // address, bytes
        written.reserve((size_t)n_tensors);
        for (int64_t i = 0; i < n_tensors; ++i) {
            if (dtypes[i] != SAGE_F32 && dtypes[i] != SAGE_BF16) return sage_ctx_fail(c, SAGE_E_ARG, "a tensor's type must be SAGE_F32 or SAGE_BF16");
            if (sizes[i] == 0) continue;
            const int w = dtypes[i] == SAGE_BF16 ? 2 : 4;
            if (!d_grads[i] || !d_out[i]) return sage_ctx_fail(c, SAGE_E_ARG, "a tensor's address is null");
            if ((uintptr_t)d_grads[i] % w || (uintptr_t)d_out[i] % w) return sage_ctx_fail(c, SAGE_E_ARG, "a tensor is not aligned to its elements");
            written.emplace_back((uintptr_t)d_out[i], sizes[i] * w);
        }
        std::sort(written.begin(), written.end());
        for (size_t i = 1; i < written.size(); ++i)
            if (written[i - 1].first + (uintptr_t)written[i - 1].second > written[i].first)
                return sage_ctx_fail(c, SAGE_E_ARG, "two of the written tensors overlap");
        for (int64_t i = 0; i < n_tensors; ++i) {                // a gradient may be written in place, and no other way over one
            if (sizes[i] == 0) continue;
            const uintptr_t lo = (uintptr_t)d_grads[i], hi = lo + (uintptr_t)sizes[i] * (dtypes[i] == SAGE_BF16 ? 2 : 4);
            auto it = std::lower_bound(written.begin(), written.end(), std::make_pair(lo, (int64_t)0));
            if (it != written.begin() && std::prev(it)->first + (uintptr_t)std::prev(it)->second > lo) --it;
            for (; it != written.end() && it->first < hi; ++it)
                if (it->first + (uintptr_t)it->second > lo && !((uintptr_t)d_out[i] == lo && it->first == lo))
                    return sage_ctx_fail(c, SAGE_E_ARG, "a written tensor overlaps a gradient other than its own");
        }
    } catch (...) {
        return sage_ctx_fail(c, SAGE_E_HIP, "out of host memory");
    }
    OnDevice dev(sage_ctx_device(c));
    if (!dev.ok) return sage_ctx_fail(c, SAGE_E_HIP, "the context's device cannot be made current");
    const hipStream_t st = (hipStream_t)stream;
    double* part = (double*)d_workspace;
    ClipFactor* factor = (ClipFactor*)((char*)d_workspace + need - VS_ALIGN);
    ClipTable t;
    int64_t elements = 0;
    for (int64_t i = 0; i < n_tensors; ++i) elements += sizes[i];
    if (elements <= CLIP_ONE && n_tensors <= CLIP_TENSORS) {
        clip_table(t, n_tensors, d_grads, d_out, sizes, dtypes, CLIP_PIECE, 0);
        k_clip_one<<<1, 1024, 0, st>>>(t, max_norm, d_norm);
        return launched(c, "sage_clip_grad_norm_device");
    }
    const int64_t block = clip_block(elements);
    uint32_t total = 0;
    for (int64_t i = 0; i < n_tensors;) {
        i = clip_table(t, n_tensors, d_grads, d_out, sizes, dtypes, block, i);
        t.block0 = total;
        if (!t.n) break;
        k_clip_squares<<<t.first[t.n], 256, 0, st>>>(t, part);
        total += t.first[t.n];
    }
    k_clip_norm<<<1, 1024, 0, st>>>(part, total, max_norm, d_norm, factor);
    for (int64_t end = n_tensors, i; end > 0; end = i) {         // the last tables first
        int full = 0;
        for (i = end; i > 0 && full < CLIP_TENSORS; --i) full += sizes[i - 1] > 0;
        clip_table(t, end, d_grads, d_out, sizes, dtypes, block, i);
        if (t.n) k_clip_scale<<<t.first[t.n], 256, 0, st>>>(t, factor);
    }
    return launched(c, "sage_clip_grad_norm_device");
}

}  // extern "C"
