// Attention of new tokens over a paged cache: ragged chunks of prompts, drafted tokens, single tokens.
//
// Token i of a sequence's n new ones, its length L with them, sits at position p = L - n + i and sees the keys
// max(0, p - W) .. p: o = softmax(scale q K^T) V and lse = log sum e^(scale q k). The rows of a tile (tokens x
// query heads of one key-value head) sweep their keys once with a running maximum and sum; paged_line.h says how
// the tiles are shared out and cut.
//
// Times are a call's among others; the kernels' medians in a trace of a process's first thirteen are in brackets (the products
// run slower then: the document's kernel goes from 1340 us down to 1030 over thirty passes). Chunks are bound by the
// products: 2048 tokens of 32 heads of 128 over 8 against 32768 keys take 1071-1081 us (1195 and the join's 22), 985-991
// TFLOP/s; nine prompts of up to 1400 tokens 295 us (352 and 24), 690, since each piece of a tile costs 10 us to begin
// and end. Single tokens are bound by memory: 64 of up to 8192 keys 287 us (280 and 6), 5.5 TB/s. Four short ones take 23 us
// (18.4 and 4.5), of which the plan is 4, the way to the first keys 5, 2.5 a block of 32 keys.
#include <algorithm>
#include <string>

#include "attention_kernels.h"
#include "dm_common.h"
#include "mfma.h"
#include "paged_line.h"

namespace dm {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ int32_t uni(int32_t x) { return __builtin_amdgcn_readfirstlane(x); }

// The rows of the tokens that belong to no sequence (all of them where the offsets do not go up): zeros, and
// a log-sum-exp of -inf.
template <int DT>
__device__ __forceinline__ void fill_outside(const PagedArgs &a, bool valid) {
    if (valid && !a.cu) return;
    const int32_t c0 = valid ? a.cu[0] : a.N, c1 = valid ? a.cu[a.S] : a.N;
    for (int32_t t = blockIdx.x; t < a.N; t += gridDim.x) {
        if (t >= c0 && t < c1) continue;
        for (int i = threadIdx.x; i < a.hq * a.d; i += blockDim.x) st<DT>(a.o, (int64_t)t * a.hq * a.d + i, 0.f);
        if (a.lse)
            for (int i = threadIdx.x; i < a.hq; i += blockDim.x) a.lse[(int64_t)t * a.hq + i] = -INFINITY;
    }
}

// The keys that a lane's row (r = lane % 32 of the piece, from `first` on) sees of the piece, and those that all of
// the wavefront's rows see.
struct RowKeys {
    int32_t lo, hi, flo, fhi;
    bool on;
    int32_t tok, head;
};
__device__ __forceinline__ RowKeys row_keys(const PagedArgs &a, const PagedPiece &x, int first) {
    RowKeys k;
    const int r = first + (threadIdx.x & 31);
    k.on = r < x.rows;
    const int32_t i = k.on ? r / x.per : 0, h = k.on ? r - i * x.per : 0;
    k.tok = x.tok + i, k.head = x.head + h;
    const int32_t pos = x.pos + i;
    k.lo = max(x.s0, a.left >= 0 ? pos - a.left : 0);
    k.hi = k.on ? min(x.s1, pos + 1) : 0;
    int32_t flo = k.on ? k.lo : INT32_MIN, fhi = k.on ? k.hi : INT32_MAX;
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
        flo = max(flo, __shfl_xor(flo, o, 64));
        fhi = min(fhi, __shfl_xor(fhi, o, 64));
    }
    k.flo = uni(flo), k.fhi = uni(fhi);
    return k;
}

__device__ __forceinline__ float lse_of(float m, float l) {
    return l == 0.f ? -INFINITY : (float)(((double)m + (double)log2f(l)) * 0.6931471805599453);
}

// ------------------------------------------------------------------------------------------
// The simple form: every type, head width, page size and stride
// ------------------------------------------------------------------------------------------
//
// A wavefront takes 32 rows and 32 keys at a time, both products on the f32 matrix cores: S^T = K q^T, whose
// output layout is the operand that O^T += V^T P^T takes. Keys and values go through one LDS tile of f32, DP columns
// wide (the head width and zeros behind it). 210 tokens of 4 heads of 64 in f32 against 300 keys each: 28 us and 5 of
// join, bound by latency. 1024 tokens of 32 heads over 8 against 5120 keys: f32 of 128 1218 us (63 TFLOP/s), 16-bit
// widths between the fast ones 2340 to 2410; 64 single tokens of 4352 keys f32 603 us, 96 wide in bf16 1468.

// VEC elements from p on.
template <int DT, int VEC>
__device__ __forceinline__ float4 load_some(const char *p) {
    if constexpr (VEC == 1) {
        return make_float4(ld<DT>(p, 0), 0.f, 0.f, 0.f);
    } else if constexpr (DT == DM_F32) {
        return *(const float4 *)p;
    } else {
        const uint2 w = *(const uint2 *)p;
        return make_float4(unpack_lo<DT>(w.x), unpack_hi<DT>(w.x), unpack_lo<DT>(w.y), unpack_hi<DT>(w.y));
    }
}

template <int DT, int DP, int VEC>
__global__ __launch_bounds__(256) void paged_simple(PagedArgs a, PagedLine l, const void *__restrict__ q,
                                                    const void *__restrict__ k, const void *__restrict__ v) {
    // (at DP = 256 the outputs and queries leave no registers for keys ahead)
    constexpr int TS = DP + 4, CPR = DP / VEC, NLD = CPR / 2, DTN = DP / 32, HALF = DP / 2, SIZE = DT == DM_F32 ? 4 : 2;
    constexpr bool AHEAD = DP <= 128;
    __shared__ PlanSmem<256, 1> plan;
    __shared__ __align__(16) float tiles[4][32 * TS];
    const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6), col = lane & 31, half = lane >> 5;
    const int32_t worker = blockIdx.x * 4 + wave;
    PagedWalk walk;
    const PagedLine lines[1] = {l};
    PagedShare shares[1];
    fill_outside<DT>(a, plan_lines(a, lines, plan, shares));
    const PagedShare &sh = shares[0];
    int64_t p = sh.total > 0 && worker < sh.workers ? sh.at(worker) : -1;
    plan_find<0>(a, lines, plan, sh, p, &walk);
    if (lane == 0 && worker < l.workers) l.jobs[worker].rows = 0;
    if (p < 0) return;
    const int64_t end = sh.at(worker + 1);
    float *tile = tiles[wave];
    const float qscale = a.scale * kLog2e;
    while (p < end) {
        int64_t next;
        int32_t last;
        const PagedPiece x = piece_of(a, l, walk, sh, worker, p, end, &next, &last);
        if (last >= 0 && lane == 0) l.jobs[worker] = PagedJob{x.tok, x.head, x.per, x.rows, x.first, last};
        const RowKeys rk = row_keys(a, x, 0);
        // (no load stands under a condition, which would have each waited for by itself: what is not there is read
        // somewhere else and cleared)
        float qf[HALF];
        {
            const int64_t row = (int64_t)rk.tok * a.qt + rk.head * a.qh;
#pragma unroll
            for (int e = 0; e < HALF; e++) qf[e] = ld<DT>(q, row + min(half * HALF + e, a.d - 1));
#pragma unroll
            for (int e = 0; e < HALF; e++) qf[e] = rk.on && half * HALF + e < a.d ? qf[e] : 0.f;
        }
        f32x16_t acc[DTN];
#pragma unroll
        for (int t = 0; t < DTN; t++) acc[t] = zero16();
        float m = -INFINITY, sum = 0.f;
        const int32_t *entries = a.table + x.s * a.max_pages;
        bool bad = false;
        int64_t ko, vo;  // this lane's key's rows in the pools, -1 for none
        auto places = [&](int32_t j0) __attribute__((always_inline)) {
            const int32_t key = min(j0 + col, max(x.s1 - 1, 0));
            const int64_t e = key / a.page_size, r = key - e * a.page_size, pg = entries[e];
            const bool is = j0 + col < x.s1 && pg >= 0 && pg < a.num_pages;
            ko = is ? pg * a.kb + r * a.kt + x.kh * a.kh : -1;
            vo = is ? pg * a.vb + r * a.vt + x.kh * a.vh : -1;
        };
        float4 kreg[NLD], vreg[NLD];
        auto load = [&](const void *pool, int64_t at, float4 (&y)[NLD]) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < NLD; u++) {
                const int i = u * 64 + lane, r = i / CPR, e = i % CPR * VEC;
                const int64_t off = __shfl((long long)at, r, 64);
                const bool is = off >= 0 && e < a.d;
                y[u] = load_some<DT, VEC>(is ? (const char *)pool + (off + e) * SIZE : (const char *)q);
                if (!is) y[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
        };
        auto put = [&](const float4 (&y)[NLD]) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < NLD; u++) {
                const int i = u * 64 + lane, r = i / CPR, e = i % CPR * VEC;
                if constexpr (VEC == 4)
                    *(float4 *)(tile + r * TS + e) = y[u];
                else
                    tile[r * TS + e] = y[u].x;
            }
        };
        auto take = [&](float4 &y, bool cut) __attribute__((always_inline)) {
            float *c = (float *)&y;
#pragma unroll
            for (int e = 0; e < VEC; e++)  // (a hidden key's weight is 0, and 0 times what is not finite is NaN)
                if (cut && !(fabsf(c[e]) < INFINITY)) c[e] = 0.f, bad = true;
        };
        auto copy = [&](const void *pool, int64_t at, bool cut) __attribute__((always_inline)) {  // by way of few registers
#pragma unroll 8
            for (int u = 0; u < NLD; u++) {
                const int i = u * 64 + lane, r = i / CPR, e = i % CPR * VEC;
                const int64_t off = __shfl((long long)at, r, 64);
                const bool is = off >= 0 && e < a.d;
                float4 y = load_some<DT, VEC>(is ? (const char *)pool + (off + e) * SIZE : (const char *)q);
                if (!is) y = make_float4(0.f, 0.f, 0.f, 0.f);
                take(y, cut);
                if constexpr (VEC == 4)
                    *(float4 *)(tile + r * TS + e) = y;
                else
                    tile[r * TS + e] = y.x;
            }
        };
        if (x.s0 < x.s1) {
            places(x.s0);
            if constexpr (AHEAD) load(k, ko, kreg);
        }
        for (int32_t j0 = x.s0; j0 < x.s1; j0 += 32) {
            const bool cut = j0 < rk.flo || j0 + 32 > rk.fhi;
            if constexpr (AHEAD) {
                put(kreg);
                load(v, vo, vreg);
            } else {
                copy(k, ko, false);
            }
            __builtin_amdgcn_wave_barrier();  // (a wavefront's LDS accesses complete in order)
            f32x16_t sc = zero16();
#pragma unroll
            for (int e = 0; e < HALF; e += 4) {
                const float4 y = *(const float4 *)(tile + col * TS + half * HALF + e);
                sc = mfma2(y.x, qf[e], sc);
                sc = mfma2(y.y, qf[e + 1], sc);
                sc = mfma2(y.z, qf[e + 2], sc);
                sc = mfma2(y.w, qf[e + 3], sc);
            }
            __builtin_amdgcn_wave_barrier();
            if (AHEAD && j0 + 32 < x.s1) {
                places(j0 + 32);
                load(k, ko, kreg);
            }
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int32_t key = j0 + crow(i, lane);
                sc[i] = key >= rk.lo && key < rk.hi ? sc[i] * qscale : -INFINITY;
                mx = fmaxf(mx, sc[i]);
            }
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            const bool grow = mx > m + 8.f;
            if (__any(grow)) {
                const float mn = grow ? mx : m, alpha = mn == -INFINITY ? 1.f : fast_exp2(m - mn);
                m = mn;
                sum *= alpha;
#pragma unroll
                for (int t = 0; t < DTN; t++)
#pragma unroll
                    for (int i = 0; i < 16; i++) acc[t][i] *= alpha;
            }
            const float ref = m == -INFINITY ? 0.f : m;
            float ps = 0.f;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                sc[i] = fast_exp2(sc[i] - ref);
                ps += sc[i];
            }
            sum += ps;
            if constexpr (AHEAD) {
#pragma unroll
                for (int u = 0; u < NLD; u++) take(vreg[u], cut);
                put(vreg);
            } else {
                copy(v, vo, cut);
            }
            __builtin_amdgcn_wave_barrier();
            // (a step's products first: with an addition a key to the sum so far, long sums of like terms lose bits)
#pragma unroll
            for (int t = 0; t < DTN; t++) {
                f32x16_t step = zero16();
#pragma unroll
                for (int i = 0; i < 16; i++) step = mfma2(tile[crow(i, lane) * TS + t * 32 + col], sc[i], step);
                acc[t] += step;
            }
            __builtin_amdgcn_wave_barrier();
            if (!AHEAD && j0 + 32 < x.s1) places(j0 + 32);
        }
        if (__any(bad)) {  // what was taken out of V, for the rows that see it
            for (int32_t j = x.s0; j < x.s1; j++) {
                const int32_t j0 = x.s0 + (j - x.s0) / 32 * 32;
                if (!(j0 < rk.flo || j0 + 32 > rk.fhi) || j < rk.lo || j >= rk.hi) continue;
                const int64_t e = j / a.page_size, pg = entries[e];
                if (pg < 0 || pg >= a.num_pages) continue;
                const int64_t row = pg * a.vb + (j - e * a.page_size) * a.vt + x.kh * a.vh;
#pragma unroll
                for (int t = 0; t < DTN; t++)
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const int c = t * 32 + crow(i, lane);
                        const float y = c < a.d ? ld<DT>(v, row + c) : 0.f;
                        if (!(fabsf(y) < INFINITY)) acc[t][i] += y;
                    }
            }
        }
        const float total = sum + __shfl_xor(sum, 32, 64);
        const float f = !x.whole ? 1.f : (total == 0.f ? 0.f : 1.f / total);  // (NaN is not 0)
        // the lanes along the rows, through LDS
#pragma unroll
        for (int t = 0; t < DTN; t++)
#pragma unroll
            for (int g = 0; g < 4; g++)
                *(float4 *)(tile + col * TS + t * 32 + g * 8 + half * 4) =
                    make_float4(acc[t][g * 4] * f, acc[t][g * 4 + 1] * f, acc[t][g * 4 + 2] * f, acc[t][g * 4 + 3] * f);
        __builtin_amdgcn_wave_barrier();
        const int64_t place = (int64_t)x.slot * l.pitch;
        if (half == 0 && rk.on) {
            if (!x.whole)
                l.ml[place + col] = make_float2(m, total);
            else if (a.lse)
                a.lse[(int64_t)rk.tok * a.hq + rk.head] = lse_of(m, total);
        }
        constexpr int LPR = DP / 4, RPL = 64 / LPR;  // lanes a row, rows at a time
        const int64_t mine = (int64_t)rk.tok * a.hq + rk.head;
        for (int r = 0; r < x.rows; r += RPL) {
            const int y = r + lane / LPR, c = lane % LPR * 4;
            const int64_t to = __shfl((long long)mine, min(y, 31), 64);
            const float4 o = *(const float4 *)(tile + min(y, 31) * TS + c);
            if (y >= x.rows) continue;
            const float f4[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (c + e >= a.d) continue;
                if (x.whole)
                    st<DT>(a.o, to * a.d + c + e, f4[e]);
                else
                    l.o[(place + y) * a.d + c + e] = f4[e];
            }
        }
        __builtin_amdgcn_wave_barrier();
        p = next;
        if (p >= end || !walk_on(a, l, walk, next)) break;
    }
}

// ------------------------------------------------------------------------------------------
// The 16-bit kernels (D = 64, 128 or 256, any page size)
// ------------------------------------------------------------------------------------------
//
// Both products run on MFMA: S^T = K q^T (keys x 32 rows) and O^T += V^T P^T, S^T's output layout being P^T's
// operand; the weights are rounded to the inputs' type for the second product (half a step a weight, as in the other
// attention kernels), scores, maxima, sums and outputs stay in f32.
//
// NARROW tiles, of up to 32 rows: a wavefront is a worker and sweeps its keys in blocks of 32 through its own LDS
// tiles. WIDE tiles, of up to 256 rows (128 at D = 256): a workgroup is a worker, its wavefronts have 32 rows each
// and sweep the same keys in tiles of 64; wavefronts w and w + 4 of a SIMD run half a step apart, so that one's
// products and the other's softmax run side by side. A sequence's rows lie in wide tiles where they are more than
// kNarrowRows.
//
// Keys are read by their rows: a key's place in the pool, in 16-byte units, is looked up well ahead of its load (64 keys
// ahead in registers; wide: 8 tiles ahead in an LDS ring), so any page size costs the same. A key of no
// page, or behind the piece, is loaded from the pool's start and zeroed on its way into LDS.

// Sequences whose rows one narrow tile holds lie in narrow tiles, larger ones in wide tiles, whose keys are read once for all
// of their rows. 32 sequences of 36 to 48 rows each, 4096 keys, in wide and in two narrow tiles: widths of 64 (2 key
// heads) 45 and 58 us, 128 (8) 165 and 230, 128 (2) 62 and 95, 256 (2) 78 and 123; 8 of them of 4000 keys 35 and 39,
// 62 and 95, 46 and 55, 50 and 59. Batches of both sizes (8 to 64 sequences of 8 to 52 rows) pay both lines' starts,
// -20% to +35%: with 48 here the geometric mean of 56 of them is the same, with 64 3% less, and the equal ones' 9 and 17% more.
constexpr int kNarrowRows = 32;
// Calls of at most so many rows a key head altogether get no wide line, only narrow tiles (two at most of a sequence): without
// a line to plan and its workgroups a call of 33 to 64 rows takes 22-32 us where both lines take 28-40 (1 to 16
// sequences of 1000 to 8000 keys, 2 key heads of 64 or 128); one sequence of 30000 keys 46 and 41. At 256, whose narrow
// line has half as many workers: 39-45 and 40-44, of 30000 keys 65 and 48.
static int64_t lone_rows(int64_t d) { return d == 256 ? kNarrowRows : 2 * kNarrowRows; }
// Sequences whose narrow sweep leaves its scores for the keys' weights: a row's take 4 bytes a key to write and to read,
// where the keys' second pass reads 2 D a head. With 32 heads of 128 and 4096 keys, kept and not, 64 sequences of
// 4 rows a head 201 and 257 us; 32 of 8 rows 194 and 195, of 12 211 and 205, of 16 228 and 207, of 32 296 and 212.
constexpr int kScoreRows = 8;
static_assert(kScoreRows <= 16, "a larger sequence's first tile has more rows");
// The reference that weights are taken against lies kLift (log2 units) below the row's maximum when it moves, and moves
// when the maximum is kTop or more above it. f16 has no weight below 2^-25, and 131072 keys of such weights beside one of 1
// are 0.3% of their sum: its weights reach up to 2^11, so that what is lost is below 2^-32 of the row's largest (the 2^5 from
// there to its largest number are left to the scores' own rounding, half a step of 4 at 2^26).
template <int DT>
constexpr float kLift = DT == DM_F16 ? 7.f : 0.f;
template <int DT>
constexpr float kTop = DT == DM_F16 ? 11.f : 8.f;
template <int D>
constexpr int paged_waves() { return D == 256 ? 4 : 8; }
constexpr uint32_t kNoKey = 0xffffffffu;

struct PoolMap {
    const char *k, *v;     // at the piece's key-value head
    const int32_t *table;  // the sequence's
    uint32_t page, row;    // 16-byte units of a page and of a row, keys' and values' alike
    uint32_t size, pages;
};
__device__ __forceinline__ PoolMap pool_of(const PagedArgs &a, const PagedPiece &x, const void *k, const void *v) {
    PoolMap m;
    m.k = (const char *)k + (int64_t)x.kh * a.kh * 2;
    m.v = (const char *)v + (int64_t)x.kh * a.vh * 2;
    m.table = a.table + x.s * a.max_pages;
    m.page = (uint32_t)(a.kb / 8), m.row = (uint32_t)(a.kt / 8);
    m.size = (uint32_t)a.page_size, m.pages = (uint32_t)a.num_pages;
    return m;
}
// Key j's entry in the table, and its place from that. (Of keys behind a piece the last one's is read: a load under a
// condition would be waited for at once.)
__device__ __forceinline__ int32_t entry_of(const PoolMap &m, int32_t j) { return m.table[(uint32_t)j / m.size]; }
__device__ __forceinline__ uint32_t place_of(const PoolMap &m, int32_t j, int32_t entry) {
    return (uint32_t)entry < m.pages ? (uint32_t)entry * m.page + ((uint32_t)j % m.size) * m.row : kNoKey;
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint4 load_nt(const char *p) {
    const u32x4 x = __builtin_nontemporal_load((const u32x4 *)p);
    return make_uint4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ uint4 only(bool ok, const uint4 &x) {
    return make_uint4(ok ? x.x : 0u, ok ? x.y : 0u, ok ? x.z : 0u, ok ? x.w : 0u);
}

// 32 rows' queries: loaded along the rows (a load then touches few cache lines), sorted into operands through the
// wavefront's own 32 rows of LDS. slots: in the order of row_frag. Nothing is waited for before settle_q.
template <int D>
struct QueryRows {
    Frag8 f[D / 16];
};
template <int D>
__device__ __forceinline__ void load_q(const PagedArgs &a, const RowKeys &k, const void *q, QueryRows<D> &w) {
    constexpr int LPR = D / 8, RPL = 64 / LPR;  // lanes a row, rows a load
    const int lane = threadIdx.x & 63;
    const int64_t off = (int64_t)k.tok * a.qt + (int64_t)k.head * a.qh;  // (without a row: the piece's first)
#pragma unroll
    for (int u = 0; u < D / 16; u++) {
        const int x = u * RPL + lane / LPR;
        const int64_t at = __shfl((long long)off, x, 64);
        w.f[u].u = *(const uint4 *)((const uint16_t *)q + at + (lane % LPR) * 8);
    }
}
template <int D>
__device__ __forceinline__ void settle_q(const PagedArgs &a, uint16_t *rows, bool slots, QueryRows<D> &w) {
    constexpr int LPR = D / 8, RPL = 64 / LPR, KS = D + 8;
    const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
#pragma unroll
    for (int u = 0; u < D / 16; u++) *(uint4 *)(rows + (u * RPL + lane / LPR) * KS + (lane % LPR) * 8) = w.f[u].u;
    __builtin_amdgcn_wave_barrier();  // (a wavefront's LDS accesses complete in order)
    const uint16_t *mine = rows + col * KS;
    const uint32_t sign = a.scale < 0.f ? 0x80008000u : 0u;  // (the softmax takes a scale above 0)
#pragma unroll
    for (int s = 0; s < D / 16; s++) {
        uint4 x;
        if (slots) {
            const uint2 l = *(const uint2 *)(mine + s * 16 + half * 4), u = *(const uint2 *)(mine + s * 16 + 8 + half * 4);
            x = make_uint4(l.x, l.y, u.x, u.y);
        } else {
            x = *(const uint4 *)(mine + s * 16 + half * 8);
        }
        w.f[s].u = make_uint4(x.x ^ sign, x.y ^ sign, x.z ^ sign, x.w ^ sign);
    }
    __builtin_amdgcn_wave_barrier();
}

// The values that were taken out of V, added for the rows that see them: the keys of [j0, j1) again, one at a time.
template <int DT, int D>
__device__ __forceinline__ void add_back16(const PoolMap &m, int32_t j0, int32_t j1, const RowKeys &rk, f32x16_t (&acc)[D / 32]) {
    const int lane = threadIdx.x & 63;
    for (int32_t j = j0; j < j1; j++) {
        const uint32_t at = place_of(m, j, entry_of(m, j));
        if (at == kNoKey || j < rk.lo || j >= rk.hi) continue;
        const uint16_t *row = (const uint16_t *)(m.v + (uint64_t)at * 16);
#pragma unroll
        for (int dt = 0; dt < D / 32; dt++) {
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                uint32_t x = *(const uint32_t *)(row + dt * 32 + crow(i, lane));  // elements i and i + 1
                x &= not_finite<DT>(x);
                acc[dt][i] += unpack_lo<DT>(x);
                acc[dt][i + 1] += unpack_hi<DT>(x);
            }
            __builtin_amdgcn_sched_barrier(0);  // (with every load of a row up front the registers run out)
        }
    }
}

// A wavefront's 32 rows from `first` on: outputs and log-sum-exps of a whole tile, or its place in the workspace, the
// lanes along the rows through its own LDS (32 rows of D + 4 floats).
template <int DT, int D>
__device__ __forceinline__ void finish_rows(const PagedArgs &a, const PagedLine &l, const PagedPiece &x, const RowKeys &rk,
                                            int first, const f32x16_t (&acc)[D / 32], float m, float sum, float *rows) {
    constexpr int JS = D + 4, LPR = D / 4, RPL = 64 / LPR;
    const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5, n = min(32, x.rows - first);
    const float f = !x.whole ? 1.f : (sum == 0.f ? 0.f : 1.f / sum);  // (NaN is not 0)
#pragma unroll
    for (int dt = 0; dt < D / 32; dt++)
#pragma unroll
        for (int g = 0; g < 4; g++)
            *(float4 *)(rows + col * JS + dt * 32 + g * 8 + half * 4) =
                make_float4(acc[dt][g * 4] * f, acc[dt][g * 4 + 1] * f, acc[dt][g * 4 + 2] * f, acc[dt][g * 4 + 3] * f);
    __builtin_amdgcn_wave_barrier();
    const int64_t place = (int64_t)x.slot * l.pitch + first;
    if (half == 0 && rk.on) {
        if (!x.whole)
            l.ml[place + col] = make_float2(m, sum);
        else if (a.lse)
            a.lse[(int64_t)rk.tok * a.hq + rk.head] = lse_of(m, sum);
    }
    const int64_t mine = (int64_t)rk.tok * a.hq + rk.head;
    for (int r = 0; r < n; r += RPL) {
        const int y = r + lane / LPR, z = min(y, 31), c = lane % LPR * 4;
        const int64_t row = __shfl((long long)mine, z, 64);
        const float4 o = *(const float4 *)(rows + z * JS + c);
        if (y >= n) continue;
        if (x.whole)
            *(uint2 *)((uint16_t *)a.o + row * D + c) = make_uint2(pack2<DT>(o.x, o.y), pack2<DT>(o.z, o.w));
        else
            *(float4 *)(l.o + (place + y) * D + c) = o;
    }
    __builtin_amdgcn_wave_barrier();
}

template <int D>
struct NarrowTile {
    static constexpr int KS = D + 8, VS = D + 32;
    alignas(16) uint16_t k[32 * KS], v[32 * VS];
};
static_assert(sizeof(NarrowTile<64>) >= 32 * 68 * 4 && sizeof(NarrowTile<256>) >= 32 * 260 * 4,
              "a tile's results go through its place");

// SCORES: the rows' scores are kept, for the weights of the keys.
template <int DT, int D, bool SCORES>
__device__ __forceinline__ void paged_narrow(const PagedArgs &a, const PagedLine &l, const PagedPiece &x, const PoolMap &map,
                                             const void *q, NarrowTile<D> &t) {
    constexpr int KS = NarrowTile<D>::KS, VS = NarrowTile<D>::VS, KST = D / 16, DTN = D / 32;
    constexpr int LPR = D / 8, RPL = 64 / LPR, NLD = 32 / RPL;  // lanes a row, rows a load, loads
    const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
    const int32_t s0 = x.s0, s1 = x.s1;
    const float qscale = fabsf(a.scale) * kLog2e;
    // the entries and places of the 64 keys at hand, a lane each, and the entries of the 64 behind them
    const int32_t end = max(s1 - 1, 0);
    int32_t ahead = entry_of(map, min(s0 + lane, end));
    const RowKeys rk = row_keys(a, x, 0);
    QueryRows<D> qr;
    load_q<D>(a, rk, q, qr);
    auto place = [&](int32_t j) __attribute__((always_inline)) { return j < s1 ? place_of(map, j, ahead) : kNoKey; };
    uint32_t at = place(s0 + lane);
    ahead = entry_of(map, min(s0 + 64 + lane, end));
    __amdgpu_buffer_rsrc_t keep;
    const bool keeps = SCORES && uni(x.row0 == 0 && x.rows <= kScoreRows);
    if constexpr (SCORES)
        keep = make_rsrc(a.scores + (((int64_t)x.s * a.hkv + x.kh) * a.score_rows + x.row0) * a.cap,
                         (uint32_t)x.rows * (uint32_t)a.cap * 4);
    uint4 sk[NLD], sv[NLD];
    uint32_t have = 0;  // the loads of this lane that are keys'
    auto load = [&](int32_t n) __attribute__((always_inline)) {  // the n-th 32 keys
        have = 0;
#pragma unroll
        for (int u = 0; u < NLD; u++) {
            const uint32_t p = __shfl(at, (n & 1) * 32 + RPL * u + lane / LPR, 64);
            const bool ok = p != kNoKey;
            have |= (uint32_t)ok << u;
            const uint64_t off = (uint64_t)(ok ? p : 0u) * 16 + (lane % LPR) * 16;
            sk[u] = load_nt(map.k + off);
            sv[u] = load_nt(map.v + off);
        }
    };
    f32x16_t acc[DTN];
#pragma unroll
    for (int dt = 0; dt < DTN; dt++) acc[dt] = zero16();
    float m = -INFINITY, sum = 0.f;
    uint32_t bad = 0;
    const int32_t blocks = (s1 - s0 + 31) / 32;
    if (blocks > 0) {
        load(0);
        settle_q<D>(a, t.k, true, qr);
        for (int32_t n = 0; n < blocks; n++) {
            const int32_t j0 = s0 + n * 32;
            const bool cut = j0 < rk.flo || j0 + 32 > rk.fhi;
            if (!__all(have == (1u << NLD) - 1)) {
#pragma unroll
                for (int u = 0; u < NLD; u++) {
                    const bool ok = have >> u & 1;
                    sk[u] = only(ok, sk[u]), sv[u] = only(ok, sv[u]);
                }
            }
#pragma unroll
            for (int u = 0; u < NLD; u++) {
                const int r = RPL * u + lane / LPR, c = (lane % LPR) * 8;
                *(uint4 *)(t.k + r * KS + c) = sk[u];
                *(uint4 *)(t.v + r * VS + c) = sv[u];
            }
            if (cut) {  // (in LDS: the loads' registers are full)
#pragma unroll 1
                for (int u = 0; u < NLD; u++) {
                    uint4 *p = (uint4 *)(t.v + (RPL * u + lane / LPR) * VS + (lane % LPR) * 8), y = *p;
                    const uint32_t out = take_out<DT>(y);
                    if (out) *p = y;
                    bad |= out;
                }
            }
            if (n & 1) {
                at = place(j0 + 32 + lane);
                ahead = entry_of(map, min(j0 + 96 + lane, end));
            }
            load(n + 1);  // (past the last: the pool's start, unused)
            f32x16_t sc = zero16();
#pragma unroll
            for (int st = 0; st < KST; st++) sc = mfma32<DT>(row_frag(t.k, KS, 0, st * 16, lane), qr.f[st], sc);
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int32_t key = j0 + crow(i, lane);
                sc[i] = !cut || (key >= rk.lo && key < rk.hi) ? sc[i] * qscale : -INFINITY;
                mx = fmaxf(mx, sc[i]);
            }
            if (keeps) {
                // (a lane without a row, and a key behind the piece: past the buffer's end, so not stored)
                const uint32_t to = rk.on ? (uint32_t)(col * a.cap + j0 + half * 4) * 4 : kNoKey;
                if (j0 + 32 <= s1) {
#pragma unroll
                    for (int g = 0; g < 4; g++)
                        buf_store16(keep, rk.on ? to + g * 32 : kNoKey, sc[g * 4], sc[g * 4 + 1], sc[g * 4 + 2], sc[g * 4 + 3]);
                } else {
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        __builtin_amdgcn_raw_buffer_store_b32(
                            __float_as_uint(sc[i]), keep, rk.on && j0 + crow(i, lane) < s1 ? to + (i / 4 * 8 + i % 4) * 4 : kNoKey, 0, 0);
                }
            }
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            const bool grow = mx - m > kTop<DT>;  // false while both are -inf
            if (__any(grow)) {
                const float mn = grow ? mx - kLift<DT> : m, alpha = mn == -INFINITY ? 1.f : fast_exp2(m - mn);
                m = mn;
                sum *= alpha;
#pragma unroll
                for (int dt = 0; dt < DTN; dt++)
#pragma unroll
                    for (int i = 0; i < 16; i++) acc[dt][i] *= alpha;
            }
            const float ref = m == -INFINITY ? 0.f : m;
            float ps = 0.f;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                sc[i] = fast_exp2(sc[i] - ref);
                ps += sc[i];
            }
            sum += ps;
            const Frag8 p0 = c_frag<DT>(sc, 0), p1 = c_frag<DT>(sc, 1);
#pragma unroll
            for (int dt = 0; dt < DTN; dt++) {
                acc[dt] = mfma32<DT>(lds_tr_frag(t.v, VS, 0, dt * 32, lane), p0, acc[dt]);
                acc[dt] = mfma32<DT>(lds_tr_frag(t.v, VS, 16, dt * 32, lane), p1, acc[dt]);
            }
        }
    }
    if (__any(bad))
        for (int32_t j0 = s0; j0 < s1; j0 += 32)
            if (j0 < rk.flo || j0 + 32 > rk.fhi) add_back16<DT, D>(map, j0, min(j0 + 32, s1), rk, acc);
    finish_rows<DT, D>(a, l, x, rk, 0, acc, m, sum + __shfl_xor(sum, 32, 64), (float *)&t);
}

template <int D>
struct WideTiles {
    static constexpr int KS = D + 8, VS = D + 32, NW = paged_waves<D>();
    alignas(16) uint16_t k[2][64 * KS], v[2][64 * VS];
    uint32_t places[1024];  // of 16 tiles' keys, see `fill`
};
struct WideFlags {
    int32_t lo[8], hi[8], bad, missing;  // values that are not finite taken out; keys of no page
};

template <int DT, int D>
__device__ __forceinline__ void paged_wide(const PagedArgs &a, const PagedLine &l, const PagedPiece &x, const PoolMap &map,
                                           const void *q, WideTiles<D> &sm, WideFlags &flags, NarrowTile<D> *area) {
    constexpr int NW = paged_waves<D>(), NT = NW * 64, KS = WideTiles<D>::KS, VS = WideTiles<D>::VS;
    constexpr int CPR = D / 8, RSTEP = NT / CPR, NCH = 64 / RSTEP;  // pieces a row, rows at a time, pieces a thread
    constexpr int KST = D / 16, DTN = D / 32, AHEAD = 2, PK = 512 / NT;
    const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5, wave = uni(threadIdx.x >> 6);
    const bool first = NW == 4 || wave < 4;  // products first in each step
    const int32_t s0 = x.s0, s1 = x.s1, nt = (s1 - s0 + 63) / 64;
    int32_t entry[PK], entry1[PK];
    // the entries of 512 keys from `key` on, and the places that these say; behind the piece the last key's (masked, but
    // loaded), and the pool's start for a key of no page
    auto look_up = [&](int32_t key, int32_t (&entry)[PK]) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < PK; u++) entry[u] = entry_of(map, min(s0 + key + u * NT + (int32_t)threadIdx.x, s1 - 1));
    };
    auto fill = [&](int32_t key, const int32_t (&entry)[PK]) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < PK; u++) {
            const int32_t j = key + u * NT + (int32_t)threadIdx.x;
            const uint32_t at = place_of(map, min(s0 + j, s1 - 1), entry[u]);
            if (at == kNoKey) flags.missing = 1;
            sm.places[j & 1023] = at == kNoKey ? 0 : at;
        }
    };
    if (nt > 0) look_up(0, entry), look_up(512, entry1);
    const RowKeys rk = row_keys(a, x, wave * 32);
    QueryRows<D> qr;
    load_q<D>(a, rk, q, qr);
    // the keys that any of the wavefront's rows sees
    int32_t wlo = rk.on ? rk.lo : INT32_MAX, whi = rk.hi;
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
        wlo = min(wlo, __shfl_xor(wlo, o, 64));
        whi = max(whi, __shfl_xor(whi, o, 64));
    }
    wlo = uni(wlo), whi = uni(whi);
    __syncthreads();  // (the last piece's results have left LDS)
    if (lane == 0) flags.lo[wave] = rk.flo, flags.hi[wave] = rk.fhi;
    if (threadIdx.x == 0) flags.bad = flags.missing = 0;
    settle_q<D>(a, (uint16_t *)&area[wave], false, qr);
    __syncthreads();  // (the queries' way through LDS is what the places and tiles lie in)
    if (nt > 0) fill(0, entry), fill(512, entry1);
    int32_t tlo = INT32_MIN, thi = INT32_MAX;  // the keys that every row of the tile sees
#pragma unroll
    for (int w = 0; w < NW; w++) tlo = max(tlo, flags.lo[w]), thi = min(thi, flags.hi[w]);
    tlo = uni(tlo), thi = uni(thi);
    __syncthreads();
    bool missing = uni(flags.missing);
    // (a scale of 0 as the smallest: a masked score stays -inf, the others' weights are alike)
    const float c2 = a.scale == 0.f ? 1.2e-38f : fabsf(a.scale) * kLog2e;

    // staging: NCH pieces of a tile's K and of its V a thread; a tile's places are read from LDS a step before its
    // keys are loaded, and kept for its values
    const int row0 = threadIdx.x / CPR, lc = threadIdx.x % CPR;
    uint4 rk4[NCH], rv4[NCH];
    uint32_t ak[NCH], av[NCH];
    const char *kbase = map.k + lc * 16, *vbase = map.v + lc * 16;
    auto offsets = [&](int32_t j) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < NCH; u++) ak[u] = sm.places[(j * 64 + row0 + u * RSTEP) & 1023];
    };
    auto load_v = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < NCH; u++) rv4[u] = *(const uint4 *)(vbase + (uint64_t)av[u] * 16);
    };
    // the keys of tile j, then the places of the tile behind it
    auto load_k = [&](int32_t j) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < NCH; u++) rk4[u] = *(const uint4 *)(kbase + (uint64_t)ak[u] * 16);
#pragma unroll
        for (int u = 0; u < NCH; u++) av[u] = ak[u];
        offsets(j + 1);
    };
    auto zeros = [&](int32_t j, uint4 (&y)[NCH]) __attribute__((always_inline)) {  // keys of no page
#pragma unroll
        for (int u = 0; u < NCH; u++) {
            const int32_t key = min(s0 + j * 64 + row0 + u * RSTEP, s1 - 1);
            if (place_of(map, key, entry_of(map, key)) == kNoKey) y[u] = zero4();
        }
    };
    auto store_k = [&](int32_t j) __attribute__((always_inline)) {
        if (missing) zeros(j, rk4);
#pragma unroll
        for (int u = 0; u < NCH; u++) *(uint4 *)(sm.k[j & 1] + (row0 + u * RSTEP) * KS + lc * 8) = rk4[u];
    };
    auto store_v = [&](int32_t j) __attribute__((always_inline)) {
        const int32_t t = s0 + j * 64;
        if (missing) zeros(j, rv4);
        if (t < tlo || t + 64 > thi) {  // (a tile that some row does not see all of)
            uint32_t bad = 0;
#pragma unroll
            for (int u = 0; u < NCH; u++) bad |= take_out<DT>(rv4[u]);
            if (__any(bad) && lane == 0) flags.bad = 1;
        }
#pragma unroll
        for (int u = 0; u < NCH; u++) *(uint4 *)(sm.v[j & 1] + (row0 + u * RSTEP) * VS + lc * 8) = rv4[u];
    };
    auto sees = [&](int32_t j) __attribute__((always_inline)) {
        const int32_t j0 = s0 + j * 64;
        return j >= 0 && j < nt && j0 < whi && j0 + 64 > wlo;
    };
    f32x16_t acc[DTN], s[2];
    Frag8 pf[2][2];
    float m = -INFINITY, sum = 0.f;
#pragma unroll
    for (int dt = 0; dt < DTN; dt++) acc[dt] = zero16();
    // O^T of step j - 1 first, whose operands are dead when S^T's take their registers; each fragment is
    // read from LDS ahead of the products in front of it.
    auto products = [&](int32_t j) __attribute__((always_inline)) {
        const uint16_t *tk = sm.k[j & 1] + col * KS + half * 8, *tv = sm.v[(j - 1) & 1];
        Frag8 vf[2][DTN], kf[AHEAD + 1][2];
        auto read_v = [&](int g) __attribute__((always_inline)) {
#pragma unroll
            for (int dt = 0; dt < DTN; dt++) vf[g & 1][dt] = lds_tr_frag(tv, VS, g * 16, dt * 32, lane);
        };
        auto read_k = [&](int st) __attribute__((always_inline)) {
#pragma unroll
            for (int t = 0; t < 2; t++) kf[st % (AHEAD + 1)][t].u = *(const uint4 *)(tk + t * 32 * KS + st * 16);
        };
        __builtin_amdgcn_s_setprio(1);
        read_v(0);  // (of a step without a tile, too: whatever lies there, unused)
        if (sees(j - 1)) {
#pragma unroll
            for (int g = 0; g < 4; g++) {
                if (g < 3) read_v(g + 1);
#pragma unroll
                for (int dt = 0; dt < DTN; dt++) acc[dt] = mfma32<DT>(vf[g & 1][dt], pf[g >> 1][g & 1], acc[dt]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (sees(j)) {
#pragma unroll
            for (int st = 0; st < AHEAD; st++) read_k(st);
#pragma unroll
            for (int t = 0; t < 2; t++) s[t] = zero16();
#pragma unroll
            for (int st = 0; st < KST; st++) {
                if (st + AHEAD < KST) read_k(st + AHEAD);
#pragma unroll
                for (int t = 0; t < 2; t++) s[t] = mfma32<DT>(kf[st % (AHEAD + 1)][t], qr.f[st], s[t]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        __builtin_amdgcn_s_setprio(0);
    };
    auto softmax = [&](int32_t jj) __attribute__((always_inline)) {
        const int32_t j0 = s0 + jj * 64;
        if (j0 < rk.flo || j0 + 64 > rk.fhi) {
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int32_t j = j0 + t * 32 + crow(i, lane);
                    s[t][i] = ((j >= rk.lo) & (j < rk.hi)) ? s[t][i] : -INFINITY;
                }
        }
        float tmax = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int i = 0; i < 16; i++) tmax = fmaxf(tmax, s[t][i]);
        tmax = fmaxf(tmax, __shfl_xor(tmax, 32, 64));
        const float tmc = tmax * c2;
        const bool grow = tmc - m > kTop<DT>;  // false while both are -inf
        if (__any(grow)) {
            const float mnew = grow ? tmc - kLift<DT> : m, alpha = grow ? fast_exp2(m - mnew) : 1.f;  // 0 from -inf
            m = mnew;
            sum *= alpha;
#pragma unroll
            for (int dt = 0; dt < DTN; dt++)
#pragma unroll
                for (int i = 0; i < 16; i++) acc[dt][i] *= alpha;
        }
        const float mneg = m == -INFINITY ? 0.f : -m;
        float ps = 0.f;  // (the tile's weights first: one at a time, long sums of like ones come out short)
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int u = 0; u < 2; u++) {
                float e[8];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    e[i] = fast_exp2(fmaf(s[t][8 * u + i], c2, mneg));
                    ps += e[i];
                }
                pf[t][u].u = make_uint4(pack2<DT>(e[0], e[1]), pack2<DT>(e[2], e[3]), pack2<DT>(e[4], e[5]),
                                        pack2<DT>(e[6], e[7]));
            }
        sum += ps;
    };
    // Wavefronts 0-3 store K_{j+1} and V_j during their softmax of step j, wavefronts 4-7, half a step
    // later, K_{j+2} and V_{j+1}: each tile is whole before its first reader's step.
    const int32_t ahead = first ? 0 : 1;
    auto stage = [&](int32_t j) __attribute__((always_inline)) {
        store_k(j + 1 + ahead);
        store_v(j + ahead);
        load_v();
        load_k(j + 2 + ahead);
        // The ring's half of the tiles j - 8 .. j - 1, whose places all have read, goes to j + 8 .. j + 15: looked up
        // now and written two steps later, three steps before any of them is read.
        if (j > 0 && (j & 7) == 0) look_up(64 * (j + 8), entry);
        if (j > 2 && (j & 7) == 2) fill(64 * (j + 6), entry);
        if (j > 2 && (j & 7) == 4) missing = uni(flags.missing);
    };
    if (nt > 0) {
        offsets(0);
        load_k(0);
        load_v();
        store_k(0);
        load_k(1);
    }
    __syncthreads();
    if (!first) {
        if (nt > 0) stage(-1);
        __syncthreads();
    }
    for (int32_t j = 0; j <= nt; j++) {
        products(j);
        __syncthreads();
        if (sees(j)) softmax(j);
        if (j < nt) stage(j);
        __syncthreads();
    }
    if (first) __syncthreads();
    const bool rows = wave * 32 < x.rows;
    if (rows && flags.bad)
        for (int32_t j0 = s0; j0 < s1; j0 += 64)
            if (j0 < tlo || j0 + 64 > thi) add_back16<DT, D>(map, j0, min(j0 + 64, s1), rk, acc);
    __syncthreads();  // (every wavefront is past its last tile, and has read whether there was a bad one)
    if (rows) finish_rows<DT, D>(a, l, x, rk, wave * 32, acc, m, sum + __shfl_xor(sum, 32, 64), (float *)&area[wave]);
}

// Everything uniform in a wavefront that the loads' scalar bases come from.
__device__ __forceinline__ void settle_piece(PagedPiece &x) {
    x.tok = uni(x.tok), x.head = uni(x.head), x.rows = uni(x.rows), x.pos = uni(x.pos), x.kh = uni(x.kh), x.s = uni(x.s);
    x.row0 = uni(x.row0), x.s0 = uni(x.s0), x.s1 = uni(x.s1), x.slot = uni(x.slot), x.whole = uni(x.whole);
}

// A call whose sequences all have few rows: every wavefront a worker.
template <int DT, int D, bool SCORES>
__device__ __forceinline__ void narrow_share(const PagedArgs &a, const PagedLine &l, const PagedShare &sh, int32_t worker,
                                             PagedWalk &walk, int64_t p, const void *q, const void *k, const void *v,
                                             NarrowTile<D> &tile) {
    if ((threadIdx.x & 63) == 0 && worker < l.workers) l.jobs[worker].rows = 0;
    if (p < 0) return;
    const int64_t end = sh.at(worker + 1);
    for (;;) {
        int64_t next;
        int32_t last;
        PagedPiece x = piece_of(a, l, walk, sh, worker, p, end, &next, &last);
        settle_piece(x);
        if (last >= 0 && (threadIdx.x & 63) == 0) l.jobs[worker] = PagedJob{x.tok, x.head, x.per, x.rows, x.first, last};
        paged_narrow<DT, D, SCORES>(a, l, x, pool_of(a, x, k, v), q, tile);
        p = next;
        if (p >= end || !walk_on(a, l, walk, next)) return;
    }
}
template <int DT, int D, bool SCORES>
__global__ __launch_bounds__(256, (D == 256 ? 1 : 2)) void paged_narrow_kernel(PagedArgs a, PagedLine l, const void *__restrict__ q,
                                                                              const void *__restrict__ k,
                                                                              const void *__restrict__ v) {
    __shared__ union {
        PlanSmem<256, 1> plan;
        NarrowTile<D> tiles[4];
    } sm;
    const int wave = uni(threadIdx.x >> 6);
    const int32_t worker = blockIdx.x * 4 + wave;
    PagedWalk walk;
    const PagedLine lines[1] = {l};
    PagedShare sh[1];
    fill_outside<DT>(a, plan_lines(a, lines, sm.plan, sh));
    const int64_t p = sh[0].total > 0 && worker < sh[0].workers ? sh[0].at(worker) : -1;
    plan_find<0>(a, lines, sm.plan, sh[0], p, &walk);
    narrow_share<DT, D, SCORES>(a, l, sh[0], worker, walk, p, q, k, v, sm.tiles[wave]);
}

// Any call: the wide tiles' line, a workgroup a worker, and the narrow tiles', a wavefront a worker. Every other
// workgroup begins with its narrow share, so that reading and multiplying go on side by side.
template <int DT, int D, bool SCORES>
__global__ __launch_bounds__((64 * paged_waves<D>()), (D == 256 ? 1 : 2)) void paged_mixed_kernel(PagedArgs a, PagedLine wide, PagedLine narrow,
                                                                                   const void *__restrict__ q,
                                                                                   const void *__restrict__ k,
                                                                                   const void *__restrict__ v) {
    constexpr int NW = paged_waves<D>();
    __shared__ PlanSmem<64 * NW, 2> plan;
    __shared__ union {
        WideTiles<D> wide;
        NarrowTile<D> tiles[NW];
    } sm;
    __shared__ WideFlags flags;
    const int wave = uni(threadIdx.x >> 6);
    const PagedLine lines[2] = {wide, narrow};
    PagedShare shares[2];
    fill_outside<DT>(a, plan_lines(a, lines, plan, shares));
    for (int turn = 0; turn < 2; turn++) {
        PagedWalk walk;
        if ((turn ^ (int)(blockIdx.x >> 3)) & 1) {
            const PagedShare &sh = shares[1];
            const int32_t worker = blockIdx.x * NW + wave;
            const int64_t p = sh.total > 0 && worker < sh.workers ? sh.at(worker) : -1;
            if (sh.total > 0) plan_find<1>(a, lines, plan, sh, p, &walk);
            narrow_share<DT, D, SCORES>(a, narrow, sh, worker, walk, p, q, k, v, sm.tiles[wave]);
            __syncthreads();
            continue;
        }
        // workgroups go to the XCDs in turn: each XCD has a part of the line of its own
        const PagedShare &sh = shares[0];
        int32_t worker = blockIdx.x;
        if (sh.workers == (int32_t)gridDim.x && sh.workers % 8 == 0)
            worker = blockIdx.x % 8 * (sh.workers / 8) + blockIdx.x / 8;
        int64_t p = sh.total > 0 && worker < sh.workers ? sh.at(worker) : -1;
        if (sh.total > 0) plan_find<0>(a, lines, plan, sh, p, &walk);
        if (threadIdx.x == 0) wide.jobs[worker].rows = 0;
        if (p < 0) continue;
        const int64_t end = sh.at(worker + 1);
        for (;;) {
            int64_t next;
            int32_t last;
            PagedPiece x = piece_of(a, wide, walk, sh, worker, p, end, &next, &last);
            settle_piece(x);
            if (last >= 0 && threadIdx.x == 0)
                wide.jobs[worker] = PagedJob{x.tok, x.head, x.per, x.rows, x.first, last};
            paged_wide<DT, D>(a, wide, x, pool_of(a, x, k, v), q, sm.wide, flags, sm.tiles);
            p = next;
            if (p >= end || !walk_on(a, wide, walk, next)) break;
        }
        __syncthreads();
    }
}

// The pieces of shared tiles joined: D / V threads a row, V columns each, the workgroup's other threads take other rows,
// or where a row's pieces are more than kJoinMany share those out (each every so-many-th of them, added in order). A
// thread needs nothing but its own loads: its reference moves as in the sweep.
constexpr int kJoinFew = 4;  // the pieces that a thread has in flight
template <int V>
struct Joined {
    float m, sum, acc[V];
};
template <int V>
__device__ __forceinline__ void join_one(Joined<V> &j, float m, float sum, const float *o) {
    const float top = fmaxf(j.m, m);
    // (a piece without weight: zeros, and a reference of -inf that may be the largest all the same)
    const float f = j.m == top ? 1.f : fast_exp2(j.m - top), g = m == top ? 1.f : fast_exp2(m - top);
    j.m = top;
    j.sum = j.sum * f + sum * g;
#pragma unroll
    for (int c = 0; c < V; c++) j.acc[c] = j.acc[c] * f + o[c] * g;
}
template <int DT, int V>
__global__ __launch_bounds__(256) void paged_join(PagedArgs a, PagedLine narrow, PagedLine wide, int32_t nblocks) {
    __shared__ float red[256 * (V + 2)];
    const int tid = threadIdx.x, per = a.d / V, slots = 256 / per, slot = tid / per, c = (tid - slot * per) * V;
    // (narrow tiles' workgroups first: y of them a job)
    const bool w = (int32_t)blockIdx.x >= nblocks;
    const PagedLine &l = w ? wide : narrow;
    const int32_t y = (l.pitch + slots - 1) / slots, i = blockIdx.x - (w ? nblocks : 0), jb = i / y;
    const PagedJob job = l.jobs[jb];
    if (job.rows == 0) return;  // (of a worker without a job the rest is not written)
    const int32_t n = job.last - job.first + 1;
    const bool few = n <= kJoinMany;
    // (many: kJoinMany jobs or more of y workgroups each are more than a tile has rows, narrow or wide)
    const int32_t r0 = few ? (i - jb * y) * slots : i - jb * y + (jb - job.first - 1) * y, r = few ? r0 + slot : r0;
    if (r0 >= job.rows) return;
    const int32_t step = few ? 1 : slots;
    const bool on = slot < slots && r < job.rows;
    Joined<V> j{-INFINITY, 0.f, {}};
    for (int32_t p0 = few ? 0 : slot; on && p0 < n; p0 += kJoinFew * step) {
        float2 ml[kJoinFew];
        float o[kJoinFew][V];
#pragma unroll
        for (int u = 0; u < kJoinFew; u++) {
            const int32_t p = min(p0 + u * step, n - 1);  // (past the last: read again, left out)
            const int64_t at = (int64_t)(2 * (job.first + p) + (p == 0 ? 1 : 0)) * l.pitch + r;
            ml[u] = l.ml[at];
            if constexpr (V == 4)
                *(float4 *)o[u] = *(const float4 *)(l.o + at * a.d + c);
            else
                o[u][0] = l.o[at * a.d + c];
        }
#pragma unroll
        for (int u = 0; u < kJoinFew; u++)
            if (p0 + u * step < n) join_one<V>(j, ml[u].x, ml[u].y, o[u]);
    }
    if (!few) {
        float *mine = red + tid * (V + 2);
        mine[0] = j.m, mine[1] = j.sum;
#pragma unroll
        for (int u = 0; u < V; u++) mine[2 + u] = j.acc[u];
        __syncthreads();
        if (slot != 0) return;
        for (int k = 1; k < min(slots, n); k++) {
            const float *other = red + (tid + k * per) * (V + 2);
            join_one<V>(j, other[0], other[1], other + 2);
        }
    }
    if (!on) return;
    const float inv = j.sum == 0.f ? 0.f : 1.f / j.sum;  // (NaN is not 0)
    const int32_t t = r / job.per;
    const int64_t row = (int64_t)(job.tok + t) * a.hq + job.head + (r - t * job.per);
    if constexpr (V == 4 && DT != DM_F32) {
        *(uint2 *)((uint16_t *)a.o + row * a.d + c) =
            make_uint2(pack2<DT>(j.acc[0] * inv, j.acc[1] * inv), pack2<DT>(j.acc[2] * inv, j.acc[3] * inv));
    } else if constexpr (V == 4) {
        *(float4 *)((float *)a.o + row * a.d + c) =
            make_float4(j.acc[0] * inv, j.acc[1] * inv, j.acc[2] * inv, j.acc[3] * inv);
    } else {
        st<DT>(a.o, row * a.d + c, j.acc[0] * inv);
    }
    if (c == 0 && a.lse) a.lse[row] = lse_of(j.m, j.sum);
}

// ------------------------------------------------------------------------------------------
// The weights that the cached keys get
// ------------------------------------------------------------------------------------------
//
// weights[s, j] += sum over the tokens and heads that see key j of e^(scale q k_j - lse). Keys lie in tiles, and a tile
// goes through every head's rows that see any of its keys: S = q K^T, whose columns are the keys, so that a key's sum
// stays in its lane. The tiles lie on a line as the attention's do, and a tile that workers share is summed by a
// second launch, so that one value is added to a weight, in a fixed order.
//
// The simple form: a wavefront is a worker, a tile 32 keys in registers, rows 32 at a time straight from memory.

// Half a row of DP elements (zeros past the row's d) for the f32 products, from `row` on; `is`: there is one.
template <int DT, int VEC, int HALF>
__device__ __forceinline__ void load_half(const void *pool, int64_t row, int d, bool is, const void *safe, float (&y)[HALF]) {
    constexpr int SIZE = DT == DM_F32 ? 4 : 2;
    const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int u = 0; u < HALF / VEC; u++) {
        const int c = half * HALF + u * VEC;
        const bool here = is && c < d;
        const float4 v = load_some<DT, VEC>(here ? (const char *)pool + (row + c) * SIZE : (const char *)safe);
        const float f4[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < VEC; e++) y[u * VEC + e] = here ? f4[e] : 0.f;
    }
}

template <int DT, int DP, int VEC>
__global__ __launch_bounds__(256) void paged_weights_simple(PagedArgs a, KeyLine l, const void *__restrict__ q,
                                                            const void *__restrict__ k, float *__restrict__ weights,
                                                            int64_t stride) {
    constexpr int HALF = DP / 2;
    __shared__ PlanSmem<256, 1> plan;
    const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
    const int32_t worker = blockIdx.x * 4 + uni(threadIdx.x >> 6);
    PagedWalk walk;
    const KeyLine lines[1] = {l};
    PagedShare shares[1];
    plan_lines(a, lines, plan, shares);
    const PagedShare &sh = shares[0];
    int64_t p = sh.total > 0 && worker < sh.workers ? sh.at(worker) : -1;
    plan_find<0>(a, lines, plan, sh, p, &walk);
    if (lane == 0) l.jobs[worker].rows = 0;
    if (p < 0) return;
    const int64_t end = sh.at(worker + 1);
    const float c2 = a.scale * kLog2e;
    for (;;) {
        int64_t next;
        int32_t last;
        const KeyPiece x = key_piece(a, l, walk, sh, worker, p, end, &next, &last);
        if (last >= 0 && lane == 0) l.jobs[worker] = PagedJob{x.s, walk.t, 0, 1, worker - 1, last};
        const int32_t len = walk.q.len, p0 = walk.q.len - walk.q.n, key = x.k0 + col;
        const int64_t e = min(key, len - 1) / a.page_size, pg = a.table[x.s * a.max_pages + e];
        const bool is = key < len && pg >= 0 && pg < a.num_pages;
        const int64_t off = is ? pg * a.kb + (key - e * a.page_size) * a.kt : 0;
        float total = 0.f;
        for (int32_t r = x.r0; r < x.r1;) {
            const int32_t kh = r / x.steps, n = min(x.r1, (kh + 1) * x.steps) - r;  // this head's steps
            float kf[HALF], qf[HALF], sub = 0.f;
            load_half<DT, VEC>(k, off + kh * a.kh, a.d, is, q, kf);
            for (int32_t i = 0; i < n; i++) {
                const int32_t row = x.from + (r - kh * x.steps + i) * 32 + col;
                const bool on = row < x.to;
                const int32_t t = on ? row / a.rep : 0, h = on ? row - t * a.rep : 0;
                const int64_t tok = walk.q.first + t;
                load_half<DT, VEC>(q, tok * a.qt + (int64_t)(kh * a.rep + h) * a.qh, a.d, on, q, qf);
                const float ls = a.lse[tok * a.hq + kh * a.rep + h];
                const float ref = on && ls != -INFINITY ? -ls * kLog2e : -INFINITY;
                f32x16_t sc = zero16();
#pragma unroll
                for (int c = 0; c < HALF; c++) sc = mfma2(qf[c], kf[c], sc);
                float part = 0.f;
#pragma unroll
                for (int u = 0; u < 16; u++) {
                    const int y = crow(u, lane);
                    const float rf = __shfl(ref, y, 64);
                    const int32_t pos = p0 + __shfl(t, y, 64);
                    const bool seen = rf != -INFINITY && key <= pos && (a.left < 0 || key >= pos - a.left);
                    part += seen ? fast_exp2(fmaf(sc[u], c2, rf)) : 0.f;
                }
                sub += part;
            }
            total += sub;
            r += n;
        }
        total += __shfl_xor(total, 32, 64);
        if (half == 0) {
            if (!x.whole)
                l.sums[(int64_t)x.slot * l.keys + col] = total;
            else if (key < len && x.r1 > 0)
                weights[x.s * stride + key] += total;
        }
        p = next;
        if (p >= end || !walk_on(a, l, walk, next)) return;
    }
}

// The 16-bit kernel: a workgroup takes a tile of keys, 64 of them a wavefront (32 at D = 256) in registers as the second
// operand, and sweeps the rows that see them, 64 at a time through LDS, head by head. A key's sum over a step's 32
// rows is taken first, then over a head's, then over the heads (one at a time, a long sum would lose bits). 1024 tokens
// of 32 heads of 128 against 16384 keys take 236-250 us (530-560 TFLOP/s): the products and the exponentials follow one
// another in a wavefront, and two wavefronts a SIMD are all that the keys' registers leave.
template <int D>
constexpr int key_cols() { return D == 256 ? 1 : 2; }  // 32-key columns of a wavefront
template <int D>
constexpr int key_tile() { return 8 * 32 * key_cols<D>(); }
template <int D>
union KeyTiles {
    static constexpr int KS = D + 8;
    PlanSmem<512, 1> plan;
    struct {
        alignas(16) uint16_t q[2][64 * KS];
        alignas(16) float ref[2][64];  // -lse in log2 units, -inf for a row that is none or sees no key
        alignas(16) int32_t pos[2][64];
    } rows;
    alignas(16) uint16_t keys[8][32 * KS];
};

template <int DT, int D>
__global__ __launch_bounds__(512, 2) void paged_weights_kernel(PagedArgs a, KeyLine l, const void *__restrict__ q,
                                                              const void *__restrict__ k, float *__restrict__ weights,
                                                              int64_t stride) {
    constexpr int KS = KeyTiles<D>::KS, COLS = key_cols<D>(), KST = D / 16, LPR = D / 8, RPL = 64 / LPR, NLD = 32 / RPL;
    constexpr int RSTEP = 512 / LPR, NCH = 64 / RSTEP;  // rows at a time, 16-byte pieces a thread, of a step's queries
    __shared__ KeyTiles<D> sm;
    const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6), col = lane & 31, half = lane >> 5;
    const int32_t worker = blockIdx.x;
    PagedWalk walk;
    const KeyLine lines[1] = {l};
    PagedShare shares[1];
    plan_lines(a, lines, sm.plan, shares);
    const PagedShare &sh = shares[0];
    int64_t p = sh.total > 0 && worker < sh.workers ? sh.at(worker) : -1;
    plan_find<0>(a, lines, sm.plan, sh, p, &walk);
    if (tid == 0) l.jobs[worker].rows = 0;
    if (p < 0) return;
    const int64_t end = sh.at(worker + 1);
    const float c2 = a.scale * kLog2e;
    const int32_t rep = a.rep, more = 64 / rep, rest = 64 - more * rep;  // 64 rows on: tokens and heads
    const int32_t left = a.left >= 0 ? a.left : 1 << 30;  // (without a window more than a row holds)
    for (;;) {
        int64_t next;
        int32_t last;
        const KeyPiece x = key_piece(a, l, walk, sh, worker, p, end, &next, &last);
        if (last >= 0 && tid == 0) l.jobs[worker] = PagedJob{x.s, walk.t, 0, 1, worker - 1, last};
        const int32_t s = uni(x.s), len = uni(walk.q.len), p0 = uni(walk.q.len - walk.q.n), tok0 = uni(walk.q.first);
        const int32_t from = uni(x.from), to = uni(x.to), steps = uni(x.steps);
        const int32_t w0 = uni(x.k0) + wave * 32 * COLS;  // the wavefront's first key
        const int32_t *entries = a.table + s * a.max_pages;
        uint32_t at = kNoKey;  // the place of key w0 + lane
        if (w0 + lane < len && lane < 32 * COLS) {
            const uint32_t e = (uint32_t)(w0 + lane) / (uint32_t)a.page_size, row = (uint32_t)(w0 + lane) - e * (uint32_t)a.page_size;
            const int32_t pg = entries[e];
            if ((uint32_t)pg < (uint32_t)a.num_pages) at = (uint32_t)pg * (uint32_t)(a.kb / 8) + row * (uint32_t)(a.kt / 8);
        }
        float total[COLS];
#pragma unroll
        for (int c = 0; c < COLS; c++) total[c] = 0.f;
        for (int32_t r = uni(x.r0), r1 = uni(x.r1); r < r1;) {
            const int32_t kh = uni(r / steps), n = min(r1, (kh + 1) * steps) - r;  // this head's steps
            const int32_t first = from + (r - kh * steps) * 64;                     // its first row
            const char *base = (const char *)k + (int64_t)kh * a.kh * 2;
            uint4 sk[COLS][NLD];
#pragma unroll
            for (int c = 0; c < COLS; c++)
#pragma unroll
                for (int u = 0; u < NLD; u++) {
                    const uint32_t y = __shfl(at, c * 32 + RPL * u + lane / LPR, 64);
                    const bool ok = y != kNoKey;
                    sk[c][u] = only(ok, *(const uint4 *)(base + (uint64_t)(ok ? y : 0u) * 16 + (lane % LPR) * 16));
                }
            // this thread's rows of a step: token and head of each, moved on by 64 rows a step
            int32_t t[NCH + 1], h[NCH + 1];
#pragma unroll
            for (int u = 0; u <= NCH; u++) {
                const int32_t y = first + (u < NCH ? tid / LPR + u * RSTEP : lane);
                t[u] = y / rep, h[u] = y - t[u] * rep;
            }
            int32_t ts = uni(first / rep), hs = uni(first - ts * rep);  // the step's first row
            uint4 sq[NCH];
            float ref = 0.f;
            int32_t pos = 0;
            auto load = [&](int32_t i) __attribute__((always_inline)) {  // step i's queries
#pragma unroll
                for (int u = 0; u < NCH; u++) {
                    const bool ok = first + i * 64 + tid / LPR + u * RSTEP < to;
                    const int64_t y = (int64_t)(tok0 + (ok ? t[u] : 0)) * a.qt + (int64_t)(kh * rep + (ok ? h[u] : 0)) * a.qh;
                    sq[u] = only(ok, *(const uint4 *)((const uint16_t *)q + y + (tid % LPR) * 8));
                }
                if (wave == 0) {
                    const bool ok = first + i * 64 + lane < to;
                    const float ls = ok ? a.lse[(int64_t)(tok0 + t[NCH]) * a.hq + kh * rep + h[NCH]] : -INFINITY;
                    ref = ls == -INFINITY ? ls : -ls * kLog2e;
                    pos = p0 + t[NCH];
                }
#pragma unroll
                for (int u = 0; u <= NCH; u++) {
                    t[u] += more, h[u] += rest;
                    if (h[u] >= rep) t[u]++, h[u] -= rep;
                }
            };
            auto store = [&](int b) __attribute__((always_inline)) {
#pragma unroll
                for (int u = 0; u < NCH; u++)
                    *(uint4 *)(sm.rows.q[b] + (tid / LPR + u * RSTEP) * KS + (tid % LPR) * 8) = sq[u];
                if (wave == 0) sm.rows.ref[b][lane] = ref, sm.rows.pos[b][lane] = pos;
            };
            load(0);
            Frag8 kf[COLS][KST];
            __syncthreads();  // (the last head's rows have been read)
#pragma unroll
            for (int c = 0; c < COLS; c++) {
                uint16_t *rows = sm.keys[wave];
#pragma unroll
                for (int u = 0; u < NLD; u++) *(uint4 *)(rows + (RPL * u + lane / LPR) * KS + (lane % LPR) * 8) = sk[c][u];
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int st = 0; st < KST; st++) kf[c][st].u = *(const uint4 *)(rows + col * KS + st * 16 + half * 8);
                __builtin_amdgcn_wave_barrier();
            }
            __syncthreads();
            store(0);
            __syncthreads();
            float sub[COLS];
#pragma unroll
            for (int c = 0; c < COLS; c++) sub[c] = 0.f;
            for (int32_t i = 0; i < n; i++) {
                const int b = i & 1;
                if (i + 1 < n) load(i + 1);
                const int tiles = first + i * 64 + 32 < to ? 2 : 1;
                // all of the step's rows see all of the wavefront's keys (those of the last token may be fewer), and none is
                // absent: its zeros times an infinite key are NaN, which a reference of -inf does not take out
                const bool full = p0 + ts >= w0 + 32 * COLS - 1 && (a.left < 0 || p0 + ts + more + 1 - a.left <= w0) &&
                                  first + i * 64 + tiles * 32 <= to;
                const uint16_t *tq = sm.rows.q[b] + col * KS + half * 8;
                for (int y = 0; y < tiles; y++) {
                    // (each fragment is read ahead of the products in front of it)
                    constexpr int READ = 3;
                    Frag8 f[READ + 1];
                    auto read = [&](int st) __attribute__((always_inline)) {
                        f[st % (READ + 1)].u = *(const uint4 *)(tq + y * 32 * KS + st * 16);
                    };
                    f32x16_t sc[COLS];
#pragma unroll
                    for (int c = 0; c < COLS; c++) sc[c] = zero16();
#pragma unroll
                    for (int st = 0; st < READ; st++) read(st);
#pragma unroll
                    for (int st = 0; st < KST; st++) {
                        if (st + READ < KST) read(st + READ);
#pragma unroll
                        for (int c = 0; c < COLS; c++) sc[c] = mfma32<DT>(f[st % (READ + 1)], kf[c][st], sc[c]);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    float rf[16];
#pragma unroll
                    for (int g = 0; g < 4; g++)
                        *(float4 *)(rf + g * 4) = *(const float4 *)(sm.rows.ref[b] + y * 32 + g * 8 + half * 4);
#pragma unroll
                    for (int e = 0; e < 16; e++)
#pragma unroll
                        for (int c = 0; c < COLS; c++) sc[c][e] = fmaf(sc[c][e], c2, rf[e]);
                    if (!full) {
#pragma unroll
                        for (int g = 0; g < 4; g++) {
                            const int4 ps = *(const int4 *)(sm.rows.pos[b] + y * 32 + g * 8 + half * 4);
                            const int32_t p4[4] = {ps.x, ps.y, ps.z, ps.w};
#pragma unroll
                            for (int e = 0; e < 4; e++)
#pragma unroll
                                for (int c = 0; c < COLS; c++) {
                                    const int32_t key = w0 + c * 32 + col;
                                    const bool seen = (key <= p4[e]) & (key >= p4[e] - left) & (rf[g * 4 + e] != -INFINITY);
                                    sc[c][g * 4 + e] = seen ? sc[c][g * 4 + e] : -INFINITY;
                                }
                        }
                    }
#pragma unroll
                    for (int c = 0; c < COLS; c++) {
                        float part = 0.f;
#pragma unroll
                        for (int e = 0; e < 16; e++) part += fast_exp2(sc[c][e]);
                        sub[c] += part;
                    }
                }
                ts += more, hs += rest;
                if (hs >= rep) ts++, hs -= rep;
                if (i + 1 < n) store(b ^ 1);
                __syncthreads();
            }
#pragma unroll
            for (int c = 0; c < COLS; c++) total[c] += sub[c];
            r += n;
        }
#pragma unroll
        for (int c = 0; c < COLS; c++) {
            const float y = total[c] + __shfl_xor(total[c], 32, 64);
            const int32_t i = wave * 32 * COLS + c * 32 + col;
            if (half == 0) {
                if (!x.whole)
                    l.sums[(int64_t)x.slot * l.keys + i] = y;
                else if (w0 + c * 32 + col < len && x.r1 > 0)
                    weights[s * stride + w0 + c * 32 + col] += y;
            }
        }
        p = next;
        if (p >= end || !walk_on(a, l, walk, next)) return;
        __syncthreads();
    }
}

// The pieces of a shared tile's sums, in the order of the workers.
__global__ __launch_bounds__(256) void paged_weights_join(PagedArgs a, KeyLine l, float *__restrict__ weights, int64_t stride) {
    const PagedJob job = l.jobs[blockIdx.x];
    if (job.rows == 0) return;
    const int32_t i = blockIdx.y * 256 + threadIdx.x, key = job.head * l.keys + i;
    if (i >= l.keys || key >= paged_seq(a, job.tok).len) return;
    float y = 0.f;
    for (int32_t w = job.first; w <= job.last; w++) y += l.sums[(int64_t)(2 * w + (w == job.first ? 1 : 0)) * l.keys + i];
    weights[job.tok * stride + key] += y;
}

// Narrow tiles: their sweep has left the scores, 4 bytes a (row, key) where the keys themselves are 2 D a head. A thread
// a key, the rows of a head first, then the heads.
__global__ __launch_bounds__(256) void paged_weights_narrow(PagedArgs a, float *__restrict__ weights, int64_t stride,
                                                            int32_t blocks, int32_t upto) {
    const int32_t s = blockIdx.x / blocks, key = (blockIdx.x - s * blocks) * 256 + threadIdx.x;
    const PagedSeq q = paged_seq(a, s);
    const int32_t rows = q.n * a.rep;
    if (q.n == 0 || (int64_t)q.n * a.rep > upto || key >= q.len) return;
    const int32_t p0 = q.len - q.n;
    float total = 0.f;
    for (int32_t kh = 0; kh < a.hkv; kh++) {
        const float *at = a.scores + ((int64_t)s * a.hkv + kh) * a.score_rows * a.cap + key;
        const float *ls = a.lse + (int64_t)q.first * a.hq + kh * a.rep;
        float sub = 0.f;
        int32_t i = 0, h = 0;
#pragma unroll 8
        for (int32_t r = 0; r < rows; r++) {
            const float l = ls[(int64_t)i * a.hq + h];
            const bool seen = key <= p0 + i && (a.left < 0 || key >= p0 + i - a.left) && l != -INFINITY;
            const float x = at[(int64_t)r * a.cap];  // (of a key that the row does not see: whatever lies there)
            sub += seen ? fast_exp2(fmaf(-l, kLog2e, x)) : 0.f;
            if (++h == a.rep) h = 0, i++;
        }
        total += sub;
    }
    weights[s * stride + key] += total;
}

// ------------------------------------------------------------------------------------------
// Host
// ------------------------------------------------------------------------------------------

static int padded(int64_t d) { return d <= 64 ? 64 : (d <= 128 ? 128 : 256); }

// A line's shape for rows of `rep` heads in tiles of rt.
static PagedLine line_of(const dm_attention_desc *d, int32_t rt, int32_t over, int32_t upto) {
    PagedLine l{};
    const int32_t rep = (int32_t)(d->hq / d->hkv);
    l.rt = rt;
    l.hc = (rep + rt - 1) / rt;
    l.m = l.hc > 1 ? 1 : rt / rep;
    l.per = l.hc > 1 ? rt : rep;
    l.over = over, l.upto = upto;
    // (without offsets no sequence has more than one token)
    const int64_t tokens = d->cu_seqlens_q ? std::min<int64_t>(d->tq, l.m) : 1;
    l.pitch = (int32_t)std::min<int64_t>(rt, tokens * rep);
    return l;
}

// The 16-bit kernels' calls: 16-byte pieces, keys' and values' pages laid out alike, places that 32 bits of
// 16-byte units hold. (A size query comes without the pool.)
static bool paged_fast_shape(const dm_attention_desc *d) {
    if ((d->dtype != DM_BF16 && d->dtype != DM_F16) || (d->d != 64 && d->d != 128 && d->d != 256)) return false;
    if (!d->strided) return true;
    const dm_strides &k = d->sk, &v = d->sv;
    return d->sq.t % 8 == 0 && d->sq.h % 8 == 0 && k.b % 8 == 0 && k.t % 8 == 0 && k.h % 8 == 0 && v.h % 8 == 0 &&
           k.b == v.b && k.t == v.t;
}
static bool paged_fast_pool(const PagedArgs &a) {
    const int64_t most = ((int64_t)1 << 32) * 8 - 8;  // elements
    return a.num_pages > 0 && a.kb < most / a.num_pages / 2 && a.kt < most / a.page_size / 2;
}

// Most bytes of scores kept (0.7% of the card's memory; calls whose table is so wide that they could need more go through
// the keys again: 64 tokens of 4 rows a head against 4096 keys 257 us for 201).
constexpr int64_t kScoreBytes = (int64_t)1 << 31;
struct PagedPlan {
    bool fast, mixed;
    PagedLine wide, narrow;  // the simple kernel's: narrow
    size_t bytes;
    KeyLine keys;            // with weights
    int64_t score_rows;      // of a sequence's head, with the narrow tiles' scores kept (0: not)
    size_t scores;
    size_t lse;              // where their own log-sum-exps lie
};
static size_t place_line(const dm_attention_desc *d, PagedLine *l, char *base, size_t at) {
    const size_t rows = (size_t)2 * l->workers * l->pitch;
    l->o = (float *)(base + at);
    at += align_up(rows * d->d * sizeof(float));
    l->ml = (float2 *)(base + at);
    at += align_up(rows * sizeof(float2));
    l->jobs = (PagedJob *)(base + at);
    return at + align_up((size_t)l->workers * sizeof(PagedJob));
}
static PagedPlan paged_plan(const dm_attention_desc *d, char *base, bool weights, bool fast) {
    PagedPlan p{};
    const int64_t rep = d->hq / d->hkv;
    p.fast = fast;
    // (whether a sequence has more rows than a narrow one's is known only on the device, but for calls that cannot)
    p.mixed = fast && (d->cu_seqlens_q ? d->tq : 1) * rep > lone_rows(d->d);
    if (p.mixed) {
        p.wide = line_of(d, d->d == 256 ? 128 : 256, kNarrowRows, INT32_MAX);
        p.wide.workers = 256;
        p.wide.unit = 64;
        // (a tile's start as long as 192 keys: 48 calls of 1 to 16 sequences, 4 to 1200 rows a key head each, widths of 64
        // to 256, in the mean 44.0 us, with 64 45.2, with 384 44.9; with 128, 256, 512 and 1024 keys a worker at least 43.3,
        // 44.0, 46.9 and 55.2: 128 is ahead for one or two sequences, 3-20%, 256 for eight of 20 tokens, 4-12%)
        p.wide.start = 192;
        p.wide.least = 256;
        p.bytes = place_line(d, &p.wide, base, p.bytes);
    }
    p.narrow = line_of(d, 32, 0, p.mixed ? kNarrowRows : INT32_MAX);
    p.narrow.workers = d->d > 128 ? 1024 : 2048;
    p.narrow.unit = 32;
    // (a worker has 32 keys at least: four tokens against 500 to 1000 keys 29 us with 128, 24.5 so. The simple kernel
    // takes longer for 32 keys than for a tile's start: 210 tokens of 4 heads of 64 in f32 39 us with the same, 35.5 so)
    p.narrow.start = fast ? 64 : 32;
    p.narrow.least = fast ? 96 : 32;
    p.bytes = place_line(d, &p.narrow, base, p.bytes);
    p.lse = p.bytes;
    if (weights) {
        p.bytes += align_up((size_t)(d->tq * d->hq) * sizeof(float));
        KeyLine &l = p.keys;
        l.keys = !fast ? 32 : (d->d == 256 ? key_tile<256>() : key_tile<128>());
        l.workers = fast ? 256 : 4096;
        l.unit = fast ? 64 : 32;
        // (rows; three prompts of 300 tokens against 600 keys, with their weights, 127 us with 1024 rows a worker at least,
        // 111 with 512, 105 with 256; 64 of 16 tokens of 8 heads against 1024 keys 79, 70, 68; a start of 64 136 and 97)
        l.start = fast ? 256 : 64;
        l.least = fast ? 256 : 128;
        l.sums = (float *)(base + p.bytes);
        p.bytes += align_up((size_t)2 * l.workers * l.keys * sizeof(float));
        l.jobs = (PagedJob *)(base + p.bytes);
        p.bytes += align_up((size_t)l.workers * sizeof(PagedJob));
        // the narrow tiles' scores, where the longest that the call could have fit
        const int64_t most = std::min<int64_t>(kScoreRows, (d->cu_seqlens_q ? d->tq : 1) * rep);
        const int64_t row = d->tk * (int64_t)sizeof(float);
        if (fast && d->b * d->hkv * most <= kScoreBytes / std::max<int64_t>(row, 1) && d->b * ((d->tk + 255) / 256) < (1 << 23) &&
            kScoreRows * row < ((int64_t)1 << 32)) {
            p.score_rows = most;
            p.scores = p.bytes;
            p.bytes += align_up((size_t)(d->b * d->hkv * most * row));
            l.over = kScoreRows;
        }
    }
    return p;
}

static const int64_t kPagedRows = (int64_t)1 << 26;  // most token x head rows: a line's length fits 63 bits
static bool paged_sizes(const dm_attention_desc *d) {
    const int64_t big = (int64_t)1 << 30;
    return d && d->hkv > 0 && d->hq >= 0 && d->hq % d->hkv == 0 && d->hq < 65536 && d->tq >= 0 && d->tq < big && d->b >= 0 &&
           d->b < big && d->tk >= 0 && d->tk <= big && d->d >= 0 && d->d <= 256 &&
           d->tq * std::max<int64_t>(d->hq, d->hkv) < kPagedRows;
}

}  // namespace dm

using namespace dm;

extern "C" {

size_t dm_attention_paged_workspace(const dm_attention_desc *d, int64_t page_size, int weights) {
    if (!paged_sizes(d) || page_size < 1 || d->hq == 0) return 0;
    // (which kernel runs also depends on the pool and the pointers' alignment)
    return std::max(paged_plan(d, nullptr, weights != 0, false).bytes,
                    paged_plan(d, nullptr, weights != 0, paged_fast_shape(d)).bytes);
}

int dm_attention_paged(const dm_attention_desc *d, const void *q, const void *k_pages, const void *v_pages,
                       int64_t num_pages, int64_t page_size, const int32_t *block_table, int64_t max_pages,
                       const int32_t *lengths, void *o, float *lse, float *weights, int64_t weights_stride,
                       void *workspace, size_t workspace_bytes, void *stream) {
    const std::string op("attention_paged");
    if (int rc = check_decode(op.c_str(), d)) return rc;
    if (d->tq < 0) return refuse(op + ": bad dimensions");
    if (page_size < 1 || max_pages < 0 || num_pages < 0)
        return refuse(op + ": page_size must be positive, max_pages and num_pages not negative");
    if (!paged_sizes(d) || num_pages >= ((int64_t)1 << 31))
        return refuse(op + ": more tokens, heads, keys or pages than this library takes");
    if (page_size >= ((int64_t)1 << 31) || max_pages >= ((int64_t)1 << 31) || d->tk != max_pages * page_size)
        return refuse(op + ": desc->tk (" + std::to_string(d->tk) + ") must be max_pages * page_size");
    if (d->cu_seqlens_k || d->mask_kind != DM_MASK_NONE)
        return refuse(op + ": the sequences are cut by cu_seqlens_q alone, with no mask");
    if (!d->cu_seqlens_q && d->tq != d->b)
        return refuse(op + ": without cu_seqlens_q there is one token a sequence, tq = b");
    if (d->strided && d->sq.t < 0) return refuse(op + ": strides must not be negative");
    if (d->b > 0 && (!lengths || (d->tk > 0 && !block_table)))
        return refuse(op + ": the block table is [S, max_pages] and the lengths [S], int32");
    if (weights && weights_stride < d->tk && d->b > 1)
        return refuse(op + ": the weights are [S, max_pages * page_size], their rows apart");
    if (workspace_bytes < dm_attention_paged_workspace(d, page_size, weights != nullptr))
        return refuse(op + ": the workspace is smaller than dm_attention_paged_workspace");
    hipStream_t st = (hipStream_t)stream;
    const int64_t rows = d->tq * d->hq;
    if (rows == 0) return DM_OK;
    if (d->tk == 0 || d->b == 0 || d->d == 0) {  // no key
        fill_zero(o, rows * d->d * dtype_bytes(d->dtype), st);
        if (lse) fill_f32(lse, -INFINITY, rows, st);
        DM_LAUNCH_CHECK("attention_paged: fill");
        return DM_OK;
    }
    PagedArgs a{};
    a.S = (int32_t)d->b, a.N = (int32_t)d->tq, a.cap = (int32_t)d->tk, a.left = (int32_t)left_of(d);
    a.hq = (int32_t)d->hq, a.hkv = (int32_t)d->hkv, a.d = (int32_t)d->d, a.rep = (int32_t)(d->hq / d->hkv);
    a.scale = scale_of(d);
    a.lengths = lengths, a.cu = d->cu_seqlens_q, a.table = block_table;
    a.page_size = page_size, a.max_pages = max_pages, a.num_pages = num_pages;
    if (d->strided) {
        a.qt = d->sq.t, a.qh = d->sq.h;
        a.kb = d->sk.b, a.kt = d->sk.t, a.kh = d->sk.h;
        a.vb = d->sv.b, a.vt = d->sv.t, a.vh = d->sv.h;
    } else {
        const int64_t row = d->hkv * d->d;
        a.qt = d->hq * d->d, a.qh = d->d;
        a.kb = a.vb = page_size * row, a.kt = a.vt = row, a.kh = a.vh = d->d;
    }
    const bool fast = paged_fast_shape(d) && paged_fast_pool(a) && aligned_16b(q) && aligned_16b(k_pages) &&
                      aligned_16b(v_pages) && aligned_16b(o);
    const PagedPlan p = paged_plan(d, (char *)workspace, weights != nullptr, fast);
    a.o = o;
    a.lse = lse ? lse : (weights ? (float *)((char *)workspace + p.lse) : nullptr);
    if (p.score_rows) a.scores = (float *)((char *)workspace + p.scores), a.score_rows = (int32_t)p.score_rows;
    // (four elements at a time where rows and bases allow it)
    const int64_t eb = dtype_bytes(d->dtype);
    const bool vec = ((d->d | a.kb | a.kt | a.kh | a.vb | a.vt | a.vh) & 3) == 0 &&
                     (((uintptr_t)k_pages | (uintptr_t)v_pages) & (4 * eb - 1)) == 0;
    const bool vecq = vec && ((a.qt | a.qh) & 3) == 0 && ((uintptr_t)q & (4 * eb - 1)) == 0;
    const PagedLine &l = p.narrow;
    const unsigned g = l.workers / 4;
    const int slots = 256 / (int)(d->d % 4 == 0 && aligned_16b(o) ? d->d / 4 : d->d);  // rows of a joining workgroup
    const int nb = l.workers * ((l.pitch + slots - 1) / slots);
    const int wb = p.mixed ? p.wide.workers * ((p.wide.pitch + slots - 1) / slots) : 0;
#define PAGED_W(DT, DP)                                                                                       \
    if (weights && !fast && vecq)                                                                             \
        paged_weights_simple<DT, DP, 4><<<p.keys.workers / 4, 256, 0, st>>>(a, p.keys, q, k_pages, weights, weights_stride); \
    else if (weights && !fast)                                                                                \
        paged_weights_simple<DT, DP, 1><<<p.keys.workers / 4, 256, 0, st>>>(a, p.keys, q, k_pages, weights, weights_stride); \
    if (p.score_rows)                                                                                         \
        paged_weights_narrow<<<(unsigned)(d->b * ((d->tk + 255) / 256)), 256, 0, st>>>(                       \
            a, weights, weights_stride, (int32_t)((d->tk + 255) / 256), kScoreRows);                         \
    if (weights && (!p.score_rows || (d->cu_seqlens_q ? d->tq : 1) * a.rep > kScoreRows)) {                                                     \
        if constexpr (DT != DM_F32) {                                                                         \
            if (fast)                                                                                         \
                paged_weights_kernel<DT, DP><<<p.keys.workers, 512, 0, st>>>(a, p.keys, q, k_pages, weights, weights_stride); \
        }                                                                                                     \
        paged_weights_join<<<dim3(p.keys.workers, (p.keys.keys + 255) / 256), 256, 0, st>>>(a, p.keys, weights, weights_stride); \
    }
#define PAGED_FAST(DT, DP, SC)                                                                                \
    if (p.mixed)                                                                                              \
        paged_mixed_kernel<DT, DP, SC><<<256, 64 * paged_waves<DP>(), 0, st>>>(a, p.wide, l, q, k_pages, v_pages); \
    else if (fast)                                                                                            \
        paged_narrow_kernel<DT, DP, SC><<<g, 256, 0, st>>>(a, l, q, k_pages, v_pages)
#define PAGED_V(DT, DP)                                                                                       \
    if constexpr (DT != DM_F32) {                                                                             \
        if (p.score_rows) {                                                                                   \
            PAGED_FAST(DT, DP, true);                                                                         \
        } else {                                                                                              \
            PAGED_FAST(DT, DP, false);                                                                        \
        }                                                                                                     \
    }                                                                                                         \
    if (!fast && vec)                                                                                         \
        paged_simple<DT, DP, 4><<<g, 256, 0, st>>>(a, l, q, k_pages, v_pages);                                \
    else if (!fast)                                                                                           \
        paged_simple<DT, DP, 1><<<g, 256, 0, st>>>(a, l, q, k_pages, v_pages);                                \
    if (d->d % 4 == 0 && aligned_16b(o))                                                                      \
        paged_join<DT, 4><<<nb + wb, 256, 0, st>>>(a, l, p.wide, nb);                                         \
    else                                                                                                      \
        paged_join<DT, 1><<<nb + wb, 256, 0, st>>>(a, l, p.wide, nb);                                         \
    PAGED_W(DT, DP)
#define PAGED(DT)               \
    if (padded(d->d) == 64) {   \
        PAGED_V(DT, 64);        \
    } else if (padded(d->d) == 128) { \
        PAGED_V(DT, 128);       \
    } else {                    \
        PAGED_V(DT, 256);       \
    }
    if (d->dtype == DM_F32) {
        PAGED(DM_F32)
    } else if (d->dtype == DM_BF16) {
        PAGED(DM_BF16)
    } else {
        PAGED(DM_F16)
    }
#undef PAGED
#undef PAGED_V
#undef PAGED_FAST
#undef PAGED_W
    probe_add(DM_PROBE_ATTN_PAGED);
    if (weights) probe_add(DM_PROBE_ATTN_WEIGHTS);
    DM_LAUNCH_CHECK("attention_paged: launch");
    return DM_OK;
}

}  // extern "C"
