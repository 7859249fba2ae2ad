// Attention of new tokens over a paged cache: ragged chunks of prompts, drafted tokens, single tokens.
//
// Token i of a sequence's n new ones, its length L with them, sits at position p = L - n + i and sees the keys
// max(0, p - W) .. p: o = softmax(scale q K^T) V and lse = log sum e^(scale q k). The rows of a tile (tokens x
// query heads of one key-value head) sweep their keys once with a running maximum and sum; paged_line.h says how
// the tiles are shared out and cut.
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
// wide (the head width and zeros behind it).

// VEC elements of a row of `n` from element e on, zeros past it.
template <int DT, int VEC>
__device__ __forceinline__ float4 load_some(const void *p, int64_t row, int e, int n) {
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if constexpr (VEC == 4) {
        if (e < n) {
            if constexpr (DT == DM_F32) {
                x = *(const float4 *)((const float *)p + row + e);
            } else {
                const uint2 w = *(const uint2 *)((const uint16_t *)p + row + e);
                x = make_float4(unpack_lo<DT>(w.x), unpack_hi<DT>(w.x), unpack_lo<DT>(w.y), unpack_hi<DT>(w.y));
            }
        }
    } else {
        if (e < n) x.x = ld<DT>(p, row + e);
    }
    return x;
}

template <int DT, int DP, int VEC>
__global__ __launch_bounds__(256) void paged_simple(PagedArgs a, PagedLine l, const void *__restrict__ q,
                                                    const void *__restrict__ k, const void *__restrict__ v) {
    constexpr int TS = DP + 4, CPR = DP / VEC, DTN = DP / 32, HALF = DP / 2;
    __shared__ PlanSmem<256> plan;
    __shared__ __align__(16) float tiles[4][32 * TS];
    const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6), col = lane & 31, half = lane >> 5;
    const int32_t worker = blockIdx.x * 4 + wave;
    PagedWalk walk;
    int64_t p;
    bool valid;
    const PagedShare sh = plan_line<256>(
        a, l, plan, [&](const PagedShare &s) { return worker < s.workers ? s.at(worker) : -1; }, &walk, &p, &valid);
    fill_outside<DT>(a, valid);
    if (lane == 0 && worker < l.workers) l.jobs[worker].rows = 0;
    if (p < 0) return;
    const int64_t end = sh.at(worker + 1);
    float *tile = tiles[wave];
    const float qscale = a.scale * kLog2e;
    while (p < end) {
        int64_t next;
        int32_t last;
        const PagedPiece x = piece_of(a, l, walk, sh, worker, p, end, &next, &last);
        if (last >= 0 && lane == 0) l.jobs[worker] = PagedJob{x.tok, x.head, x.per, x.rows, worker - 1, last};
        const RowKeys rk = row_keys(a, x, 0);
        float qf[HALF];
        {
            const int64_t row = (int64_t)rk.tok * a.qt + rk.head * a.qh;
#pragma unroll
            for (int e = 0; e < HALF; e++) {
                const int c = half * HALF + e;
                qf[e] = rk.on && c < a.d ? ld<DT>(q, row + c) : 0.f;
            }
        }
        f32x16_t acc[DTN];
#pragma unroll
        for (int t = 0; t < DTN; t++) acc[t] = zero16();
        float m = -INFINITY, sum = 0.f;
        const int32_t *entries = a.table + x.s * a.max_pages;
        bool bad = false;
        for (int32_t j0 = x.s0; j0 < x.s1; j0 += 32) {
            const bool cut = j0 < rk.flo || j0 + 32 > rk.fhi;
            int64_t ko = -1, vo = -1;
            if (j0 + col < x.s1) {
                const int64_t e = (j0 + col) / a.page_size, r = j0 + col - e * a.page_size, pg = entries[e];
                if (pg >= 0 && pg < a.num_pages) {
                    ko = pg * a.kb + r * a.kt + x.kh * a.kh;
                    vo = pg * a.vb + r * a.vt + x.kh * a.vh;
                }
            }
#pragma unroll 8
            for (int u = 0; u < CPR / 2; u++) {
                const int i = u * 64 + lane, r = i / CPR, e = i % CPR * VEC;
                const int64_t off = __shfl((long long)ko, r, 64);
                const float4 y = off >= 0 ? load_some<DT, VEC>(k, off, e, a.d) : make_float4(0.f, 0.f, 0.f, 0.f);
                if constexpr (VEC == 4)
                    *(float4 *)(tile + r * TS + e) = y;
                else
                    tile[r * TS + e] = y.x;
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
#pragma unroll 8
            for (int u = 0; u < CPR / 2; u++) {
                const int i = u * 64 + lane, r = i / CPR, e = i % CPR * VEC;
                const int64_t off = __shfl((long long)vo, r, 64);
                float4 y = off >= 0 ? load_some<DT, VEC>(v, off, e, a.d) : make_float4(0.f, 0.f, 0.f, 0.f);
                if (cut) {  // (a hidden key's weight is 0, and 0 times what is not finite is NaN)
                    float *c = (float *)&y;
#pragma unroll
                    for (int y = 0; y < VEC; y++)
                        if (!(fabsf(c[y]) < INFINITY)) c[y] = 0.f, bad = true;
                }
                if constexpr (VEC == 4)
                    *(float4 *)(tile + r * TS + e) = y;
                else
                    tile[r * TS + e] = y.x;
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
        for (int r = 0; r < x.rows; r++) {
            const int64_t to = (int64_t)__shfl(rk.tok, r, 64) * a.hq + __shfl(rk.head, r, 64);
            for (int e = lane; e < a.d; e += 64) {
                const float y = tile[r * TS + e];
                if (x.whole)
                    st<DT>(a.o, to * a.d + e, y);
                else
                    l.o[(place + r) * a.d + e] = y;
            }
        }
        __builtin_amdgcn_wave_barrier();
        p = next;
        if (p >= end || !walk_on(a, l, walk, next)) break;
    }
}

// The pieces of a shared tile joined, a wavefront a row: the largest reference, then the outputs and sums by it, in
// the order of the workers.
template <int DT>
__global__ __launch_bounds__(256) void paged_join(PagedArgs a, PagedLine l) {
    const PagedJob job = l.jobs[blockIdx.x];
    const int lane = threadIdx.x & 63, r = blockIdx.y * 4 + uni(threadIdx.x >> 6);
    if (r >= job.rows) return;
    const int n = job.last - job.first + 1;
    auto place = [&](int i) { return (int64_t)(2 * (job.first + i) + (i == 0 ? 1 : 0)) * l.pitch + r; };
    float top = -INFINITY;
    for (int i = lane; i < n; i += 64) top = fmaxf(top, l.ml[place(i)].x);
    top = wave_max(top);
    float sum = 0.f, acc[4] = {};
    for (int i0 = 0; i0 < n; i0 += 64) {
        const float2 ml = i0 + lane < n ? l.ml[place(i0 + lane)] : make_float2(-INFINITY, 0.f);
        const float f = ml.x == top ? 1.f : fast_exp2(ml.x - top), s = ml.y * f;
        for (int i = 0; i < min(64, n - i0); i++) {
            const float y = __shfl(s, i, 64), g = __shfl(f, i, 64);
            if (__shfl(ml.y, i, 64) == 0.f) continue;  // (no key of the piece has a weight)
            sum += y;
            const float *o = l.o + place(i0 + i) * a.d;
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (lane + 64 * u < a.d) acc[u] += g * o[lane + 64 * u];
        }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int32_t i = r / job.per;
    const int64_t row = (int64_t)(job.tok + i) * a.hq + job.head + (r - i * job.per);
#pragma unroll
    for (int u = 0; u < 4; u++)
        if (lane + 64 * u < a.d) st<DT>(a.o, row * a.d + lane + 64 * u, acc[u] * inv);
    if (lane == 0 && a.lse) a.lse[row] = lse_of(top, sum);
}

// ------------------------------------------------------------------------------------------
// The weights that the cached keys get
// ------------------------------------------------------------------------------------------
//
// weights[s, j] += sum over the tokens and heads that see key j of e^(scale q k_j - lse). A wavefront takes 32 keys
// of a sequence and goes through every head's rows that see any of them, 32 at a time: S = q K^T, whose columns are
// the keys, so that a key's sum stays in its lane and no other wavefront adds to it.
template <int DT, int DP>
__global__ __launch_bounds__(256) void paged_weights_simple(PagedArgs a, const void *__restrict__ q,
                                                            const void *__restrict__ k, float *__restrict__ weights,
                                                            int64_t stride) {
    constexpr int HALF = DP / 2;
    const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
    const int32_t nw = gridDim.x * 4, mine = uni(blockIdx.x * 4 + (threadIdx.x >> 6));
    const float qscale = a.scale * kLog2e;
    int32_t base = 0;  // (the 32-key blocks of the sequences in front, modulo nw)
    for (int32_t s = 0; s < a.S; s++) {
        const PagedSeq sq = paged_seq(a, s);
        const int32_t blocks = sq.n > 0 ? (sq.len + 31) / 32 : 0;
        const int32_t p0 = sq.len - sq.n;
        for (int32_t b = (mine - base + nw) % nw; b < blocks; b += nw) {
            const int32_t j0 = b * 32, key = j0 + col;
            int64_t off = -1;
            if (key < sq.len) {
                const int64_t e = key / a.page_size, r = key - e * a.page_size, pg = a.table[s * a.max_pages + e];
                if (pg >= 0 && pg < a.num_pages) off = pg * a.kb + r * a.kt;
            }
            // the tokens that see any of the keys
            const int32_t t0 = max(0, j0 - p0);
            const int32_t t1 = a.left >= 0 ? (int32_t)min((int64_t)sq.n, (int64_t)j0 + 32 + a.left - p0) : sq.n;
            float total = 0.f;
            for (int32_t kh = 0; kh < a.hkv && t0 < t1; kh++) {
                float kf[HALF];
#pragma unroll
                for (int e = 0; e < HALF; e++) {
                    const int c = half * HALF + e;
                    kf[e] = off >= 0 && c < a.d ? ld<DT>(k, off + kh * a.kh + c) : 0.f;
                }
                const int64_t r1 = (int64_t)t1 * a.rep;
                for (int64_t r0 = (int64_t)t0 * a.rep; r0 < r1; r0 += 32) {
                    const int64_t r = r0 + col;
                    const bool on = r < r1;
                    const int32_t i = on ? (int32_t)(r / a.rep) : t0, h = on ? (int32_t)(r - (int64_t)i * a.rep) : 0;
                    const int64_t tok = sq.first + i, row = tok * a.qt + (kh * a.rep + h) * a.qh;
                    const float ls = on ? a.lse[tok * a.hq + kh * a.rep + h] : -INFINITY;
                    const float ref = ls * kLog2e;
                    f32x16_t sc = zero16();
#pragma unroll
                    for (int e = 0; e < HALF; e++) {
                        const int c = half * HALF + e;
                        sc = mfma2(on && c < a.d ? ld<DT>(q, row + c) : 0.f, kf[e], sc);
                    }
#pragma unroll
                    for (int u = 0; u < 16; u++) {
                        const int x = crow(u, lane);
                        const float rf = __shfl(ref, x, 64);
                        const int32_t pos = p0 + __shfl(i, x, 64);
                        const bool seen = rf != -INFINITY && key <= pos && (a.left < 0 || key >= pos - a.left);
                        total += seen ? fast_exp2(sc[u] * qscale - rf) : 0.f;
                    }
                }
            }
            total += __shfl_xor(total, 32, 64);
            if (half == 0 && key < sq.len && t0 < t1) weights[s * stride + key] += total;
        }
        base = (int32_t)(((int64_t)base + blocks) % nw);
    }
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

struct PagedPlan {
    PagedLine line;
    size_t bytes;
    size_t lse;  // where the weights' own log-sum-exps lie
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
static PagedPlan paged_plan(const dm_attention_desc *d, char *base, bool weights) {
    PagedPlan p{};
    p.line = line_of(d, 32, 0, INT32_MAX);
    p.line.workers = d->d > 128 ? 1024 : 2048;
    p.line.unit = 32;
    p.line.start = 64;
    p.line.least = 192;
    p.bytes = place_line(d, &p.line, base, 0);
    p.lse = p.bytes;
    if (weights) p.bytes += align_up((size_t)(d->tq * d->hq) * sizeof(float));
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
    return paged_plan(d, nullptr, weights != 0).bytes;
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
    const PagedPlan p = paged_plan(d, (char *)workspace, weights != nullptr);
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
    a.o = o;
    a.lse = lse ? lse : (weights ? (float *)((char *)workspace + p.lse) : nullptr);
    // (four elements at a time where rows and bases allow it)
    const int64_t eb = dtype_bytes(d->dtype);
    const bool vec = ((d->d | a.kb | a.kt | a.kh | a.vb | a.vt | a.vh) & 3) == 0 &&
                     (((uintptr_t)k_pages | (uintptr_t)v_pages) & (4 * eb - 1)) == 0;
    const PagedLine &l = p.line;
    const unsigned g = l.workers / 4;
#define PAGED_V(DT, DP)                                                              \
    if (vec)                                                                         \
        paged_simple<DT, DP, 4><<<g, 256, 0, st>>>(a, l, q, k_pages, v_pages);       \
    else                                                                             \
        paged_simple<DT, DP, 1><<<g, 256, 0, st>>>(a, l, q, k_pages, v_pages);       \
    paged_join<DT><<<dim3(l.workers, (l.pitch + 3) / 4), 256, 0, st>>>(a, l);        \
    if (weights) paged_weights_simple<DT, DP><<<1024, 256, 0, st>>>(a, q, k_pages, weights, weights_stride)
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
    probe_add(DM_PROBE_ATTN_PAGED);
    if (weights) probe_add(DM_PROBE_ATTN_WEIGHTS);
    DM_LAUNCH_CHECK("attention_paged: launch");
    return DM_OK;
}

}  // extern "C"
