// Norms of queries and keys for each head with the position rotation in the same pass, the
// gradients of both, and the form that writes keys and values into a cache's pages.
//
// A head x of a token at position p, all in f32 and rounded once:
//   r = (mean(x^2) + eps)^-1/2,  y = x r w,  pairs (a, b) of y's first 2 n values -> (a c - b s, a s + b c)
// with c, s of p inv_freq[j]. Backward, z the output's gradient: u = z turned back,
//   dw += u x r,  dx = r (g - x r^2 mean(g x)) with g = u w.
// The angle is p inv_freq[j] / 2 pi in turns, in 64 bits, and only its fractional part goes on in
// f32: in 32 bits the product itself is off by up to p 2^-24, a sixteenth of a radian a million
// positions out.
//
// Bandwidth-bound: every head is read once and written once.
#include <algorithm>
#include <string>

#include "attention_kernels.h"
#include "dm_common.h"
#include "mfma.h"

namespace dm {

// What the kernels take of a call.
struct RopeArgs {
    int64_t tokens, T;  // B x T tokens; a token's batch row is token / T
    int32_t hq, hkv, d, n;
    int32_t weight_dtype, interleaved;
    float eps, unit;  // unit: 1 with unit_offset
    const void *positions;
    int32_t positions_i64;
    int64_t positions_b;
    const void *wq, *wk;
    const float *inv_freq;
    Strd q, k, v, gq, gk;
};
struct RopePages {
    int64_t num_pages, page_size, max_pages;
    int32_t nseq;
    const int32_t *block_table, *lengths, *cu;
    Strd k, v;
};
enum { kRopeFwd = 0, kRopePaged = 1 };

// cos and sin of position p times the frequency.
__device__ __forceinline__ float2 turn_of(int64_t p, float freq) {
    const double t = (double)p * ((double)freq * 0.15915494309189533577);
    float s, c;
    sincospif((float)(t - rint(t)) * 2.f, &s, &c);
    return make_float2(c, s);
}

// The token's position, and (paged) the first elements of its rows in the pages, -1 where it writes
// none; false for a token of no sequence or of a position below zero.
__device__ __forceinline__ bool place_paged(const RopePages &pg, int64_t token, int64_t *p, int64_t *krow,
                                            int64_t *vrow) {
    *krow = *vrow = -1;
    *p = 0;
    int32_t s;
    int64_t after = 0;
    if (pg.cu) {
        if (pg.nseq <= 0) return false;
        s = sequence_of(pg.cu, pg.nseq, token);
        const int64_t end = pg.cu[s + 1];
        if (token < pg.cu[s] || token >= end) return false;
        after = end - 1 - token;
    } else {
        s = (int32_t)token;
    }
    *p = (int64_t)pg.lengths[s] - 1 - after;
    if (*p < 0) {
        *p = 0;
        return false;
    }
    const int64_t at = *p / pg.page_size, row = *p - at * pg.page_size;
    if (at < pg.max_pages) {
        const int64_t page = pg.block_table[s * pg.max_pages + at];
        if (page >= 0 && page < pg.num_pages) {
            *krow = page * pg.k.b + row * pg.k.t;
            *vrow = page * pg.v.b + row * pg.v.t;
        }
    }
    return true;
}

__device__ __forceinline__ int64_t place_plain(const RopeArgs &a, int64_t b, int64_t t) {
    if (!a.positions) return t;
    const int64_t i = b * a.positions_b + t;
    return a.positions_i64 ? ((const int64_t *)a.positions)[i] : (int64_t)((const int32_t *)a.positions)[i];
}

// A head's pair index and partner of element e (e < 2 n), and whether e is the pair's first.
__device__ __forceinline__ void pair_of(int e, int n, int interleaved, int *j, int *other, bool *first) {
    if (interleaved) {
        *j = e >> 1, *other = e ^ 1, *first = !(e & 1);
    } else {
        *first = e < n;
        *j = *first ? e : e - n;
        *other = *first ? e + n : e - n;
    }
}

// The simple forms, for any width, alignment and number of pairs: a wavefront takes a head, four
// elements 64 apart in a lane, and finds a pair's other element in the wavefront's row of LDS.
template <int DT, int MODE>
__global__ __launch_bounds__(256) void rope_generic(RopeArgs a, RopePages pg, const void *__restrict__ q,
                                                    const void *__restrict__ k, const void *__restrict__ v,
                                                    void *__restrict__ qo, void *__restrict__ ko,
                                                    void *__restrict__ vo) {
    __shared__ float rows[4][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float *row = rows[wave];
    const int heads = a.hq + a.hkv * (MODE == kRopePaged ? 2 : 1);
    const int64_t total = a.tokens * heads;
    const int64_t each = (int64_t)gridDim.x * 4;
    // (every wavefront makes the same number of rounds: the barriers below are the workgroup's)
    for (int64_t base = (int64_t)blockIdx.x * 4; base < total; base += each) {
        const int64_t w = base + wave;
        const bool on = w < total;
        const int64_t token = on ? w / heads : 0;
        const int h = on ? (int)(w - token * heads) : 0;
        const int64_t b = token / a.T, t = token - b * a.T;
        int64_t p, krow = -1, vrow = -1;
        bool is = true;
        if (MODE == kRopePaged)
            is = place_paged(pg, token, &p, &krow, &vrow);
        else
            p = place_plain(a, b, t);
        if (MODE == kRopePaged && h >= a.hq + a.hkv) {  // a value head: as it is
            const int hv = h - a.hq - a.hkv;
            if (on && is && vrow >= 0)
                for (int e = lane; e < a.d; e += 64)
                    st<DT>(vo, vrow + hv * pg.v.h + e, ld<DT>(v, b * a.v.b + t * a.v.t + hv * a.v.h + e));
        }
        const bool isq = h < a.hq;
        const int hh = isq ? h : h - a.hq;
        const bool head = on && h < a.hq + a.hkv;
        const void *src = isq ? q : k;
        const Strd sd = isq ? a.q : a.k;
        const void *wt = isq ? a.wq : a.wk;
        const int64_t from = b * sd.b + t * sd.t + hh * sd.h;
        float x[4], ss = 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int e = lane + 64 * i;
            x[i] = head && e < a.d ? ld<DT>(src, from + e) : 0.f;
            ss += x[i] * x[i];
        }
        const float r = rsqrtf(wave_sum(ss) / a.d + a.eps);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int e = lane + 64 * i;
            const float wv = wt && e < a.d ? ld_any(a.weight_dtype, wt, e) + a.unit : 1.f;
            x[i] *= r * wv;
            row[e] = x[i];
        }
        __syncthreads();
        if (!head || (MODE == kRopePaged && !isq && krow < 0)) continue;
        void *dst = isq ? qo : ko;
        const int64_t to = isq ? (token * a.hq + hh) * a.d
                               : (MODE == kRopePaged ? krow + hh * pg.k.h : (token * a.hkv + hh) * a.d);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int e = lane + 64 * i;
            if (e >= a.d) continue;
            float y = x[i];
            if (e < 2 * a.n) {
                int j, other;
                bool first;
                pair_of(e, a.n, a.interleaved, &j, &other, &first);
                const float2 cs = turn_of(p, a.inv_freq[j]);
                y = first ? y * cs.x - row[other] * cs.y : row[other] * cs.y + y * cs.x;
            }
            st<DT>(dst, to + e, MODE == kRopePaged && !is ? 0.f : y);
        }
    }
}

// The gradients of the simple form. A wavefront's heads all add to the same four elements of a
// lane; the workgroup's sums go to parts [workgroups][2][D] and rope_weights adds those in order.
template <int DT>
__global__ __launch_bounds__(256) void rope_bwd_generic(RopeArgs a, const void *__restrict__ q,
                                                        const void *__restrict__ k,
                                                        const void *__restrict__ gq,
                                                        const void *__restrict__ gk, void *__restrict__ dq,
                                                        void *__restrict__ dk, float *__restrict__ parts) {
    __shared__ float rows[4][256], sums[4][2][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float *row = rows[wave];
    const int heads = a.hq + a.hkv;
    const int64_t total = a.tokens * heads;
    const int64_t each = (int64_t)gridDim.x * 4;
    float dw[2][4] = {};
    for (int64_t base = (int64_t)blockIdx.x * 4; base < total; base += each) {
        const int64_t w = base + wave;
        const bool on = w < total;
        const int64_t token = on ? w / heads : 0;
        const int h = on ? (int)(w - token * heads) : 0;
        const int64_t b = token / a.T, t = token - b * a.T, p = place_plain(a, b, t);
        const bool isq = h < a.hq;
        const int hh = isq ? h : h - a.hq;
        const void *src = isq ? q : k, *grad = isq ? gq : gk, *wt = isq ? a.wq : a.wk;
        const Strd sd = isq ? a.q : a.k, sg = isq ? a.gq : a.gk;
        const int64_t from = b * sd.b + t * sd.t + hh * sd.h, gfrom = b * sg.b + t * sg.t + hh * sg.h;
        float x[4], z[4], ss = 0.f;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int e = lane + 64 * i;
            x[i] = on && e < a.d ? ld<DT>(src, from + e) : 0.f;
            z[i] = on && e < a.d ? ld<DT>(grad, gfrom + e) : 0.f;
            ss += x[i] * x[i];
            row[e] = z[i];
        }
        const float r = rsqrtf(wave_sum(ss) / a.d + a.eps);
        __syncthreads();
        float gx = 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int e = lane + 64 * i;
            if (e < 2 * a.n) {
                int j, other;
                bool first;
                pair_of(e, a.n, a.interleaved, &j, &other, &first);
                const float2 cs = turn_of(p, a.inv_freq[j]);
                z[i] = first ? z[i] * cs.x + row[other] * cs.y : z[i] * cs.x - row[other] * cs.y;
            }
            const float add = on ? z[i] * (x[i] * r) : 0.f;
            if (isq)
                dw[0][i] += add;
            else
                dw[1][i] += add;
            z[i] *= wt && e < a.d ? ld_any(a.weight_dtype, wt, e) + a.unit : 1.f;
            gx += z[i] * (x[i] * r);
        }
        const float mean = wave_sum(gx) / a.d;
        void *dst = isq ? dq : dk;
        const int64_t to = (token * (isq ? a.hq : a.hkv) + hh) * a.d;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int e = lane + 64 * i;
            if (on && e < a.d) st<DT>(dst, to + e, r * (z[i] - x[i] * r * mean));
        }
    }
#pragma unroll
    for (int x = 0; x < 2; x++)
#pragma unroll
        for (int i = 0; i < 4; i++) sums[wave][x][lane + 64 * i] = dw[x][i];
    __syncthreads();
    for (int e = threadIdx.x; e < 2 * a.d; e += 256) {
        const int x = e / a.d, c = e - x * a.d;
        parts[(int64_t)blockIdx.x * 2 * a.d + e] =
            (sums[0][x][c] + sums[1][x][c]) + (sums[2][x][c] + sums[3][x][c]);
    }
}

// The workgroups' weight gradients added in order: a workgroup takes 16 columns, its 16 groups of
// threads every sixteenth part each.
__global__ __launch_bounds__(256) void rope_weights(const float *__restrict__ parts, int64_t nparts, int d,
                                                    int weight_dtype, void *dwq, void *dwk) {
    __shared__ float sums[16][17];
    const int c = threadIdx.x & 15, g = threadIdx.x >> 4;
    const int64_t col = (int64_t)blockIdx.x * 16 + c;
    float s = 0.f;
    if (col < 2 * d)
        for (int64_t i = g; i < nparts; i += 16) s += parts[i * 2 * d + col];
    sums[g][c] = s;
    __syncthreads();
    if (g == 0 && col < 2 * d) {
        float t = 0.f;
        for (int i = 0; i < 16; i++) t += sums[i][c];
        void *to = col < d ? dwq : dwk;
        if (to) st_any(weight_dtype, to, col < d ? col : col - d, t);
    }
}

constexpr int64_t kRopeParts = 1024;  // workgroups of the backward at most

static int64_t bwd_workgroups(const dm_qk_norm_rope_desc *d) {
    const int64_t tokens = d->b * d->t;
    return std::max<int64_t>(1, std::min(tokens, kRopeParts));
}

static Strd strd(const dm_strides &s) { return Strd{s.b, s.t, s.h}; }

// sizes that products of them cannot overflow
static bool sane(int64_t x) { return x >= 0 && x < ((int64_t)1 << 31); }

static int check_rope(const std::string &op, const dm_qk_norm_rope_desc *d) {
    if (!d) return refuse(op + ": null descriptor");
    if (!sane(d->b) || !sane(d->t) || d->hq < 0 || d->hkv < 0 || d->d < 0 || d->hq > 65536 || d->hkv > 65536 ||
        (d->t > 0 && d->b > (((int64_t)1 << 40) / d->t)))
        return refuse(op + ": bad dimensions");
    if (d->d > 256) return refuse(op + ": head dimension above 256 is not implemented");
    if (d->n < 0 || 2 * d->n > d->d)
        return refuse(op + ": the frequencies are [n] with 2 n at most the head dimension (" +
                      std::to_string(d->d) + "), got n = " + std::to_string(d->n));
    if (d->dtype != DM_F32 && d->dtype != DM_BF16 && d->dtype != DM_F16)
        return refuse(op + ": dtype must be f32, bf16 or f16");
    if (d->weight_dtype != DM_F32 && d->weight_dtype != d->dtype)
        return refuse(op + ": the weights must be f32 or the queries' dtype");
    if (!(d->eps >= 0.f)) return refuse(op + ": eps must not be negative");
    if (d->positions_b < 0) return refuse(op + ": strides must not be negative");
    if (d->strided && !(strides_ok(strd(d->sq)) && strides_ok(strd(d->sk)) && strides_ok(strd(d->sv)) &&
                        strides_ok(strd(d->sgq)) && strides_ok(strd(d->sgk))))
        return refuse(op + ": strides must not be negative");
    return DM_OK;
}

static RopeArgs rope_args(const dm_qk_norm_rope_desc *d, const void *wq, const void *wk, const float *freq) {
    RopeArgs a{};
    a.tokens = d->b * d->t, a.T = d->t;
    a.hq = (int32_t)d->hq, a.hkv = (int32_t)d->hkv, a.d = (int32_t)d->d, a.n = (int32_t)d->n;
    a.weight_dtype = d->weight_dtype, a.interleaved = d->interleaved != 0;
    a.eps = d->eps, a.unit = d->unit_offset ? 1.f : 0.f;
    a.positions = d->positions, a.positions_i64 = d->positions_i64, a.positions_b = d->positions_b;
    a.wq = wq, a.wk = wk, a.inv_freq = freq;
    const Strd cq{d->t * d->hq * d->d, d->hq * d->d, d->d}, ck{d->t * d->hkv * d->d, d->hkv * d->d, d->d};
    a.q = a.gq = cq, a.k = a.gk = a.v = ck;
    if (d->strided)
        a.q = strd(d->sq), a.k = strd(d->sk), a.v = strd(d->sv), a.gq = strd(d->sgq), a.gk = strd(d->sgk);
    return a;
}

template <int MODE>
static int run_rope(const char *op, const dm_qk_norm_rope_desc *d, const RopeArgs &a, const RopePages &pg,
                    const void *q, const void *k, const void *v, void *qo, void *ko, void *vo,
                    hipStream_t st) {
    const int64_t rows = a.tokens * (a.hq + a.hkv * (MODE == kRopePaged ? 2 : 1));
    const unsigned grid = (unsigned)std::min<int64_t>((rows + 3) / 4, 16384);
    if (d->dtype == DM_F32)
        rope_generic<DM_F32, MODE><<<grid, 256, 0, st>>>(a, pg, q, k, v, qo, ko, vo);
    else if (d->dtype == DM_BF16)
        rope_generic<DM_BF16, MODE><<<grid, 256, 0, st>>>(a, pg, q, k, v, qo, ko, vo);
    else
        rope_generic<DM_F16, MODE><<<grid, 256, 0, st>>>(a, pg, q, k, v, qo, ko, vo);
    probe_add(DM_PROBE_QK_NORM_ROPE);
    DM_LAUNCH_CHECK((std::string(op) + ": launch").c_str());
    return DM_OK;
}

}  // namespace dm

using namespace dm;

extern "C" {

int dm_qk_norm_rope(const dm_qk_norm_rope_desc *d, const void *q, const void *k, const void *q_weight,
                    const void *k_weight, const float *inv_freq, void *q_out, void *k_out, void *stream) {
    const char *op = "qk_norm_rope";
    if (int rc = check_rope(op, d)) return rc;
    if (d->b * d->t * (d->hq + d->hkv) == 0 || d->d == 0) return DM_OK;
    return run_rope<kRopeFwd>(op, d, rope_args(d, q_weight, k_weight, inv_freq), RopePages{}, q, k, nullptr,
                              q_out, k_out, nullptr, (hipStream_t)stream);
}

size_t dm_qk_norm_rope_bwd_workspace(const dm_qk_norm_rope_desc *d) {
    if (!d || d->d <= 0 || d->d > 256 || !sane(d->b) || !sane(d->t)) return 0;
    return align_up((size_t)kRopeParts * 2 * d->d * sizeof(float));
}

int dm_qk_norm_rope_bwd(const dm_qk_norm_rope_desc *d, const void *q, const void *k, const void *q_weight,
                        const void *k_weight, const float *inv_freq, const void *grad_q, const void *grad_k,
                        void *dq, void *dk, void *dq_weight, void *dk_weight, void *workspace,
                        size_t workspace_bytes, void *stream) {
    const std::string op("qk_norm_rope_backward");
    if (int rc = check_rope(op, d)) return rc;
    if (workspace_bytes < dm_qk_norm_rope_bwd_workspace(d))
        return refuse(op + ": the workspace is smaller than dm_qk_norm_rope_bwd_workspace");
    if (d->d == 0) return DM_OK;
    hipStream_t st = (hipStream_t)stream;
    const RopeArgs a = rope_args(d, q_weight, k_weight, inv_freq);
    float *parts = (float *)workspace;
    const int64_t nparts = a.tokens * (a.hq + a.hkv) > 0 ? bwd_workgroups(d) : 0;
    if (nparts > 0) {
        if (d->dtype == DM_F32)
            rope_bwd_generic<DM_F32><<<(unsigned)nparts, 256, 0, st>>>(a, q, k, grad_q, grad_k, dq, dk, parts);
        else if (d->dtype == DM_BF16)
            rope_bwd_generic<DM_BF16><<<(unsigned)nparts, 256, 0, st>>>(a, q, k, grad_q, grad_k, dq, dk, parts);
        else
            rope_bwd_generic<DM_F16><<<(unsigned)nparts, 256, 0, st>>>(a, q, k, grad_q, grad_k, dq, dk, parts);
    }
    if (dq_weight || dk_weight)
        rope_weights<<<(unsigned)((2 * a.d + 15) / 16), 256, 0, st>>>(parts, nparts, a.d, a.weight_dtype,
                                                                      dq_weight, dk_weight);
    probe_add(DM_PROBE_QK_NORM_ROPE_BWD);
    DM_LAUNCH_CHECK((op + ": launch").c_str());
    return DM_OK;
}

int dm_qk_norm_rope_paged(const dm_qk_norm_rope_desc *d, const dm_kv_pages *pages, const void *q,
                          const void *k, const void *v, const void *q_weight, const void *k_weight,
                          const float *inv_freq, void *q_out, void *k_pages, void *v_pages, void *stream) {
    const std::string op("qk_norm_rope_paged");
    if (int rc = check_rope(op, d)) return rc;
    if (!pages) return refuse(op + ": null pages");
    if (d->b != 1) return refuse(op + ": the tokens lie along the time, B = 1");
    if (pages->page_size < 1 || !sane(pages->page_size) || !sane(pages->num_pages) || !sane(pages->max_pages) ||
        !sane(pages->nseq))
        return refuse(op + ": page_size must be positive, num_pages, max_pages and nseq not negative");
    if (!strides_ok(strd(pages->sk)) || !strides_ok(strd(pages->sv)))
        return refuse(op + ": strides must not be negative");
    if (!pages->cu_seqlens && pages->nseq != d->t)
        return refuse(op + ": without cu_seqlens there is one token a sequence, got " + std::to_string(d->t) +
                      " tokens and " + std::to_string(pages->nseq) + " sequences");
    if (pages->nseq > 0 && (!pages->lengths || (pages->max_pages > 0 && !pages->block_table)))
        return refuse(op + ": the block table is [S, max_pages] and the lengths [S], int32");
    if (d->t * (d->hq + d->hkv) == 0 || d->d == 0) return DM_OK;
    RopePages pg{};
    pg.num_pages = pages->num_pages, pg.page_size = pages->page_size, pg.max_pages = pages->max_pages;
    pg.nseq = (int32_t)pages->nseq;
    pg.block_table = pages->block_table, pg.lengths = pages->lengths, pg.cu = pages->cu_seqlens;
    pg.k = strd(pages->sk), pg.v = strd(pages->sv);
    return run_rope<kRopePaged>(op.c_str(), d, rope_args(d, q_weight, k_weight, inv_freq), pg, q, k, v, q_out,
                                k_pages, v_pages, (hipStream_t)stream);
}

}  // extern "C"
