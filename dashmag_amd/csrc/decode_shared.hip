// Paged decode for a batch whose sequences share prefixes: groups of rows hold the same first keys,
// which are read once for the group.
//
// With q_r the query of row r (a member and one of the query heads of a key-value head) and the keys
// split into ranges s, softmax(q K^T) V = sum_s e^(L_s - L) O_s with O_s and L_s = log sum e^(q K_s^T) of a
// range alone and L the log-sum-exp of the L_s. So the keys of a group's prefix are ranges of their
// own, taken by all rows of the group together, and a row's own keys behind the prefix are ranges
// that it takes alone; decode_shared_merge joins them.
//
// A workgroup takes one range of keys for a tile of rows of one key-value head. The ranges are cut on
// the device, evenly over the keys that there are, so the grid needs no length on the host and a
// call reads nothing back. A call whose groups do not go up runs with every row's keys its own.
#include <algorithm>
#include <string>

#include "attention_kernels.h"
#include "dm_common.h"
#include "mfma.h"

namespace dm {

struct SharedArgs {
    int64_t B, S, left;
    int32_t hq, hkv, d, rep;
    float scale;
    const int32_t *lengths, *groups, *prefix, *block_table;
    int32_t ngroups;
    int64_t page_size, max_pages, num_pages;
    int64_t qb, qh, kb, kt, kh, vb, vt, vh;
    int32_t nsp, nso;     // ranges of a prefix, and of a row's own keys
    int64_t ptiles;       // prefix tiles of a key-value head (an upper bound, see tile_of)
    int32_t otiles;       // tiles of a row's own heads
    float *part_o;        // [B, Hq, nsp + nso, D], each range's output normalised
    float *part_lse;      // [B, Hq, nsp + nso] natural log, -inf for a range without keys (its output unwritten)
};

constexpr int kOwnRows = 32;  // rows of a tile of own keys

__device__ __forceinline__ int64_t clamp_len(const SharedArgs &a, int64_t x) {
    return x < 0 ? 0 : (x > a.S ? a.S : x);
}
__device__ __forceinline__ int64_t len_of(const SharedArgs &a, int64_t m) {
    return a.lengths ? clamp_len(a, a.lengths[m]) : a.S;
}
__device__ __forceinline__ int64_t low_of(const SharedArgs &a, int64_t len) {
    const int64_t lo = a.left >= 0 ? len - 1 - a.left : 0;
    return lo < 0 ? 0 : lo;
}
// The page of key j of sequence m, or -1.
__device__ __forceinline__ int64_t shared_page(const SharedArgs &a, int64_t m, int64_t j) {
    const int64_t pg = a.block_table[m * a.max_pages + j / a.page_size];
    return pg >= 0 && pg < a.num_pages ? pg : -1;
}

// Whether the groups go up from 0 at least to B at most. For the whole workgroup.
__device__ __forceinline__ bool groups_ok(const SharedArgs &a) {
    if (a.ngroups == 0) return false;
    bool ok = true;
    for (int i = threadIdx.x; i < a.ngroups; i += blockDim.x) {
        const int x = a.groups[i], y = a.groups[i + 1];
        ok = ok && x >= 0 && x <= y && y <= a.B;
    }
    return __syncthreads_and(ok);
}

// What a workgroup does: range `slot` of the rows r0 .. r0 + nrow - 1 (row r: member m0 + r / rep, query
// head kh rep + r % rep) over the keys [s0, s1), which lie on `table`'s pages; a member sees those of
// its own range that lie within [base, cap).
struct SharedItem {
    int64_t m0, table, s0, s1, base, cap;
    int32_t r0, nrow, kh, slot;
    bool prefix;
};

struct SharedScratch {
    unsigned long long best[16];
    int32_t least[16];
};

// Fills in the workgroup's item; false: there is nothing to do (its rows' part is another's, or
// none's). unit: the ranges are multiples of this many keys (a multiple of 16). RT: rows of a prefix tile.
template <int RT>
__device__ __forceinline__ bool item_of(const SharedArgs &a, int unit, SharedScratch &sc, SharedItem &it) {
    const bool ok = groups_ok(a);
    int64_t x = blockIdx.x;
    it.kh = (int32_t)(x % a.hkv);
    x /= a.hkv;
    const int64_t np = a.ptiles * a.nsp;
    int64_t lo, hi;
    it.prefix = x < np;
    if (it.prefix) {
        if (!ok) return false;
        const int64_t tile = x % a.ptiles;
        it.slot = (int32_t)(x / a.ptiles);
        // Group g's tiles begin at groups[g] rep / RT + g (rounded down): far enough apart for its
        // rows, whatever the groups' sizes.
        int32_t g0 = 0, g1 = a.ngroups - 1;
        while (g0 < g1) {
            const int32_t mid = (g0 + g1 + 1) >> 1;
            if ((int64_t)a.groups[mid] * a.rep / RT + mid <= tile)
                g0 = mid;
            else
                g1 = mid - 1;
        }
        const int64_t m0 = a.groups[g0], m1 = a.groups[g0 + 1];
        const int64_t first = (tile - (m0 * a.rep / RT + g0)) * RT;
        const int64_t rows = (m1 - m0) * a.rep;
        if (first < 0 || first >= rows) return false;
        it.m0 = m0, it.r0 = (int32_t)first, it.nrow = (int32_t)min((int64_t)RT, rows - first);
        it.base = 0, it.cap = clamp_len(a, a.prefix[g0]);
        // the longest member (the first of them), and the shortest that sees any key
        unsigned long long best = 0;
        int32_t least = INT32_MAX;
        for (int64_t m = m0 + threadIdx.x; m < m1; m += blockDim.x) {
            const int64_t len = len_of(a, m);
            best = max(best, ((unsigned long long)len << 32) | (uint32_t)(0xffffffffu - (uint32_t)m));
            if (len > 0) least = min(least, (int32_t)min(len, (int64_t)INT32_MAX));
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) {
            best = max(best, __shfl_xor(best, o, 64));
            least = min(least, __shfl_xor(least, o, 64));
        }
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) sc.best[wave] = best, sc.least[wave] = least;
        __syncthreads();
        for (int w = 0; w < (int)blockDim.x / 64; w++) best = max(best, sc.best[w]), least = min(least, sc.least[w]);
        __syncthreads();
        it.table = (int64_t)(0xffffffffu - (uint32_t)best);
        const int64_t longest = (int64_t)(best >> 32);
        hi = min(it.cap, longest);
        lo = longest > 0 ? low_of(a, least) : 0;
    } else {
        x -= np;
        const int64_t b = x % a.B;
        x /= a.B;
        const int32_t ot = (int32_t)(x % a.otiles), split = (int32_t)(x / a.otiles);
        it.m0 = it.table = b;
        it.r0 = ot * kOwnRows, it.nrow = min(kOwnRows, a.rep - it.r0);
        it.slot = a.nsp + split;
        it.base = 0, it.cap = a.S;
        bool grouped = false;
        if (ok) {
            const int32_t g = sequence_of(a.groups, a.ngroups, b);
            grouped = b >= a.groups[g] && b < a.groups[g + 1];
            if (grouped) it.base = clamp_len(a, a.prefix[g]);
        }
        if (!grouped && split == 0)  // the prefix's ranges, which no other workgroup writes
            for (int i = threadIdx.x; i < it.nrow * a.nsp; i += blockDim.x)
                a.part_lse[(b * a.hq + it.kh * a.rep + it.r0 + i / a.nsp) * (a.nsp + a.nso) + i % a.nsp] = -INFINITY;
        hi = len_of(a, b);
        lo = max(it.base, low_of(a, hi));
    }
    const int64_t from = lo & ~(int64_t)15, n = it.prefix ? a.nsp : a.nso;
    const int64_t split = it.prefix ? it.slot : it.slot - a.nsp;
    const int64_t each = hi > from ? ((hi - from + n - 1) / n + unit - 1) / unit * unit : 0;
    it.s0 = max(lo, from + split * each);
    it.s1 = min(hi, from + (split + 1) * each);
    if (it.s0 >= it.s1) {
        for (int r = threadIdx.x; r < it.nrow; r += blockDim.x) {
            const int rr = it.r0 + r;
            const int64_t row = (it.m0 + rr / a.rep) * a.hq + it.kh * a.rep + rr % a.rep;
            a.part_lse[row * (a.nsp + a.nso) + it.slot] = -INFINITY;
        }
        return false;
    }
    return true;
}

// Row r of an item (it may be past its rows): its place among the partial results, and the keys of
// the item that it sees.
struct SharedRow {
    int64_t member, part;
    int32_t head;
    int64_t lo, hi;
};
__device__ __forceinline__ SharedRow row_of(const SharedArgs &a, const SharedItem &it, int r) {
    SharedRow w;
    const bool on = r < it.nrow;
    const int rr = it.r0 + (on ? r : 0);
    w.member = it.m0 + rr / a.rep;
    w.head = it.kh * a.rep + rr % a.rep;
    w.part = ((w.member * a.hq + w.head) * (a.nsp + a.nso)) + it.slot;
    const int64_t len = len_of(a, w.member);
    w.lo = max(max(low_of(a, len), it.base), it.s0);
    w.hi = on ? min(min(len, it.cap), it.s1) : 0;
    return w;
}

// The simple form, for every type, head width, page size and stride: 32 rows and 16 keys at a time in
// LDS as f32, eight threads a row, each two of its scores and every eighth column of its output.
constexpr int kGenKeys = 16;
template <int DT>
__global__ __launch_bounds__(256) void decode_shared_generic(SharedArgs a, const void *__restrict__ q,
                                                             const void *__restrict__ k,
                                                             const void *__restrict__ v) {
    __shared__ float qs[32][257], kv[kGenKeys][257], ps[32][kGenKeys + 1];
    __shared__ SharedScratch sc;
    SharedItem it;
    if (!item_of<32>(a, kGenKeys, sc, it)) return;
    const int tid = threadIdx.x, r = tid >> 3, c = tid & 7;
    const SharedRow row = row_of(a, it, r);
    for (int i = tid; i < 32 * a.d; i += 256) {
        const int x = i / a.d, e = i - x * a.d;
        const int rr = it.r0 + (x < it.nrow ? x : 0);
        qs[x][e] = ld<DT>(q, (it.m0 + rr / a.rep) * a.qb + (it.kh * a.rep + rr % a.rep) * a.qh + e) * a.scale;
    }
    float acc[32], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < 32; i++) acc[i] = 0.f;
    for (int64_t j0 = it.s0; j0 < it.s1; j0 += kGenKeys) {
        const int n = (int)min((int64_t)kGenKeys, it.s1 - j0);
        __syncthreads();
        for (int i = tid; i < n * a.d; i += 256) {
            const int x = i / a.d, e = i - x * a.d;
            const int64_t pg = shared_page(a, it.table, j0 + x);
            kv[x][e] = pg >= 0 ? ld<DT>(k, pg * a.kb + (j0 + x) % a.page_size * a.kt + it.kh * a.kh + e) : 0.f;
        }
        __syncthreads();
        float s[2], mx = -INFINITY;
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int x = c + 8 * u;
            const int64_t j = j0 + x;
            s[u] = -INFINITY;
            if (j >= row.lo && j < row.hi) {
                float t = 0.f;
                for (int e = 0; e < a.d; e++) t += qs[r][e] * kv[x][e];
                s[u] = t;
            }
            mx = fmaxf(mx, s[u]);
        }
#pragma unroll
        for (int o = 4; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
        const float mn = fmaxf(m, mx);
        const float alpha = mn == -INFINITY ? 1.f : expf(m - mn);
        m = mn;
        l *= alpha;
#pragma unroll
        for (int u = 0; u < 2; u++) {
            // (a masked key's weight is a marker below zero: what its value holds stays out)
            const int64_t j = j0 + c + 8 * u;
            const bool seen = j >= row.lo && j < row.hi;
            const float p = seen ? expf(s[u] - mn) : 0.f;
            ps[r][c + 8 * u] = seen ? p : -1.f;
            l += p;
        }
        __syncthreads();
        for (int i = tid; i < n * a.d; i += 256) {
            const int x = i / a.d, e = i - x * a.d;
            const int64_t pg = shared_page(a, it.table, j0 + x);
            kv[x][e] = pg >= 0 ? ld<DT>(v, pg * a.vb + (j0 + x) % a.page_size * a.vt + it.kh * a.vh + e) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 32; i++) acc[i] *= alpha;
        for (int x = 0; x < n; x++) {
            const float p = ps[r][x];
            if (p < 0.f) continue;
#pragma unroll
            for (int i = 0; i < 32; i++)
                if (c + 8 * i < a.d) acc[i] += p * kv[x][c + 8 * i];
        }
    }
#pragma unroll
    for (int o = 4; o >= 1; o >>= 1) l += __shfl_xor(l, o, 64);
    if (r >= it.nrow) return;
    // (l is NaN where a score is: the row's result is NaN then, as the softmax's)
    const bool none = l == 0.f;
#pragma unroll
    for (int i = 0; i < 32; i++)
        if (!none && c + 8 * i < a.d) a.part_o[row.part * a.d + c + 8 * i] = acc[i] / l;
    if (c == 0) a.part_lse[row.part] = none ? -INFINITY : m + logf(l);
}

// The ranges of a row joined, a workgroup a row: its four wavefronts take every fourth range each, a
// lane the columns lane, lane + 64, ...; a range of no key is not read.
constexpr int kSharedSplits = 512;  // most ranges of a row
template <int DT>
__global__ __launch_bounds__(256) void decode_shared_merge(SharedArgs a, void *__restrict__ o) {
    __shared__ float w[kSharedSplits], red[4][256], tops[4], sums[4];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = a.nsp + a.nso;
    float mx = -INFINITY;
    bool nan = false;
    for (int s = tid; s < n; s += 256) {
        const float x = a.part_lse[row * n + s];
        w[s] = x;
        nan |= x != x;
        mx = fmaxf(mx, x);
    }
    mx = wave_max(mx);
    if (lane == 0) tops[wave] = mx;
    nan = __syncthreads_or(nan);
    const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    float sum = 0.f;
    for (int s = tid; s < n; s += 256) {
        const float x = w[s] == -INFINITY ? 0.f : (w[s] == top ? 1.f : expf(w[s] - top));
        w[s] = x;
        sum += x;
    }
    sum = wave_sum(sum);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    float acc[4] = {};
    for (int s = wave; s < n; s += 4) {
        if (w[s] == 0.f) continue;
        const float *po = a.part_o + (row * n + s) * a.d;
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (lane + 64 * i < a.d) acc[i] += w[s] * po[lane + 64 * i];
    }
#pragma unroll
    for (int i = 0; i < 4; i++) red[wave][lane + 64 * i] = acc[i];
    __syncthreads();
    if (tid < a.d) {
        const float t = (red[0][tid] + red[1][tid]) + (red[2][tid] + red[3][tid]);
        st<DT>(o, row * a.d + tid, nan ? NAN : (sum > 0.f ? t / sum : 0.f));
    }
}

// The split of a call: ranges of the prefixes and of the rows' own keys, so that there are about
// kSharedTarget workgroups of each kind where the cache is long enough for ranges of 128 keys.
constexpr int64_t kSharedTarget = 1024;
struct SharedPlan {
    int32_t rows;  // rows of a prefix tile
    int64_t ptiles;
    int32_t otiles, nsp, nso;
};
static SharedPlan shared_plan(const dm_attention_desc *d, int64_t ngroups) {
    SharedPlan p{};
    const int64_t rep = d->hq / d->hkv;
    p.rows = 32;
    p.ptiles = ngroups > 0 ? d->b * rep / p.rows + ngroups : 0;
    p.otiles = (int32_t)((rep + kOwnRows - 1) / kOwnRows);
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>(kSharedSplits / 2, (d->tk + 127) / 128));
    auto split = [&](int64_t tiles) {
        return tiles > 0 ? (int32_t)std::min(most, std::max<int64_t>(1, kSharedTarget / tiles)) : 0;
    };
    p.nsp = split(p.ptiles * d->hkv);
    p.nso = split(d->b * p.otiles * d->hkv);
    return p;
}

// sizes whose products below fit 64 bits, and grids of fewer than 2^32 threads
static bool shared_sizes(const dm_attention_desc *d, int64_t ngroups) {
    const int64_t big = (int64_t)1 << 31;
    return d && d->hkv > 0 && d->b >= 0 && d->b < big && d->hq >= 0 && d->hq < 65536 && d->tk >= 0 &&
           d->tk < big && d->d >= 0 && d->d <= 256 && ngroups >= 0 && ngroups < big &&
           (d->b + ngroups) * std::max<int64_t>(d->hq, d->hkv) < ((int64_t)1 << 23);
}

}  // namespace dm

using namespace dm;

extern "C" {

size_t dm_attention_decode_shared_workspace(const dm_attention_desc *d, int64_t page_size, int64_t ngroups) {
    if (!shared_sizes(d, ngroups)) return 0;
    const SharedPlan p = shared_plan(d, ngroups);
    const size_t parts = (size_t)(d->b * d->hq) * (p.nsp + p.nso);
    return align_up(parts * d->d * sizeof(float)) + align_up(parts * sizeof(float));
}

int dm_attention_decode_shared(const dm_attention_desc *d, const void *q, const void *k_pages,
                               const void *v_pages, int64_t num_pages, int64_t page_size,
                               const int32_t *block_table, int64_t max_pages, const int32_t *lengths,
                               const int32_t *groups, int64_t ngroups, const int32_t *prefix_lengths, void *o,
                               void *workspace, size_t workspace_bytes, void *stream) {
    const std::string op("attention_decode_shared");
    if (int rc = check_decode(op.c_str(), d)) return rc;
    if (page_size < 1 || max_pages < 0 || num_pages < 0 || ngroups < 0)
        return refuse(op + ": page_size must be positive, max_pages, num_pages and ngroups not negative");
    if (!shared_sizes(d, ngroups)) return refuse(op + ": more rows, groups or keys than this library takes");
    if (page_size >= ((int64_t)1 << 31) || max_pages >= ((int64_t)1 << 31) || d->tk != max_pages * page_size)
        return refuse(op + ": desc->tk (" + std::to_string(d->tk) + ") must be max_pages * page_size");
    if (d->cu_seqlens_k) return refuse(op + ": a paged cache takes a block table, not cu_seqlens_k");
    if (d->tk > 0 && d->b > 0 && !block_table) return refuse(op + ": the block table is [B, max_pages] int32");
    if (ngroups > 0 && (!groups || !prefix_lengths))
        return refuse(op + ": groups is [G + 1] and the prefix lengths [G], int32");
    if (workspace_bytes < dm_attention_decode_shared_workspace(d, page_size, ngroups))
        return refuse(op + ": the workspace is smaller than dm_attention_decode_shared_workspace");
    hipStream_t st = (hipStream_t)stream;
    const int64_t rows = d->b * d->hq;
    if (rows == 0 || d->d == 0) return DM_OK;
    if (d->tk == 0) {
        fill_zero(o, rows * d->d * dtype_bytes(d->dtype), st);
        DM_LAUNCH_CHECK("attention_decode_shared: fill");
        return DM_OK;
    }
    const SharedPlan p = shared_plan(d, ngroups);
    SharedArgs a{};
    a.B = d->b, a.S = d->tk, a.left = left_of(d);
    a.hq = (int32_t)d->hq, a.hkv = (int32_t)d->hkv, a.d = (int32_t)d->d, a.rep = (int32_t)(d->hq / d->hkv);
    a.scale = scale_of(d);
    a.lengths = lengths, a.groups = groups, a.prefix = prefix_lengths, a.block_table = block_table;
    a.ngroups = (int32_t)ngroups;
    a.page_size = page_size, a.max_pages = max_pages, a.num_pages = num_pages;
    if (d->strided) {
        a.qb = d->sq.b, a.qh = d->sq.h;
        a.kb = d->sk.b, a.kt = d->sk.t, a.kh = d->sk.h;
        a.vb = d->sv.b, a.vt = d->sv.t, a.vh = d->sv.h;
    } else {
        const int64_t row = d->hkv * d->d;
        a.qb = d->hq * d->d, a.qh = d->d;
        a.kb = a.vb = page_size * row, a.kt = a.vt = row, a.kh = a.vh = d->d;
    }
    a.nsp = p.nsp, a.nso = p.nso, a.ptiles = p.ptiles, a.otiles = p.otiles;
    const size_t parts = (size_t)rows * (p.nsp + p.nso);
    a.part_o = (float *)workspace;
    a.part_lse = (float *)((char *)workspace + align_up(parts * d->d * sizeof(float)));
    const int64_t grid = (p.ptiles * p.nsp + d->b * p.otiles * p.nso) * d->hkv;
#define SHARED_GEN(DT)                                                                \
    decode_shared_generic<DT><<<(unsigned)grid, 256, 0, st>>>(a, q, k_pages, v_pages); \
    decode_shared_merge<DT><<<(unsigned)rows, 256, 0, st>>>(a, o)
    if (d->dtype == DM_F32) {
        SHARED_GEN(DM_F32);
    } else if (d->dtype == DM_BF16) {
        SHARED_GEN(DM_BF16);
    } else {
        SHARED_GEN(DM_F16);
    }
#undef SHARED_GEN
    probe_add(DM_PROBE_DECODE_SHARED);
    DM_LAUNCH_CHECK("attention_decode_shared: launch");
    return DM_OK;
}

}  // extern "C"
