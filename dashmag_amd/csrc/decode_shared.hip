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

// ------------------------------------------------------------------------------------------
// The 16-bit kernel (D = 64, 128 or 256, pages of a multiple of 16 keys)
// ------------------------------------------------------------------------------------------
//
// Both products run on MFMA: S^T = K q^T (keys x 32 rows) and O^T += V^T P^T, S^T's output layout being
// P^T's operand. The weights are rounded to the inputs' type for the second product, as the other
// attention kernels do; sums, maxima and outputs stay in f32.
//
// NARROW items (a row's own keys; the prefix of a group of few rows): the keys are what there is to
// share out, so each wavefront sweeps keys of its own in blocks of 32 through its own LDS tiles, for
// up to 32 rows, and the wavefronts' results are joined in LDS.
//
// WIDE items (the prefix of a group of many rows): the rows are shared out, 32 a wavefront, and all
// sweep the same keys in tiles of 64. Wavefronts w and w + 4 of a SIMD run half a step apart, so
// that one's products and the other's softmax run side by side.
//
// Keys arrive in 16-key blocks, each on one page: a buffer resource of the block's rows up to the
// item's end reads zeros behind it, and a page outside the pages, or in front of the item's start,
// reads as zeros too.

template <int D>
constexpr int shared_waves() { return D == 256 ? 4 : 8; }

// The pages' geometry in 32 bits: byte strides of a row, shifts where the page size is a power of two.
struct PageMap {
    const char *k, *v;  // at the item's key-value head
    const int32_t *table;
    uint32_t kt, vt;    // bytes
    int32_t shift;      // log2 page_size, -1 otherwise
};

// The page of the 16-key block at key j, -1 for none or a block behind `end`.
__device__ __forceinline__ int32_t block_page(const SharedArgs &a, const PageMap &m, int32_t j, int32_t end) {
    if (j >= end) return -1;
    const uint32_t at = m.shift >= 0 ? (uint32_t)j >> m.shift : (uint32_t)j / (uint32_t)a.page_size;
    const int32_t pg = m.table[at];
    return pg >= 0 && pg < a.num_pages ? pg : -1;
}
__device__ __forceinline__ uint32_t row_in_page(const SharedArgs &a, const PageMap &m, int32_t j) {
    return m.shift >= 0 ? (uint32_t)j & ((1u << m.shift) - 1u) : (uint32_t)j % (uint32_t)a.page_size;
}
// The resource of the 16-key block at key j on page pg: its rows in front of `end`.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t block_rsrc(const char *base, int64_t page_bytes, uint32_t row_bytes,
                                                             uint32_t row, int32_t pg, int32_t j, int32_t end) {
    const uint32_t n = (uint32_t)max(0, min(16, end - j));
    return make_rsrc(base + (pg >= 0 ? pg * page_bytes + (int64_t)row * row_bytes : 0), pg >= 0 ? n * row_bytes : 0u);
}

template <int DT>
__device__ __forceinline__ bool not_finite(uint32_t w) {
    constexpr uint32_t e = DT == DM_BF16 ? 0x7f80u : 0x7c00u;
    return (w & e) == e || ((w >> 16) & e) == e;
}
// Values that are not finite taken out of a piece of V (whoever sees them adds them at the end).
template <int DT>
__device__ __forceinline__ bool take_out(uint4 &x) {
    constexpr uint32_t e = DT == DM_BF16 ? 0x7f80u : 0x7c00u;
    bool any = false;
    uint32_t *w = (uint32_t *)&x;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (not_finite<DT>(w[i])) {
            any = true;
            w[i] &= ((w[i] & e) == e ? 0u : 0xffffu) | ((((w[i] >> 16) & e) == e) ? 0u : 0xffff0000u);
        }
    return any;
}

template <int D>
struct SharedSmem {
    static constexpr int NW = shared_waves<D>(), KS = D + 8, VS = D + 32;
    struct Narrow {
        uint16_t k[32 * KS], v[32 * VS];
    };
    struct Wide {
        uint16_t k[2][64 * KS], v[2][64 * VS];
    };
    union {
        Narrow narrow[NW];
        Wide wide;
        float join[NW * 32 * (D + 2)];
    };
    SharedScratch sc;
    int32_t lo[NW], hi[NW], bad;
};

// What the lanes of a wavefront know of their rows: the queries as the second operand, and the keys seen.
template <int D>
struct RowState {
    Frag8 qf[D / 16];
    int32_t lo, hi;    // this lane's row
    int32_t flo, fhi;  // the keys that all of the wavefront's rows see
    bool on;
};

template <int DT, int D>
__device__ __forceinline__ void load_rows(const SharedArgs &a, const SharedItem &it, const void *q, int r,
                                          bool slots, RowState<D> &w) {
    const int half = (threadIdx.x >> 5) & 1;
    const SharedRow row = row_of(a, it, r);
    w.on = r < it.nrow;
    w.lo = (int32_t)row.lo, w.hi = (int32_t)max(row.hi, (int64_t)0);
    const uint16_t *qp = (const uint16_t *)q + row.member * a.qb + (int64_t)row.head * a.qh;
    const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;  // (the softmax below takes a scale above 0)
#pragma unroll
    for (int s = 0; s < D / 16; s++) {
        uint4 x = zero4();
        if (w.on) {
            if (slots) {  // narrow: the slots 4 h + e and 8 + 4 h + e of row_frag
                const uint2 l = *(const uint2 *)(qp + s * 16 + half * 4), u = *(const uint2 *)(qp + s * 16 + 8 + half * 4);
                x = make_uint4(l.x, l.y, u.x, u.y);
            } else {
                x = *(const uint4 *)(qp + s * 16 + half * 8);
            }
        }
        w.qf[s].u = make_uint4(x.x ^ flip, x.y ^ flip, x.z ^ flip, x.w ^ flip);
    }
    int32_t flo = w.on ? w.lo : INT32_MIN, fhi = w.on ? w.hi : INT32_MAX;
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
        flo = max(flo, __shfl_xor(flo, o, 64));
        fhi = min(fhi, __shfl_xor(fhi, o, 64));
    }
    w.flo = __builtin_amdgcn_readfirstlane(flo);
    w.fhi = __builtin_amdgcn_readfirstlane(fhi);
}

// The values that were taken out, added for the rows that see them: every key of [j0, j1) again, one
// at a time (a key that is not finite in a place that some row of the tile does not see).
template <int DT, int D>
__device__ __forceinline__ void add_back(const SharedArgs &a, const PageMap &m, int32_t j0, int32_t j1, int32_t lo,
                                         int32_t hi, f32x16_t (&acc)[D / 32]) {
    const int lane = threadIdx.x & 63;
    for (int32_t j = j0; j < j1; j++) {
        const int32_t pg = block_page(a, m, j & ~15, j1);
        if (pg < 0 || j < lo || j >= hi) continue;
        const uint16_t *row = (const uint16_t *)(m.v + pg * a.vb * 2 + (int64_t)row_in_page(a, m, j) * m.vt);
#pragma unroll
        for (int dt = 0; dt < D / 32; dt++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const uint32_t x = row[dt * 32 + crow(i, lane)];
                if (not_finite<DT>(x)) acc[dt][i] += unpack_lo<DT>(x);
            }
    }
}

// One item's results: unnormalised O^T (this lane's row, the D / 2 columns of its half), the reference m
// (log2 units) and the sum l of this lane's half.
template <int D>
struct Partial {
    f32x16_t acc[D / 32];
    float m, l;
};

template <int DT, int D>
__device__ __forceinline__ void shared_narrow(const SharedArgs &a, const SharedItem &it, const PageMap &map,
                                              const void *q, SharedSmem<D> &sm) {
    constexpr int NW = shared_waves<D>(), KS = SharedSmem<D>::KS, VS = SharedSmem<D>::VS;
    constexpr int LPR = D / 8, RPL = 64 / LPR, NLD = 32 / RPL;  // lanes a row, rows a load, loads
    constexpr int KST = D / 16, DTN = D / 32;
    const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    RowState<D> rs;
    load_rows<DT, D>(a, it, q, col, true, rs);
    const float qscale = fabsf(a.scale) * 1.4426950408889634f;
    const int32_t s0 = (int32_t)it.s0, s1 = (int32_t)it.s1, a0 = s0 & ~15;
    const int32_t per = ((s1 - a0 + NW - 1) / NW + 31) & ~31;
    const int32_t w0 = max(s0, a0 + wave * per), w1 = min(s1, a0 + (wave + 1) * per), b0 = w0 & ~15;
    typename SharedSmem<D>::Narrow &t = sm.narrow[wave];
    uint4 sk[NLD], sv[NLD];
    int32_t pg[2];
    auto pages = [&](int32_t j) __attribute__((always_inline)) {
        pg[0] = block_page(a, map, j, w1);
        pg[1] = block_page(a, map, j + 16, w1);
    };
    auto load = [&](int32_t j0) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int32_t j = j0 + 16 * h;
            const uint32_t row = pg[h] >= 0 ? row_in_page(a, map, j) : 0u;
            const __amdgpu_buffer_rsrc_t kr = block_rsrc(map.k, a.kb * 2, map.kt, row, pg[h], j, w1);
            const __amdgpu_buffer_rsrc_t vr = block_rsrc(map.v, a.vb * 2, map.vt, row, pg[h], j, w1);
#pragma unroll
            for (int u = h * NLD / 2; u < (h + 1) * NLD / 2; u++) {
                const uint32_t r = RPL * u - 16 * h + lane / LPR, c = (lane % LPR) * 16;
                const bool in = j + (int32_t)r >= w0;
                sk[u] = buf_load16_nt(kr, in ? r * map.kt + c : 0xffffffffu);
                sv[u] = buf_load16_nt(vr, in ? r * map.vt + c : 0xffffffffu);
            }
        }
    };
    Partial<D> p;
    p.m = -INFINITY, p.l = 0.f;
#pragma unroll
    for (int dt = 0; dt < DTN; dt++) p.acc[dt] = zero16();
    bool bad = false;
    if (w0 < w1) {
        const int nblk = (w1 - b0 + 31) / 32;
        pages(b0);
        load(b0);
        pages(b0 + 32);
        for (int n = 0; n < nblk; n++) {
            const int32_t j0 = b0 + n * 32;
            const bool cut = j0 < rs.flo || j0 + 32 > rs.fhi;
            if (cut) {
#pragma unroll
                for (int u = 0; u < NLD; u++) bad |= take_out<DT>(sv[u]);
            }
#pragma unroll
            for (int u = 0; u < NLD; u++) {
                const int r = RPL * u + lane / LPR, c = (lane % LPR) * 8;
                *(uint4 *)(t.k + r * KS + c) = sk[u];
                *(uint4 *)(t.v + r * VS + c) = sv[u];
            }
            load(j0 + 32);
            pages(j0 + 64);
            f32x16_t sc = zero16();
#pragma unroll
            for (int st = 0; st < KST; st++) sc = mfma32<DT>(row_frag(t.k, KS, 0, st * 16, lane), rs.qf[st], sc);
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int32_t key = j0 + crow(i, lane);
                sc[i] = !cut || (key >= rs.lo && key < rs.hi) ? sc[i] * qscale : -INFINITY;
                mx = fmaxf(mx, sc[i]);
            }
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            const bool grow = mx > p.m + 8.f;
            if (__any(grow)) {
                const float mn = grow ? mx : p.m;
                const float alpha = mn == -INFINITY ? 1.f : fast_exp2(p.m - mn);
                p.m = mn;
                p.l *= alpha;
#pragma unroll
                for (int dt = 0; dt < DTN; dt++)
#pragma unroll
                    for (int i = 0; i < 16; i++) p.acc[dt][i] *= alpha;
            }
            const float ref = p.m == -INFINITY ? 0.f : p.m;
            float ps = 0.f;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                sc[i] = fast_exp2(sc[i] - ref);
                ps += sc[i];
            }
            p.l += ps;
            const Frag8 p0 = c_frag<DT>(sc, 0), p1 = c_frag<DT>(sc, 1);
#pragma unroll
            for (int dt = 0; dt < DTN; dt++) {
                p.acc[dt] = mfma32<DT>(lds_tr_frag(t.v, VS, 0, dt * 32, lane), p0, p.acc[dt]);
                p.acc[dt] = mfma32<DT>(lds_tr_frag(t.v, VS, 16, dt * 32, lane), p1, p.acc[dt]);
            }
        }
    }
    if (__any(bad)) {
        for (int32_t j0 = b0; j0 < w1; j0 += 32)
            if (j0 < rs.flo || j0 + 32 > rs.fhi)
                add_back<DT, D>(a, map, max(j0, w0), min(j0 + 32, w1), rs.lo, rs.hi, p.acc);
    }
    const float l = p.l + __shfl_xor(p.l, 32, 64);
    // the wavefronts' results joined through LDS: [wave][row][D], their references and sums behind
    __syncthreads();
    float *sa = sm.join, *sm_m = sa + NW * 32 * D, *sm_l = sm_m + NW * 32;
    if (col < it.nrow) {
#pragma unroll
        for (int dt = 0; dt < DTN; dt++)
#pragma unroll
            for (int g4 = 0; g4 < 4; g4++)
                *(float4 *)(sa + (wave * 32 + col) * D + dt * 32 + g4 * 8 + half * 4) =
                    make_float4(p.acc[dt][g4 * 4], p.acc[dt][g4 * 4 + 1], p.acc[dt][g4 * 4 + 2], p.acc[dt][g4 * 4 + 3]);
        if (half == 0) sm_m[wave * 32 + col] = p.m, sm_l[wave * 32 + col] = l;
    }
    __syncthreads();
    for (int x = threadIdx.x; x < it.nrow * (D / 4); x += NW * 64) {
        const int r = x / (D / 4), d = x % (D / 4) * 4;
        float M = -INFINITY;
        for (int w = 0; w < NW; w++) M = fmaxf(M, sm_m[w * 32 + r]);
        float L = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        if (M != -INFINITY)
            for (int w = 0; w < NW; w++) {
                if (sm_m[w * 32 + r] == -INFINITY) continue;
                const float f = fast_exp2(sm_m[w * 32 + r] - M);
                const float4 y = *(const float4 *)(sa + (w * 32 + r) * D + d);
                L += sm_l[w * 32 + r] * f;
                o.x += y.x * f, o.y += y.y * f, o.z += y.z * f, o.w += y.w * f;
            }
        const SharedRow row = row_of(a, it, r);
        if (L != 0.f) {  // (NaN is not 0)
            const float inv = 1.f / L;
            *(float4 *)(a.part_o + row.part * D + d) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
        }
        if (d == 0) a.part_lse[row.part] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
    }
}

template <int DT, int D>
__device__ __forceinline__ void shared_wide(const SharedArgs &a, const SharedItem &it, const PageMap &map,
                                            const void *q, SharedSmem<D> &sm) {
    constexpr int NW = shared_waves<D>(), NT = NW * 64, KS = SharedSmem<D>::KS, VS = SharedSmem<D>::VS;
    constexpr int CPR = D / 8, RPW = 64 / CPR, RSTEP = NT / CPR, NCH = 64 / RSTEP;  // pieces a row, rows a wavefront
    constexpr int KST = D / 16, DTN = D / 32;
    const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool first = NW == 4 || wave < 4;  // products first in each step
    RowState<D> rs;
    load_rows<DT, D>(a, it, q, wave * 32 + col, false, rs);
    // (the queries are waited for here: behind the tiles' loads they would leave a wait for all of
    // those in the loop)
    __builtin_amdgcn_s_waitcnt(0x0F70);
    const bool rows = wave * 32 < it.nrow;  // this wavefront has rows
    if (lane == 0) sm.lo[wave] = rs.flo, sm.hi[wave] = rs.fhi;
    if (threadIdx.x == 0) sm.bad = 0;
    __syncthreads();
    int32_t tlo = INT32_MIN, thi = INT32_MAX;  // the keys that every row of the tile sees
#pragma unroll
    for (int w = 0; w < NW; w++) tlo = max(tlo, sm.lo[w]), thi = min(thi, sm.hi[w]);
    tlo = __builtin_amdgcn_readfirstlane(tlo), thi = __builtin_amdgcn_readfirstlane(thi);
    const int32_t s0 = (int32_t)it.s0, s1 = (int32_t)it.s1, k0 = s0 & ~15;
    const int32_t nt = (s1 - k0 + 63) / 64;
    const float c2 = fabsf(a.scale) * 1.4426950408889634f;

    // staging: NCH pieces of a tile's K and of its V a thread; a wavefront's rows of a piece lie in one
    // 16-key block, whose page is looked up a step before its keys are loaded, and two before its values
    const int wr = wave * RPW, lr = lane / CPR, lc = lane % CPR;
    uint4 rk[NCH], rv[NCH];
    int32_t pk[NCH], pn[NCH];
    auto tile_key = [&](int32_t j) { return k0 + min(j, nt - 1) * 64; };
    auto look_up = [&](int32_t j) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < NCH; u++) pn[u] = block_page(a, map, tile_key(j) + ((wr + u * RSTEP) & ~15), s1);
    };
    auto load = [&](int32_t j, const char *base, int64_t page_bytes, uint32_t row_bytes, const int32_t (&pg)[NCH],
                    uint4 (&x)[NCH]) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < NCH; u++) {
            const int32_t b = tile_key(j) + ((wr + u * RSTEP) & ~15);
            const uint32_t r = ((wr + u * RSTEP) & 15) + lr;
            const __amdgpu_buffer_rsrc_t rs_ = block_rsrc(base, page_bytes, row_bytes,
                                                          pg[u] >= 0 ? row_in_page(a, map, b) : 0u, pg[u], b, s1);
            x[u] = buf_load16(rs_, b + (int32_t)r >= s0 ? r * row_bytes + lc * 16 : 0xffffffffu);
        }
    };
    auto load_k = [&](int32_t j) __attribute__((always_inline)) { load(j, map.k, a.kb * 2, map.kt, pn, rk); };
    auto load_v = [&](int32_t j) __attribute__((always_inline)) { load(j, map.v, a.vb * 2, map.vt, pk, rv); };
    auto next_pages = [&](int32_t j) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < NCH; u++) pk[u] = pn[u];
        look_up(j);
    };
    auto store_k = [&](int32_t j) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < NCH; u++) *(uint4 *)(sm.wide.k[j & 1] + (wr + u * RSTEP + lr) * KS + lc * 8) = rk[u];
    };
    auto store_v = [&](int32_t j) __attribute__((always_inline)) {
        const int32_t t = k0 + j * 64;
        if (t < tlo || t + 64 > thi) {  // (a tile that some row does not see all of)
            bool bad = false;
#pragma unroll
            for (int u = 0; u < NCH; u++) bad |= take_out<DT>(rv[u]);
            if (__any(bad) && lane == 0) sm.bad = 1;
        }
#pragma unroll
        for (int u = 0; u < NCH; u++) *(uint4 *)(sm.wide.v[j & 1] + (wr + u * RSTEP + lr) * VS + lc * 8) = rv[u];
    };
    Partial<D> p;
    p.m = -INFINITY, p.l = 0.f;
#pragma unroll
    for (int dt = 0; dt < DTN; dt++) p.acc[dt] = zero16();
    f32x16_t s[2];
    Frag8 pf[2][2];
    auto products = [&](int32_t j) __attribute__((always_inline)) {
        __builtin_amdgcn_s_setprio(1);
        if (rows && j < nt) {
            const uint16_t *sk = sm.wide.k[j & 1];
#pragma unroll
            for (int t = 0; t < 2; t++) s[t] = zero16();
#pragma unroll
            for (int st = 0; st < KST; st++)
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    Frag8 x;
                    x.u = *(const uint4 *)(sk + (t * 32 + col) * KS + half * 8 + st * 16);
                    s[t] = mfma32<DT>(x, rs.qf[st], s[t]);
                }
        }
        __builtin_amdgcn_sched_barrier(0);
        if (rows && j > 0) {
            const uint16_t *v = sm.wide.v[(j - 1) & 1];
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int dt = 0; dt < DTN; dt++)
                        p.acc[dt] = mfma32<DT>(lds_tr_frag(v, VS, t * 32 + u * 16, dt * 32, lane), pf[t][u], p.acc[dt]);
        }
        __builtin_amdgcn_s_setprio(0);
    };
    auto softmax = [&](int32_t jj) __attribute__((always_inline)) {
        const int32_t j0 = k0 + jj * 64;
        if (j0 < rs.flo || j0 + 64 > rs.fhi) {
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int32_t j = j0 + t * 32 + crow(i, lane);
                    s[t][i] = (j >= rs.lo) & (j < rs.hi) ? s[t][i] : -INFINITY;
                }
        }
        float tmax = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int i = 0; i < 16; i++) tmax = fmaxf(tmax, s[t][i]);
        tmax = fmaxf(tmax, __shfl_xor(tmax, 32, 64));
        const float tmc = tmax * c2;
        const bool grow = tmc - p.m > 8.f;  // false while both are -inf
        if (__any(grow)) {
            const float mnew = grow ? tmc : p.m;
            const float alpha = grow ? fast_exp2(p.m - mnew) : 1.f;  // 0 from -inf
            p.m = mnew;
            p.l *= alpha;
#pragma unroll
            for (int dt = 0; dt < DTN; dt++)
#pragma unroll
                for (int i = 0; i < 16; i++) p.acc[dt][i] *= alpha;
        }
        const float mneg = p.m == -INFINITY ? 0.f : -p.m;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int u = 0; u < 2; u++) {
                float e[8];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    e[i] = fast_exp2(fmaf(s[t][8 * u + i], c2, mneg));
                    p.l += e[i];
                }
                pf[t][u].u = make_uint4(pack2<DT>(e[0], e[1]), pack2<DT>(e[2], e[3]), pack2<DT>(e[4], e[5]),
                                        pack2<DT>(e[6], e[7]));
            }
    };
    // Wavefronts 0-3 store K_{j+1} and V_j during their softmax of step j, wavefronts 4-7, half a step
    // later, K_{j+2} and V_{j+1}: each tile is whole before its first reader's step.
    const int32_t ahead = first ? 0 : 1;
    auto stage = [&](int32_t j) __attribute__((always_inline)) {
        store_k(j + 1 + ahead);
        store_v(j + ahead);
        load_v(j + 1 + ahead);
        load_k(j + 2 + ahead);
        next_pages(j + 3 + ahead);
    };
    look_up(0);
    load_k(0);
    store_k(0);
    next_pages(1);
    load_v(0);
    load_k(1);
    next_pages(2);
    __syncthreads();
    if (!first) {
        stage(-1);
        __syncthreads();
    }
    for (int32_t j = 0; j <= nt; j++) {
        products(j);
        __syncthreads();
        if (rows && j < nt) softmax(j);
        if (j < nt) stage(j);
        __syncthreads();
    }
    if (first) __syncthreads();
    if (!rows) return;
    if (sm.bad)
        for (int32_t j0 = k0; j0 < s1; j0 += 64)
            if (j0 < tlo || j0 + 64 > thi)
                add_back<DT, D>(a, map, max(j0, s0), min(j0 + 64, s1), rs.lo, rs.hi, p.acc);
    const float l = p.l + __shfl_xor(p.l, 32, 64);
    if (!rs.on) return;
    const SharedRow row = row_of(a, it, wave * 32 + col);
    if (l != 0.f) {
        const float inv = 1.f / l;
#pragma unroll
        for (int dt = 0; dt < DTN; dt++)
#pragma unroll
            for (int g4 = 0; g4 < 4; g4++)
                *(float4 *)(a.part_o + row.part * D + dt * 32 + g4 * 8 + half * 4) =
                    make_float4(p.acc[dt][g4 * 4] * inv, p.acc[dt][g4 * 4 + 1] * inv, p.acc[dt][g4 * 4 + 2] * inv,
                                p.acc[dt][g4 * 4 + 3] * inv);
    }
    if (half == 0) a.part_lse[row.part] = l == 0.f ? -INFINITY : (p.m + log2f(l)) * 0.6931471805599453f;
}

template <int DT, int D, bool WIDE>
__global__ __launch_bounds__(64 * shared_waves<D>(), 1) void decode_shared_mfma(SharedArgs a,
                                                                                  const void *__restrict__ q,
                                                                                  const void *__restrict__ k,
                                                                                  const void *__restrict__ v) {
    __shared__ SharedSmem<D> sm;
    SharedItem it;
    if (!item_of<WIDE ? 32 * shared_waves<D>() : 32>(a, WIDE ? 64 : 32, sm.sc, it)) return;
    PageMap map;
    map.k = (const char *)k + (int64_t)it.kh * a.kh * 2;
    map.v = (const char *)v + (int64_t)it.kh * a.vh * 2;
    map.table = a.block_table + it.table * a.max_pages;
    map.kt = (uint32_t)(a.kt * 2), map.vt = (uint32_t)(a.vt * 2);
    map.shift = (a.page_size & (a.page_size - 1)) ? -1 : __builtin_ctzll(a.page_size);
    if (WIDE && it.prefix)
        shared_wide<DT, D>(a, it, map, q, sm);
    else
        shared_narrow<DT, D>(a, it, map, q, sm);
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

// The 16-bit kernel's calls: rows in 16-byte pieces, a block's bytes in 32 bits.
static bool shared_mfma_takes(const dm_attention_desc *d, int64_t page_size) {
    if ((d->dtype != DM_BF16 && d->dtype != DM_F16) || (d->d != 64 && d->d != 128 && d->d != 256) ||
        page_size % 16 != 0)
        return false;
    if (!d->strided) return true;
    auto ok = [&](const dm_strides &x) {
        return x.b % 8 == 0 && x.t % 8 == 0 && x.h % 8 == 0 && x.t >= d->d && x.t < ((int64_t)1 << 24);
    };
    return d->sq.b % 8 == 0 && d->sq.h % 8 == 0 && ok(d->sk) && ok(d->sv);
}

// The split of a call: ranges of the prefixes and of the rows' own keys, so that there are about
// kSharedTarget workgroups of each kind where the cache is long enough for ranges of 128 keys.
constexpr int64_t kSharedTarget = 256;
struct SharedPlan {
    bool wide;
    int32_t rows;  // rows of a prefix tile
    int64_t ptiles;
    int32_t otiles, nsp, nso;
};
static SharedPlan shared_plan(const dm_attention_desc *d, bool mfma, int64_t ngroups) {
    SharedPlan p{};
    const int64_t rep = d->hq / d->hkv;
    p.wide = mfma && ngroups > 0 && d->b * rep > 32 * ngroups;
    p.rows = p.wide ? (d->d == 256 ? 128 : 256) : 32;
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
    // (which kernel runs also depends on the pointers' alignment)
    const SharedPlan p = shared_plan(d, false, ngroups), m = shared_plan(d, shared_mfma_takes(d, page_size), ngroups);
    const size_t parts = (size_t)(d->b * d->hq) * std::max(p.nsp + p.nso, m.nsp + m.nso);
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
    const bool mfma = shared_mfma_takes(d, page_size) && aligned_16b(q) && aligned_16b(k_pages) && aligned_16b(v_pages);
    const SharedPlan p = shared_plan(d, mfma, ngroups);
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
    const unsigned g = (unsigned)grid;
#define SHARED_W(DT, D)                                                                            \
    if (p.wide)                                                                                    \
        decode_shared_mfma<DT, D, true><<<g, 64 * shared_waves<D>(), 0, st>>>(a, q, k_pages, v_pages); \
    else                                                                                           \
        decode_shared_mfma<DT, D, false><<<g, 64 * shared_waves<D>(), 0, st>>>(a, q, k_pages, v_pages)
#define SHARED(DT)                                                             \
    if (!mfma) {                                                               \
        decode_shared_generic<DT><<<g, 256, 0, st>>>(a, q, k_pages, v_pages);  \
    } else if constexpr (DT != DM_F32) {                                       \
        if (d->d == 64) {                                                      \
            SHARED_W(DT, 64);                                                  \
        } else if (d->d == 128) {                                              \
            SHARED_W(DT, 128);                                                 \
        } else {                                                               \
            SHARED_W(DT, 256);                                                 \
        }                                                                      \
    }                                                                          \
    decode_shared_merge<DT><<<(unsigned)rows, 256, 0, st>>>(a, o)
    if (d->dtype == DM_F32) {
        SHARED(DM_F32);
    } else if (d->dtype == DM_BF16) {
        SHARED(DM_BF16);
    } else {
        SHARED(DM_F16);
    }
#undef SHARED
#undef SHARED_W
    probe_add(DM_PROBE_DECODE_SHARED);
    DM_LAUNCH_CHECK("attention_decode_shared: launch");
    return DM_OK;
}

}  // extern "C"
