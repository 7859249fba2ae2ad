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
//
// Measured in bf16, with the merge, MFMA rates counting 4 D a (row, key) pair (a large product on this card
// runs at 1240 TFLOP/s, a large copy at 5.0 TB/s):
//   256 rows, a prefix of 32768 keys, 512 of their own, 32 heads of 128 over 8: 197 us, 707 TFLOP/s. Bound by
//     the prefix's products: alone they take 394 thousand cycles on 192 compute units (184 us at 2.14 GHz) and
//     313 thousand on all 256 (154 us at 2.03 GHz, 893 TFLOP/s), the cycles of the attention forward for as many
//     products (323 thousand); after some launches back to back the clock falls and they take 200 and 174 us. A
//     64-key step of 256 rows takes 3900 cycles, 2060 of them MFMA issue.
//   64 rows, 16384 and 1024 keys, the same heads: 75 us: 216 MB, 43 us at a copy's rate, and about 6 us until
//     the first keys arrive (the groups, the lengths, the page, the keys: each waits for the one in front).
//   8 rows, 6144 and 200 keys, 8 heads of 256 over 2: 20 us; 45 rows in 5 groups, 16 heads of 64 over 2 in f16,
//     window 6000: 23 us: the same chain, one or a few steps, the ranges' join and the merge's launch.
#include <algorithm>
#include <string>

#include "attention_kernels.h"
#include "dm_common.h"
#include "mfma.h"

namespace dm {

struct SharedArgs {
    int32_t B, S, left;   // left: the window's, -1 for none
    int32_t hq, hkv, d, rep;
    float scale;
    const int32_t *lengths, *groups, *prefix, *block_table;
    int32_t ngroups;
    int64_t page_size, max_pages, num_pages;
    int64_t qb, qh, kb, kt, kh, vb, vt, vh;
    int32_t nsp, nso;     // ranges of a prefix, and of a row's own keys
    int32_t ptiles;       // prefix tiles of a key-value head (an upper bound, see first_tile)
    int32_t otiles;       // tiles of a row's own heads
    float *part_o;        // [B, Hq, nsp + nso, D], each range's output normalised
    float *part_lse;      // [B, Hq, nsp + nso] natural log, -inf for a range without keys (its output unwritten)
};

constexpr int kOwnRows = 32;  // rows of a tile of own keys

__device__ __forceinline__ int32_t uniform(int32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int32_t clamp_len(const SharedArgs &a, int32_t x) { return min(max(x, 0), a.S); }
__device__ __forceinline__ int32_t len_of(const SharedArgs &a, int32_t m) {
    return a.lengths ? clamp_len(a, a.lengths[m]) : a.S;
}
__device__ __forceinline__ int32_t low_of(const SharedArgs &a, int32_t len) {
    return a.left >= 0 ? max(len - 1 - a.left, 0) : 0;
}
// The page of key j of sequence m, or -1.
__device__ __forceinline__ int64_t shared_page(const SharedArgs &a, int64_t m, int64_t j) {
    const int64_t pg = a.block_table[m * a.max_pages + j / a.page_size];
    return pg >= 0 && pg < a.num_pages ? pg : -1;
}

// What a workgroup or a wavefront does: range `slot` of the rows r0 .. r0 + nrow - 1 (row r: member
// m0 + r / rep, query head kh rep + r % rep) over the keys [s0, s1), which lie on `table`'s pages; a
// member sees those of its own range that lie in front of `cap`. Every field but len is the wavefront's.
struct SharedItem {
    int32_t m0, m1, table, s0, s1, base, cap, r0, nrow, kh, slot;
    bool prefix;
    int32_t len;  // own keys: the member's; prefix: a lane's of the members m0 + lane (-1 past the last)
};

// The first tile of group g, whose rows start at row s (of all rows of a key-value head): behind every
// tile of the groups in front, since ceil(r / RT) <= floor((x + r - 1) / RT) - floor(x / RT) + 1.
template <int RT>
__device__ __forceinline__ int32_t first_tile(int32_t s, int32_t g) {
    constexpr int shift = RT == 32 ? 5 : (RT == 128 ? 7 : 8);
    static_assert(RT == 1 << shift, "a tile's rows");
    return ((s - g) >> shift) + g;
}

// Row r of an item: its member, its query head and its place among the partial results.
__device__ __forceinline__ void head_of(const SharedArgs &a, const SharedItem &it, int r, int32_t *member, int32_t *head) {
    const uint32_t rr = it.r0 + r;
    *member = it.m0 + (it.prefix ? (int32_t)(rr / (uint32_t)a.rep) : 0);
    *head = it.kh * a.rep + (int32_t)(it.prefix ? rr % (uint32_t)a.rep : rr);
}
__device__ __forceinline__ int64_t part_of(const SharedArgs &a, const SharedItem &it, int r) {
    int32_t member, head;
    head_of(a, it, r, &member, &head);
    return ((int64_t)member * a.hq + head) * (a.nsp + a.nso) + it.slot;
}

// Which rows the item of `index` has (false: none, or there is no such item), and for a prefix its group's
// last row; its keys come with range_of. A whole wavefront; with several for an item each does the same, and the
// first (`writes`) writes. RT: rows of a prefix tile.
template <int RT>
__device__ __forceinline__ bool rows_of(const SharedArgs &a, int32_t index, bool writes, SharedItem &it) {
    const int lane = threadIdx.x & 63;
    const int32_t np = a.ptiles * a.nsp;
    uint32_t x = (uint32_t)index;
    it.kh = (int32_t)(x % (uint32_t)a.hkv);
    x /= (uint32_t)a.hkv;
    it.prefix = x < (uint32_t)np;
    int32_t b = 0, tile = 0, ot = 0;
    if (it.prefix) {
        tile = (int32_t)(x % (uint32_t)a.ptiles), it.slot = (int32_t)(x / (uint32_t)a.ptiles);
    } else {
        x -= np;
        b = (int32_t)(x % (uint32_t)a.B);
        x /= (uint32_t)a.B;
        ot = (int32_t)(x % (uint32_t)a.otiles), it.slot = a.nsp + (int32_t)(x / (uint32_t)a.otiles);
        it.len = len_of(a, b);
    }
    // the group (the last that starts at the tile or in front of it, the first that holds the row), if the
    // groups go up from 0 at least to B at most: 64 of them at a time, a lane each
    bool ok = true;
    int32_t g = -1, m0 = 0, m1 = 0, plen = 0;
    for (int32_t g0 = 0; g0 < a.ngroups; g0 += 64) {
        const int32_t i = g0 + lane;
        const bool on = i < a.ngroups;
        const int32_t s = on ? a.groups[i] : 0, e = on ? a.groups[i + 1] : 0, pl = on ? a.prefix[i] : 0;
        ok = ok && s >= 0 && s <= e && e <= a.B;
        const bool here = it.prefix ? on && first_tile<RT>(s * a.rep, i) <= tile : on && s <= b && b < e;
        const unsigned long long v = __ballot(here);
        if (v) {
            const int at = it.prefix ? 63 - __builtin_clzll(v) : __builtin_ctzll(v);
            g = g0 + at;
            m0 = __builtin_amdgcn_readlane(s, at), m1 = __builtin_amdgcn_readlane(e, at);
            plen = clamp_len(a, __builtin_amdgcn_readlane(pl, at));
        }
    }
    ok = __all(ok);
    if (it.prefix) {
        if (!ok || g < 0) return false;
        const int32_t first = (tile - first_tile<RT>(m0 * a.rep, g)) * RT, rows = (m1 - m0) * a.rep;
        if (first >= rows) return false;
        it.m0 = m0, it.m1 = m1, it.r0 = first, it.nrow = min(RT, rows - first), it.cap = plen;
        it.len = m0 + lane < m1 ? len_of(a, m0 + lane) : -1;
        return true;
    }
    const bool grouped = ok && g >= 0;
    it.m0 = it.table = b;
    it.r0 = ot * kOwnRows, it.nrow = min(kOwnRows, a.rep - it.r0);
    it.base = grouped ? plen : 0, it.cap = a.S;
    if (!grouped && it.slot == a.nsp && writes)  // the prefix's ranges, which nobody else writes
        for (int i = lane; i < it.nrow * a.nsp; i += 64)
            a.part_lse[((int64_t)b * a.hq + it.kh * a.rep + it.r0 + i / a.nsp) * (a.nsp + a.nso) + i % a.nsp] = -INFINITY;
    return true;
}

// The item's keys: false where there are none, which is then written down. unit: ranges are multiples of
// this many keys (a multiple of 16).
__device__ __forceinline__ bool range_of(const SharedArgs &a, int unit, bool writes, SharedItem &it) {
    const int lane = threadIdx.x & 63;
    int32_t lo, hi;
    if (it.prefix) {
        // the longest member, and the shortest that sees any key
        int32_t most = -1, least = INT32_MAX, at = 0;
        for (int32_t m = it.m0 + lane; m < it.m1; m += 64) {
            const int32_t l = m < it.m0 + 64 ? it.len : len_of(a, m);
            if (l > most) most = l, at = m;
            if (l > 0) least = min(least, l);
        }
        int32_t longest = most;
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) longest = max(longest, __shfl_xor(longest, o, 64));
        longest = uniform(longest);
        it.table = __builtin_amdgcn_readlane(at, __builtin_ctzll(__ballot(most == longest)));
        hi = min(it.cap, longest);
        lo = 0;
        if (a.left >= 0 && longest > 0) {
#pragma unroll
            for (int o = 32; o >= 1; o >>= 1) least = min(least, __shfl_xor(least, o, 64));
            lo = low_of(a, uniform(least));
        }
    } else {
        hi = uniform(it.len);
        lo = max(it.base, low_of(a, hi));
    }
    const int32_t from = lo & ~15, n = it.prefix ? a.nsp : a.nso, split = it.prefix ? it.slot : it.slot - a.nsp;
    const int32_t each = hi > from ? (int32_t)(((uint32_t)(hi - from) + n - 1) / (uint32_t)n + unit - 1) / unit * unit : 0;
    const int64_t start = from + (int64_t)split * each;
    it.s0 = (int32_t)max((int64_t)lo, min(start, (int64_t)hi));
    it.s1 = (int32_t)min((int64_t)hi, start + each);
    if (it.s0 < it.s1) return true;
    if (writes)
        for (int r = lane; r < it.nrow; r += 64) a.part_lse[part_of(a, it, r)] = -INFINITY;
    return false;
}

// The simple form, for every type, head width, page size and stride: 32 rows and 16 keys at a time in
// LDS as f32, eight threads a row, each two of its scores and every eighth column of its output. Bound by
// its LDS reads, two for a multiply-add of the scores and one of the outputs: 256 bf16 rows of 32768 + 512
// keys, 32 heads of 128, in pages of 8 take 26.7 ms here, in pages of 16 0.2 below. (64 rows of 4096 + 256 keys,
// 32 heads over 8: f32 128 wide 0.85 ms, bf16 96 wide 0.67; row by row the paged decode takes 4.9 and 6.2.)
constexpr int kGenKeys = 16;
template <int DT>
__global__ __launch_bounds__(256) void decode_shared_generic(SharedArgs a, const void *__restrict__ q,
                                                             const void *__restrict__ k,
                                                             const void *__restrict__ v) {
    __shared__ float qs[32][257], kv[kGenKeys][257], ps[32][kGenKeys + 1];
    SharedItem it;
    if (!rows_of<32>(a, blockIdx.x, threadIdx.x < 64, it) || !range_of(a, kGenKeys, threadIdx.x < 64, it)) return;
    const int tid = threadIdx.x, r = tid >> 3, c = tid & 7;
    int32_t member, head, low = it.s0, high = r < it.nrow ? it.s1 : 0;
    head_of(a, it, r < it.nrow ? r : 0, &member, &head);
    const int64_t part = part_of(a, it, r < it.nrow ? r : 0);
    if (it.prefix) {
        const int32_t len = len_of(a, member);
        low = max(low_of(a, len), it.s0), high = min(min(len, it.cap), high);
    }
    for (int i = tid; i < 32 * a.d; i += 256) {
        const int x = i / a.d, e = i - x * a.d;
        const int rr = it.r0 + (x < it.nrow ? x : 0);
        qs[x][e] = ld<DT>(q, (int64_t)(it.m0 + rr / a.rep) * a.qb + (it.kh * a.rep + rr % a.rep) * a.qh + e) * a.scale;
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
            if (j >= low && j < high) {
                float t = 0.f;
                for (int e = 0; e < a.d; e++) t += qs[r][e] * kv[x][e];
                s[u] = t;
            }
            mx = fmaxf(mx, s[u]);
        }
#pragma unroll
        for (int o = 4; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
        // (while every score that the row has seen is -inf, their weights are 0 and not e^(-inf + inf))
        const float mn = fmaxf(m, mx), ref = mn == -INFINITY ? 0.f : mn;
        const float alpha = mn == -INFINITY ? 1.f : expf(m - mn);
        m = mn;
        l *= alpha;
#pragma unroll
        for (int u = 0; u < 2; u++) {
            // (a masked key's weight is a marker below zero: what its value holds stays out)
            const int64_t j = j0 + c + 8 * u;
            const bool seen = j >= low && j < high;
            s[u] = seen ? expf(s[u] - ref) : 0.f;
            ps[r][c + 8 * u] = seen ? s[u] : -1.f;
        }
        l += s[0] + s[1];
        __syncthreads();
        for (int i = tid; i < n * a.d; i += 256) {
            const int x = i / a.d, e = i - x * a.d;
            const int64_t pg = shared_page(a, it.table, j0 + x);
            kv[x][e] = pg >= 0 ? ld<DT>(v, pg * a.vb + (j0 + x) % a.page_size * a.vt + it.kh * a.vh + e) : 0.f;
        }
        __syncthreads();
        // (the step's 16 products first: with one addition a key a sum over 2^14 keys of like weights is off by
        // as much as 2^-12)
        float w[kGenKeys];
#pragma unroll
        for (int x = 0; x < kGenKeys; x++) w[x] = ps[r][x];
#pragma unroll
        for (int i = 0; i < 32; i++) {
            if (c + 8 * i >= a.d) continue;
            float t = 0.f;
#pragma unroll
            for (int x = 0; x < kGenKeys; x++) t += w[x] < 0.f ? 0.f : w[x] * kv[x][c + 8 * i];
            acc[i] = acc[i] * alpha + t;
        }
    }
#pragma unroll
    for (int o = 4; o >= 1; o >>= 1) l += __shfl_xor(l, o, 64);
    if (r >= it.nrow) return;
    // (l is NaN where a score is: the row's result is NaN then, as the softmax's)
    const bool none = l == 0.f;
#pragma unroll
    for (int i = 0; i < 32; i++)
        if (!none && c + 8 * i < a.d) a.part_o[part * a.d + c + 8 * i] = acc[i] / l;
    if (c == 0) a.part_lse[part] = none ? -INFINITY : m + logf(l);
}

// ------------------------------------------------------------------------------------------
// The 16-bit kernel (D = 64, 128 or 256, pages of a multiple of 16 keys)
// ------------------------------------------------------------------------------------------
//
// Both products run on MFMA: S^T = K q^T (keys x 32 rows) and O^T += V^T P^T, S^T's output layout being
// P^T's operand. The weights are rounded to the inputs' type for the second product, whose operands have one
// type and which in f32 would run at a sixteenth of the rate; the other attention kernels do the same. Off by half a
// step a weight, so that an output's error against 64 bits is 0.0023 in bf16 and 0.00028 in f16, where the output's
// own rounding makes 0.0017 and 0.00021. Sums, maxima and outputs stay in f32.
//
// NARROW items (a row's own keys; the prefix of a group of few rows): the keys are what there is to
// share out, so each wavefront sweeps keys of its own in blocks of 32 through its own LDS tiles, for
// up to 32 rows, and the wavefronts' results are joined in LDS.
//
// WIDE items (the prefix of a group of many rows): the rows are shared out, 32 a wavefront, and all
// sweep the same keys in tiles of 64. Wavefronts w and w + 4 of a SIMD run half a step apart, so
// that one's products and the other's softmax run side by side. (At D = 256 a wavefront a SIMD: its outputs
// and queries alone are 192 registers.)
//
// Keys arrive in 16-key blocks, each on one page: a buffer resource of the block's rows up to the
// item's end reads zeros behind it, and a page outside the pages, or in front of the item's start,
// reads as zeros too.

template <int D, bool WIDE>
constexpr int shared_waves() { return D == 256 || !WIDE ? 4 : 8; }

// Where the keys of an item lie: byte strides of a page and of a row (keys' and values' alike).
struct PageMap {
    const char *k, *v;  // at the item's key-value head
    const int32_t *table;
    uint32_t page, row;
    uint32_t size;      // rows of a page
};

// The offset of the 16-key block at key j, kNoBlock for a page outside the pages or a block behind `end`.
constexpr uint64_t kNoBlock = ~(uint64_t)0;
__device__ __forceinline__ uint64_t block_at(const SharedArgs &a, const PageMap &m, int32_t j, int32_t end) {
    if (j >= end) return kNoBlock;
    const uint32_t e = (uint32_t)j / m.size;
    const int32_t pg = m.table[e];
    return pg >= 0 && pg < a.num_pages ? (uint64_t)(uint32_t)pg * m.page + ((uint32_t)j - e * m.size) * m.row : kNoBlock;
}

// All ones in each 16-bit half of w that is not finite: its exponent plus one carries into the sign's
// place. (Arithmetic alone: a comparison an element would hold a mask of lanes for each.)
template <int DT>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
    constexpr uint32_t e = DT == DM_BF16 ? 0x7f807f80u : 0x7c007c00u, one = DT == DM_BF16 ? 0x00800080u : 0x04000400u;
    const uint32_t m = ((w & e) + one) & 0x80008000u;
    return (m - (m >> 15)) | m;
}
// Values that are not finite taken out of a piece of V (whoever sees them adds them at the end).
template <int DT>
__device__ __forceinline__ uint32_t take_out(uint4 &x) {
    uint32_t *w = (uint32_t *)&x, any = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t m = not_finite<DT>(w[i]);
        w[i] &= ~m;
        any |= m;
    }
    return any;
}

template <int D, bool WIDE>
struct SharedSmem {
    static constexpr int NW = shared_waves<D, WIDE>(), KS = D + 8, VS = D + 32;
    struct Narrow {
        alignas(16) uint16_t k[32 * KS], v[32 * VS];
    };
    struct Wide {
        alignas(16) uint16_t k[2][64 * KS], v[2][64 * VS];
    };
    static_assert(!WIDE || NW * 32 * KS * 2 <= (int)sizeof(Wide), "the queries go through the tiles' places");
    union {
        Narrow narrow[NW];
        Wide wide[WIDE];
        alignas(16) float join[WIDE ? 1 : NW * 32 * (D + 6)];
    };
    int32_t lo[NW], hi[NW], bad;
    uint64_t blocks[WIDE ? 512 : 1];  // wide: the offsets of 128 tiles' blocks, see fill
    int64_t places[WIDE ? 1 : 32];    // narrow: the rows' places among the partial results
};

// What the lanes of a wavefront know of their rows: the queries as the second operand, and the keys seen.
template <int D>
struct RowState {
    Frag8 qf[D / 16];
    int32_t len;       // prefix: the member's
    int32_t lo, hi;    // this lane's row
    int32_t flo, fhi;  // the keys that all of the wavefront's rows see
    bool on;
};

// The loads of 32 rows' queries (and of this lane's row's length), which need no key; nothing here waits for
// them. The lanes go along the rows, so that a load touches few cache lines: settle_rows sorts the pieces.
template <int DT, int D>
__device__ __forceinline__ void load_rows(const SharedArgs &a, const SharedItem &it, const void *q, int first, RowState<D> &w) {
    constexpr int LPR = D / 8, RPL = 64 / LPR;  // lanes a row, rows a load
    const int lane = threadIdx.x & 63, r = first + (lane & 31);
    w.on = r < it.nrow;
    int32_t member, head;
    head_of(a, it, w.on ? r : 0, &member, &head);  // (without a row: the first row's, nobody reads what becomes of it)
    w.len = it.prefix ? len_of(a, member) : 0;
    const int64_t off = member * a.qb + head * a.qh;
#pragma unroll
    for (int u = 0; u < D / 16; u++) {
        const int x = u * RPL + lane / LPR;
        const int64_t at = ((int64_t)__shfl((int)(off >> 32), x, 64) << 32) | (uint32_t)__shfl((int)off, x, 64);
        w.qf[u].u = *(const uint4 *)((const uint16_t *)q + at + (lane % LPR) * 8);
    }
}
// Through the wavefront's own rows of LDS, 32 of KS values, into operands; slots: in the order of row_frag
// (4 h + e and 8 + 4 h + e).
template <int D>
__device__ __forceinline__ void settle_rows(uint16_t *rows, bool slots, RowState<D> &w) {
    constexpr int LPR = D / 8, RPL = 64 / LPR, KS = D + 8;
    const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
#pragma unroll
    for (int u = 0; u < D / 16; u++) *(uint4 *)(rows + (u * RPL + lane / LPR) * KS + (lane % LPR) * 8) = w.qf[u].u;
    __builtin_amdgcn_wave_barrier();  // (a wavefront's LDS accesses complete in order)
    const uint16_t *mine = rows + col * KS;
#pragma unroll
    for (int s = 0; s < D / 16; s++) {
        if (slots) {
            const uint2 l = *(const uint2 *)(mine + s * 16 + half * 4), u = *(const uint2 *)(mine + s * 16 + 8 + half * 4);
            w.qf[s].u = make_uint4(l.x, l.y, u.x, u.y);
        } else {
            w.qf[s].u = *(const uint4 *)(mine + s * 16 + half * 8);
        }
    }
    __builtin_amdgcn_wave_barrier();
}

// The keys that the rows see, once the item's are known.
template <int D>
__device__ __forceinline__ void bound_rows(const SharedArgs &a, const SharedItem &it, RowState<D> &w) {
    w.lo = it.s0, w.hi = it.s1;
    if (it.prefix) w.lo = max(low_of(a, w.len), it.s0), w.hi = min(min(w.len, it.cap), it.s1);
    if (!w.on) w.hi = 0;
    int32_t flo = w.on ? w.lo : INT32_MIN, fhi = w.on ? w.hi : INT32_MAX;
    if (it.prefix) {
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) {
            flo = max(flo, __shfl_xor(flo, o, 64));
            fhi = min(fhi, __shfl_xor(fhi, o, 64));
        }
    }
    w.flo = uniform(flo), w.fhi = uniform(fhi);
    if (a.scale < 0.f) {  // (the softmax takes a scale above 0: the queries' signs instead)
#pragma unroll
        for (int s = 0; s < D / 16; s++) {
            uint4 &x = w.qf[s].u;
            x = make_uint4(x.x ^ 0x80008000u, x.y ^ 0x80008000u, x.z ^ 0x80008000u, x.w ^ 0x80008000u);
        }
    }
}

// The values that were taken out, added for the rows that see them: every key of [j0, j1) again, one
// at a time (a key that is not finite in a place that some row of the tile does not see).
template <int DT, int D>
__device__ __forceinline__ void add_back(const SharedArgs &a, const PageMap &m, int32_t j0, int32_t j1, int32_t lo,
                                         int32_t hi, f32x16_t (&acc)[D / 32]) {
    const int lane = threadIdx.x & 63;
    for (int32_t j = j0; j < j1; j++) {
        const uint64_t at = block_at(a, m, j, j1);
        if (at == kNoBlock || j < lo || j >= hi) continue;
        const uint16_t *row = (const uint16_t *)(m.v + at);
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

// One item's results: unnormalised O^T (this lane's row, the D / 2 columns of its half), the reference m
// (log2 units) and the sum l of this lane's half.
template <int D>
struct Partial {
    f32x16_t acc[D / 32];
    float m, l;
};

// A wavefront's rows (n from r0 on) with the sums l over both halves: normalised partial results, through its
// own `rows` of LDS so that the lanes go along the rows. (A range whose weights are 0 is zeros that nobody reads.)
template <int D>
__device__ __forceinline__ void put_rows(const SharedArgs &a, const SharedItem &it, int r0, const Partial<D> &p, float l,
                                         float *rows) {
    constexpr int JS = D + 4, LPR = D / 4, RPL = 64 / LPR;
    const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5, n = min(32, it.nrow - r0);
    const int64_t part = part_of(a, it, r0 + (col < n ? col : 0));
    const float inv = l == 0.f ? 0.f : 1.f / l;  // (NaN is not 0)
#pragma unroll
    for (int dt = 0; dt < D / 32; dt++)
#pragma unroll
        for (int g4 = 0; g4 < 4; g4++)
            *(float4 *)(rows + col * JS + dt * 32 + g4 * 8 + half * 4) =
                make_float4(p.acc[dt][g4 * 4] * inv, p.acc[dt][g4 * 4 + 1] * inv, p.acc[dt][g4 * 4 + 2] * inv,
                            p.acc[dt][g4 * 4 + 3] * inv);
    __builtin_amdgcn_wave_barrier();
    if (half == 0 && col < n) a.part_lse[part] = l == 0.f ? -INFINITY : (p.m + log2f(l)) * 0.6931471805599453f;
    for (int r = 0; r < n; r += RPL) {
        const int x = r + lane / LPR, y = min(x, 31);
        const int64_t to = ((int64_t)__shfl((int)(part >> 32), y, 64) << 32) | (uint32_t)__shfl((int)part, y, 64);
        const float4 o = *(const float4 *)(rows + y * JS + lane % LPR * 4);
        if (x < n) *(float4 *)(a.part_o + to * D + lane % LPR * 4) = o;
    }
}

// TEAM: the wavefronts that share the item's keys, the whole workgroup or one.
template <int DT, int D, bool WIDE, int TEAM>
__device__ __forceinline__ void shared_narrow(const SharedArgs &a, const SharedItem &it, const PageMap &map,
                                              RowState<D> &rs, SharedSmem<D, WIDE> &sm) {
    constexpr int NW = TEAM, KS = SharedSmem<D, WIDE>::KS, VS = SharedSmem<D, WIDE>::VS;
    constexpr int LPR = D / 8, RPL = 64 / LPR, NLD = 32 / RPL;  // lanes a row, rows a load, loads
    constexpr int KST = D / 16, DTN = D / 32;
    const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
    const int slot = uniform(threadIdx.x >> 6), wave = TEAM == 1 ? 0 : slot;
    const float qscale = fabsf(a.scale) * 1.4426950408889634f;
    Partial<D> p;
    p.m = -INFINITY, p.l = 0.f;
#pragma unroll
    for (int dt = 0; dt < DTN; dt++) p.acc[dt] = zero16();
    const int32_t s0 = it.s0, s1 = it.s1, a0 = s0 & ~15;
    const int32_t per = ((s1 - a0 + NW - 1) / NW + 31) & ~31;
    const int32_t w0 = max(s0, a0 + wave * per), w1 = min(s1, a0 + (wave + 1) * per), b0 = w0 & ~15;
    typename SharedSmem<D, WIDE>::Narrow &t = sm.narrow[slot];
    uint4 sk[NLD], sv[NLD];
    // the offsets of 64 blocks of 16 keys from block `from` on, a lane each
    uint64_t at;
    auto look_up = [&](int32_t from) __attribute__((always_inline)) { at = block_at(a, map, b0 + 16 * (from + lane), w1); };
    auto load = [&](int32_t n) __attribute__((always_inline)) {  // the n-th 32 keys
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int32_t j = b0 + 32 * n + 16 * h, i = (2 * n + h) & 63;
            const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)at, i);
            const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)(at >> 32), i);
            const bool none = hi == 0xffffffffu;
            const uint64_t from = none ? 0 : ((uint64_t)hi << 32) | lo;
            const uint32_t bytes = uniform(none ? 0 : max(0, min(16, w1 - j))) * map.row;
            const __amdgpu_buffer_rsrc_t kr = make_rsrc(map.k + from, bytes), vr = make_rsrc(map.v + from, bytes);
#pragma unroll
            for (int u = h * NLD / 2; u < (h + 1) * NLD / 2; u++) {
                const uint32_t r = RPL * u - 16 * h + lane / LPR;
                const uint32_t off = j + (int32_t)r >= w0 ? r * map.row + (lane % LPR) * 16 : 0xffffffffu;
                sk[u] = buf_load16_nt(kr, off);
                sv[u] = buf_load16_nt(vr, off);
            }
        }
    };
    uint32_t bad = 0;
    if (w0 < w1) {
        const int nblk = (w1 - b0 + 31) / 32;
        look_up(0);
        load(0);
        settle_rows<D>(t.k, true, rs);
        bound_rows<D>(a, it, rs);
        for (int n = 0; n < nblk; n++) {
            const int32_t j0 = b0 + n * 32;
            const bool cut = j0 < rs.flo || j0 + 32 > rs.fhi;
#pragma unroll
            for (int u = 0; u < NLD; u++) {
                const int r = RPL * u + lane / LPR, c = (lane % LPR) * 8;
                *(uint4 *)(t.k + r * KS + c) = sk[u];
                *(uint4 *)(t.v + r * VS + c) = sv[u];
            }
            if (cut) {  // (in LDS: the loads' registers are full)
#pragma unroll 1
                for (int u = 0; u < NLD; u++) {
                    uint4 *x = (uint4 *)(t.v + (RPL * u + lane / LPR) * VS + (lane % LPR) * 8), y = *x;
                    const uint32_t m = take_out<DT>(y);
                    if (m) *x = y;
                    bad |= m;
                }
            }
            if ((n & 31) == 31) look_up(2 * n + 2);
            load(n + 1);
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
    if constexpr (TEAM == 1) {
        static_assert(sizeof(t) >= 32 * (D + 4) * sizeof(float), "the results go through the tile's place");
        __builtin_amdgcn_wave_barrier();
        put_rows<D>(a, it, 0, p, l, (float *)&t);
        return;
    }
    // the wavefronts' results joined through LDS: [wave][row][D] (rows four banks apart), their references
    // and sums behind, which become the factors of the sum
    constexpr int JS = D + 4;
    __syncthreads();
    float *sa = sm.join, *sm_m = sa + NW * 32 * JS, *sm_l = sm_m + NW * 32;
    if (col < it.nrow) {
#pragma unroll
        for (int dt = 0; dt < DTN; dt++)
#pragma unroll
            for (int g4 = 0; g4 < 4; g4++)
                *(float4 *)(sa + (wave * 32 + col) * JS + dt * 32 + g4 * 8 + half * 4) =
                    make_float4(p.acc[dt][g4 * 4], p.acc[dt][g4 * 4 + 1], p.acc[dt][g4 * 4 + 2], p.acc[dt][g4 * 4 + 3]);
        if (half == 0) sm_m[wave * 32 + col] = p.m, sm_l[wave * 32 + col] = l;
    }
    __syncthreads();
    const int r = threadIdx.x;
    if (r < it.nrow) {
        float M = -INFINITY, L = 0.f, f[NW];
#pragma unroll
        for (int w = 0; w < NW; w++) M = fmaxf(M, sm_m[w * 32 + r]);
#pragma unroll
        for (int w = 0; w < NW; w++) {
            // (a reference of -inf: the wavefront's sums are 0, or NaN where all scores are)
            const float m = sm_m[w * 32 + r];
            f[w] = m == M ? 1.f : fast_exp2(m - M);
            L += sm_l[w * 32 + r] * f[w];
        }
        const float inv = L == 0.f ? 0.f : 1.f / L;  // (NaN is not 0)
#pragma unroll
        for (int w = 0; w < NW; w++) sm_l[w * 32 + r] = f[w] * inv;
        const int64_t part = part_of(a, it, r);
        sm.places[r] = part;
        a.part_lse[part] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
    }
    __syncthreads();
    for (int x = threadIdx.x; x < it.nrow * (D / 4); x += NW * 64) {
        const int r = x / (D / 4), d = x % (D / 4) * 4;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float f = sm_l[w * 32 + r];
            const float4 y = *(const float4 *)(sa + (w * 32 + r) * JS + d);
            o.x += y.x * f, o.y += y.y * f, o.z += y.z * f, o.w += y.w * f;
        }
        *(float4 *)(a.part_o + sm.places[r] * D + d) = o;
    }
}

template <int DT, int D>
__device__ __forceinline__ void shared_wide(const SharedArgs &a, const SharedItem &it, const PageMap &map,
                                            RowState<D> &rs, SharedSmem<D, true> &sm) {
    constexpr int NW = shared_waves<D, true>(), NT = NW * 64, KS = SharedSmem<D, true>::KS, VS = SharedSmem<D, true>::VS;
    constexpr int CPR = D / 8, RSTEP = NT / CPR, NCH = 64 / RSTEP;  // pieces a row, rows at a time, pieces a thread
    constexpr int KST = D / 16, DTN = D / 32, AHEAD = 2;
    const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool first = NW == 4 || wave < 4;  // products first in each step
    const int32_t s0 = it.s0, s1 = it.s1, k0 = s0 & ~15;
    auto fill = [&](int32_t block) __attribute__((always_inline)) {
        sm.blocks[block & 511] = block_at(a, map, k0 + 16 * block, s1);
    };
    fill(threadIdx.x);
    if (NT < 512) fill(threadIdx.x + 256);
    settle_rows<D>((uint16_t *)&sm.wide[0] + wave * 32 * KS, false, rs);  // (read whole before the barrier below)
    bound_rows<D>(a, it, rs);
    const bool rows = wave * 32 < it.nrow;  // this wavefront has rows
    if (lane == 0) sm.lo[wave] = rs.flo, sm.hi[wave] = rs.fhi;
    if (threadIdx.x == 0) sm.bad = 0;
    __syncthreads();
    int32_t tlo = INT32_MIN, thi = INT32_MAX;  // the keys that every row of the tile sees
#pragma unroll
    for (int w = 0; w < NW; w++) tlo = max(tlo, sm.lo[w]), thi = min(thi, sm.hi[w]);
    tlo = __builtin_amdgcn_readfirstlane(tlo), thi = __builtin_amdgcn_readfirstlane(thi);
    const int32_t nt = (s1 - k0 + 63) / 64;
    // (a scale of 0 as the smallest: a masked score stays -inf, the others' weights are alike)
    const float c2 = a.scale == 0.f ? 1.2e-38f : fabsf(a.scale) * 1.4426950408889634f;

    // staging: NCH pieces of a tile's K and of its V a thread. The offsets of the tiles' blocks lie in
    // LDS, a ring of 128 tiles: 64 of them are looked up 64 steps before they are read.
    const int row0 = threadIdx.x / CPR, lc = threadIdx.x % CPR;
    uint4 rk[NCH], rv[NCH];
    // A tile's offsets are read from LDS a step before its keys are loaded, and kept for its values.
    uint64_t ak[NCH], av[NCH];
    auto offsets = [&](int32_t j) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < NCH; u++) ak[u] = sm.blocks[(j * 4 + ((row0 + u * RSTEP) >> 4)) & 511];
    };
    // (a piece of no key is read from the first page and zeroed when it is stored: with its load left out
    // the compiler waits for the others' at once)
    bool okk[NCH], okv[NCH];
    auto load = [&](int32_t j, const char *base, const uint64_t (&at)[NCH], uint4 (&x)[NCH],
                    bool (&ok)[NCH]) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < NCH; u++) {
            const int r = row0 + u * RSTEP;
            ok[u] = at[u] != kNoBlock && (uint32_t)(k0 + j * 64 + r - s0) < (uint32_t)(s1 - s0);
            x[u] = *(const uint4 *)(base + (ok[u] ? at[u] : 0) + ((uint32_t)(r & 15) * map.row + lc * 16));
        }
    };
    auto load_v = [&](int32_t j) __attribute__((always_inline)) { load(j, map.v, av, rv, okv); };
    // the keys of tile j, then the offsets of the tile behind it
    auto load_k = [&](int32_t j) __attribute__((always_inline)) {
        load(j, map.k, ak, rk, okk);
#pragma unroll
        for (int u = 0; u < NCH; u++) av[u] = ak[u];
        offsets(j + 1);
    };
    auto zeroed = [](const uint4 &x, bool ok) {
        return make_uint4(ok ? x.x : 0u, ok ? x.y : 0u, ok ? x.z : 0u, ok ? x.w : 0u);
    };
    auto store_k = [&](int32_t j) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < NCH; u++)
            *(uint4 *)(sm.wide[0].k[j & 1] + (row0 + u * RSTEP) * KS + lc * 8) = zeroed(rk[u], okk[u]);
    };
    auto store_v = [&](int32_t j) __attribute__((always_inline)) {
        const int32_t t = k0 + j * 64;
#pragma unroll
        for (int u = 0; u < NCH; u++) rv[u] = zeroed(rv[u], okv[u]);
        if (t < tlo || t + 64 > thi) {  // (a tile that some row does not see all of)
            uint32_t bad = 0;
#pragma unroll
            for (int u = 0; u < NCH; u++) bad |= take_out<DT>(rv[u]);
            if (__any(bad) && lane == 0) sm.bad = 1;
        }
#pragma unroll
        for (int u = 0; u < NCH; u++) *(uint4 *)(sm.wide[0].v[j & 1] + (row0 + u * RSTEP) * VS + lc * 8) = rv[u];
    };
    Partial<D> p;
    p.m = -INFINITY, p.l = 0.f;
#pragma unroll
    for (int dt = 0; dt < DTN; dt++) p.acc[dt] = zero16();
    f32x16_t s[2];
    Frag8 pf[2][2];
    // O^T of step j - 1 first, whose operands are dead when S^T's take their registers; each fragment is
    // read from LDS ahead of the products in front of it.
    auto products = [&](int32_t j) __attribute__((always_inline)) {
        const uint16_t *tk = sm.wide[0].k[j & 1] + col * KS + half * 8, *tv = sm.wide[0].v[(j - 1) & 1];
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
        if (rows && j > 0) {
#pragma unroll
            for (int g = 0; g < 4; g++) {
                if (g < 3) read_v(g + 1);
#pragma unroll
                for (int dt = 0; dt < DTN; dt++) p.acc[dt] = mfma32<DT>(vf[g & 1][dt], pf[g >> 1][g & 1], p.acc[dt]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (rows && j < nt) {
#pragma unroll
            for (int st = 0; st < AHEAD; st++) read_k(st);
#pragma unroll
            for (int t = 0; t < 2; t++) s[t] = zero16();
#pragma unroll
            for (int st = 0; st < KST; st++) {
                if (st + AHEAD < KST) read_k(st + AHEAD);
#pragma unroll
                for (int t = 0; t < 2; t++) s[t] = mfma32<DT>(kf[st % (AHEAD + 1)][t], rs.qf[st], s[t]);
                __builtin_amdgcn_sched_barrier(0);
            }
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
                    s[t][i] = ((j >= rs.lo) & (j < rs.hi)) ? s[t][i] : -INFINITY;
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
        float ps = 0.f;  // (the tile's weights first: one at a time 2^19 like ones were summed 2^-8 short)
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
        p.l += ps;
    };
    // Wavefronts 0-3 store K_{j+1} and V_j during their softmax of step j, wavefronts 4-7, half a step
    // later, K_{j+2} and V_{j+1}: each tile is whole before its first reader's step.
    const int32_t ahead = first ? 0 : 1;
    auto stage = [&](int32_t j) __attribute__((always_inline)) {
        store_k(j + 1 + ahead);
        store_v(j + ahead);
        load_v(j + 1 + ahead);
        load_k(j + 2 + ahead);
        // (the ring's half that it goes to held tiles j - 64 .. j - 1, read by all; only wavefronts 0-3)
        if (first && (j & 63) == 0 && j > 0) fill(4 * (j + 64) + threadIdx.x);
    };
    offsets(0);
    load_k(0);
    load_v(0);
    store_k(0);
    load_k(1);
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
    // (every wavefront is past its last tile)
    static_assert(sizeof(sm.narrow) >= NW * 32 * (D + 4) * sizeof(float), "the results go through the tiles' places");
    put_rows<D>(a, it, wave * 32, p, l, (float *)&sm.narrow[0] + wave * 32 * (D + 4));
}

template <int DT, int D, bool WIDE>
__global__ __launch_bounds__((64 * shared_waves<D, WIDE>()), (D == 256 ? 1 : 2)) void decode_shared_mfma(SharedArgs a, int32_t items,
                                                                                        const void *__restrict__ q,
                                                                                        const void *__restrict__ k,
                                                                                        const void *__restrict__ v) {
    constexpr int NW = shared_waves<D, WIDE>(), RT = WIDE ? 32 * NW : 32;
    __shared__ SharedSmem<D, WIDE> sm;
    // the prefixes' items first, a workgroup each, then the rows' own keys, a wavefront each
    const int32_t np = a.ptiles * a.nsp * a.hkv;
    const int wave = uniform(threadIdx.x >> 6);
    const bool prefix = (int32_t)blockIdx.x < np, writes = !prefix || wave == 0;
    const int32_t index = prefix ? (int32_t)blockIdx.x : np + ((int32_t)blockIdx.x - np) * NW + wave;
    SharedItem it{};
    RowState<D> rs;
    if (!uniform(index < items && rows_of<RT>(a, index, writes, it))) return;
    // (the queries' loads are in flight while the item's keys are found)
    const bool wide = WIDE && prefix;
    load_rows<DT, D>(a, it, q, wide ? wave * 32 : 0, rs);
    if (!uniform(range_of(a, wide ? 64 : 32, writes, it))) return;
    // (the wavefront's, which the compiler does not see of every one: the loads below take scalar bases)
    it.m0 = uniform(it.m0), it.table = uniform(it.table), it.s0 = uniform(it.s0), it.s1 = uniform(it.s1);
    it.cap = uniform(it.cap), it.r0 = uniform(it.r0), it.nrow = uniform(it.nrow), it.kh = uniform(it.kh);
    it.slot = uniform(it.slot);
    PageMap map;
    map.k = (const char *)k + (int64_t)it.kh * a.kh * 2;
    map.v = (const char *)v + (int64_t)it.kh * a.vh * 2;
    map.table = a.block_table + it.table * a.max_pages;
    map.page = (uint32_t)(a.kb * 2), map.row = (uint32_t)(a.kt * 2), map.size = (uint32_t)a.page_size;
    if (!prefix) {
        shared_narrow<DT, D, WIDE, 1>(a, it, map, rs, sm);
        return;
    }
    if constexpr (WIDE)
        shared_wide<DT, D>(a, it, map, rs, sm);
    else
        shared_narrow<DT, D, WIDE, NW>(a, it, map, rs, sm);
}

// The ranges of a row joined, a workgroup a row: the ranges that hold keys are listed with their
// weights (those of weight 0 too: zero times a result that is not finite is NaN), and thread t sums, for
// the columns of its piece t % pieces (four of them where D is a multiple of 4, one otherwise), every
// groups-th of the list, eight loads in flight; the groups are added in order.
constexpr int kSharedSplits = 512;  // most ranges of a row
template <int DT, int V>
__global__ __launch_bounds__(256) void decode_shared_merge(SharedArgs a, void *__restrict__ o) {
    __shared__ float w[kSharedSplits], red[256 * V], tops[4], sums[4];
    __shared__ int32_t list[kSharedSplits], counts[4];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = a.nsp + a.nso;
    const float x0 = tid < n ? a.part_lse[row * n + tid] : -INFINITY;
    const float x1 = tid + 256 < n ? a.part_lse[row * n + tid + 256] : -INFINITY;
    const float mx = wave_max(fmaxf(x0, x1));
    if (lane == 0) tops[wave] = mx;
    const bool nan = __syncthreads_or(x0 != x0 || x1 != x1);
    const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    auto weight = [&](float x) { return x == -INFINITY ? 0.f : (x == top ? 1.f : expf(x - top)); };
    const float w0 = weight(x0), w1 = weight(x1);
    const float part = wave_sum(w0 + w1);
    const bool has0 = x0 != -INFINITY, has1 = x1 != -INFINITY;
    const unsigned long long b0 = __ballot(has0), b1 = __ballot(has1);
    if (lane == 0) sums[wave] = part, counts[wave] = __popcll(b0) + __popcll(b1);
    __syncthreads();
    const float sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    int at = 0, m = 0;
    for (int i = 0; i < 4; i++) {
        if (i < wave) at += counts[i];
        m += counts[i];
    }
    const unsigned long long below = ((unsigned long long)1 << lane) - 1;
    if (has0) {
        const int i = at + __popcll(b0 & below);
        list[i] = tid, w[i] = w0;
    }
    if (has1) {
        const int i = at + __popcll(b0) + __popcll(b1 & below);
        list[i] = tid + 256, w[i] = w1;
    }
    __syncthreads();
    const int pieces = a.d / V, groups = 256 / pieces, p = tid % pieces, g = tid / pieces;
    float acc[V] = {};
    if (g < groups) {
        const float *po = a.part_o + row * n * a.d + p * V;
        for (int i = g; i < m; i += 8 * groups) {
            float x[8][V], f[8];
#pragma unroll
            for (int u = 0; u < 8; u++) {
                const int k = i + u * groups;
                f[u] = k < m ? w[k] : 0.f;
                const float *at = po + (int64_t)list[k < m ? k : i] * a.d;
                if constexpr (V == 4)
                    *(float4 *)x[u] = *(const float4 *)at;
                else
                    x[u][0] = *at;
            }
#pragma unroll
            for (int u = 0; u < 8; u++)
#pragma unroll
                for (int c = 0; c < V; c++) acc[c] += i + u * groups < m ? f[u] * x[u][c] : 0.f;
        }
    }
#pragma unroll
    for (int c = 0; c < V; c++) red[tid * V + c] = acc[c];
    __syncthreads();
    if (tid < pieces) {
        const float inv = sum > 0.f ? 1.f / sum : 0.f;
#pragma unroll
        for (int c = 0; c < V; c++) {
            float t = red[tid * V + c];
            for (int i = 1; i < groups; i++) t += red[(i * pieces + tid) * V + c];
            st<DT>(o, row * a.d + tid * V + c, nan ? NAN : t * inv);
        }
    }
}

// The same for rows of at most 64 ranges and a D of pieces of 4, a wavefront a row: lane i has the weight of
// range i, and the lanes are D / 4 columns by 64 / (D / 4) groups.
template <int DT>
__global__ __launch_bounds__(256) void decode_shared_merge_few(SharedArgs a, int64_t rows, void *__restrict__ o) {
    __shared__ float w[4][64];
    __shared__ int32_t list[4][64];
    __shared__ float4 red[4][64];
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), n = a.nsp + a.nso;
    const int64_t row = (int64_t)blockIdx.x * 4 + wave;
    if (row >= rows) return;
    const float x = lane < n ? a.part_lse[row * n + lane] : -INFINITY;
    const bool nan = __any(x != x);
    const float top = wave_max(x);
    const float f = x == -INFINITY ? 0.f : (x == top ? 1.f : expf(x - top));
    const float sum = wave_sum(f);
    const unsigned long long has = __ballot(x != -INFINITY);
    const int m = __popcll(has);
    if (x != -INFINITY) {
        const int i = __popcll(has & (((unsigned long long)1 << lane) - 1));
        list[wave][i] = lane, w[wave][i] = f;
    }
    __builtin_amdgcn_wave_barrier();
    const int pieces = a.d / 4, groups = 64 / pieces, p = lane % pieces, g = lane / pieces;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (g < groups) {
        const float *po = a.part_o + row * n * a.d + p * 4;
        for (int i = g; i < m; i += 8 * groups) {
            float4 y[8];
            float fu[8];
#pragma unroll
            for (int u = 0; u < 8; u++) {
                const int k = i + u * groups;
                fu[u] = k < m ? w[wave][k] : 0.f;
                y[u] = *(const float4 *)(po + (int64_t)list[wave][k < m ? k : i] * a.d);
            }
#pragma unroll
            for (int u = 0; u < 8; u++) {
                const bool on = i + u * groups < m;
                acc.x += on ? fu[u] * y[u].x : 0.f, acc.y += on ? fu[u] * y[u].y : 0.f;
                acc.z += on ? fu[u] * y[u].z : 0.f, acc.w += on ? fu[u] * y[u].w : 0.f;
            }
        }
    }
    red[wave][lane] = acc;
    __builtin_amdgcn_wave_barrier();
    if (lane >= pieces) return;
    for (int i = 1; i < groups; i++) {
        const float4 y = red[wave][i * pieces + lane];
        acc.x += y.x, acc.y += y.y, acc.z += y.z, acc.w += y.w;
    }
    const float inv = nan ? NAN : (sum > 0.f ? 1.f / sum : 0.f);
    const float y[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
    if constexpr (DT == DM_F32)
        *(float4 *)((float *)o + row * a.d + lane * 4) = make_float4(y[0], y[1], y[2], y[3]);
    else
        *(uint2 *)((uint16_t *)o + row * a.d + lane * 4) = make_uint2(pack2<DT>(y[0], y[1]), pack2<DT>(y[2], y[3]));
}

// The 16-bit kernel's calls: 16-byte pieces, keys' and values' pages laid out alike, a page under 2 GB.
static bool shared_mfma_takes(const dm_attention_desc *d, int64_t page_size) {
    if ((d->dtype != DM_BF16 && d->dtype != DM_F16) || (d->d != 64 && d->d != 128 && d->d != 256) ||
        page_size % 16 != 0)
        return false;
    const int64_t most = (int64_t)1 << 30;
    if (!d->strided) return d->hkv * d->d < most / page_size;
    const dm_strides &k = d->sk, &v = d->sv;
    return d->sq.b % 8 == 0 && d->sq.h % 8 == 0 && k.b % 8 == 0 && k.t % 8 == 0 && k.h % 8 == 0 && v.h % 8 == 0 &&
           k.b == v.b && k.t == v.t && k.t >= d->d && k.b < most && k.t < most / page_size;
}

// The split of a call.
//
// Wide where a group has more than 32 rows a key-value head in the mean, a narrow tile's. (One group, 16384
// keys, 4 key-value heads, narrow and wide: 16 and 32 rows of 128: 19.1 and 20.1 us, 23.4 and 24.1; 48 and 64:
// 25.3 and 24.6, 25.0 and 25.2; 128: 31.6, 27.3. Rows of 64: 32 16.1, 19.1, 128 23.5, 20.9; rows of 256: 32 30.9,
// 35.0, 48 38.9, 35.9.)
//
// A prefix's item is a workgroup: about kPrefixItems of them, so that some compute units are left to the rows'
// own keys meanwhile (one reads, the other multiplies). (256 rows, 32768 + 512 keys and 64 rows, 16384 + 1024:
// 96 304 and 65 us, 128 238 and 66, 160 210 and 71, 192 197 and 72, 224 213 and 74, 256 218 and 77: the first call
// is bound by the prefix's products, the second by its own keys.) A row's own item is a wavefront (the
// generic kernel: a workgroup): about kOwnItems of them. (1024, with 192 at 222 and 75: 227 and 91 us; the small
// calls are alike.) No
// range is meant for fewer than 128 keys of a prefix (64: 8 rows of 6144 + 200 keys of 256 26 us, 128 20), 32 of a
// row's own, by the longest that the table can hold.
constexpr int64_t kPrefixItems = 192, kOwnItems = 2048, kGenericItems = 1024;
struct SharedPlan {
    bool wide;
    int32_t rows;  // rows of a prefix tile
    int64_t ptiles;
    int32_t otiles, nsp, nso;
    int64_t items;
};
static SharedPlan shared_plan(const dm_attention_desc *d, bool mfma, int64_t ngroups) {
    SharedPlan p{};
    const int64_t rep = d->hq / d->hkv;
    p.wide = mfma && ngroups > 0 && d->b * rep > 32 * ngroups;
    p.rows = p.wide ? (d->d == 256 ? 128 : 256) : 32;
    // (first_tile of the group behind the last)
    p.ptiles = ngroups > 0 && d->b * rep > 0 ? std::max<int64_t>(0, (d->b * rep - ngroups) / p.rows) + ngroups : 0;
    p.otiles = (int32_t)((rep + kOwnRows - 1) / kOwnRows);
    auto split = [&](int64_t tiles, int64_t target, int64_t keys) {
        const int64_t most = std::min<int64_t>(kSharedSplits / 2, (d->tk + keys - 1) / keys);
        return tiles > 0 ? (int32_t)std::max<int64_t>(1, std::min(most, target / tiles)) : 0;
    };
    p.nsp = split(p.ptiles * d->hkv, mfma ? kPrefixItems : kGenericItems, 128);
    p.nso = split(d->b * p.otiles * d->hkv, mfma ? kOwnItems : kGenericItems, mfma ? 32 : 128);
    p.items = (p.ptiles * p.nsp + d->b * p.otiles * p.nso) * d->hkv;
    return p;
}

// sizes whose products below fit 64 bits, keys whose ranges fit 32, and grids of fewer than 2^32 threads
static bool shared_sizes(const dm_attention_desc *d, int64_t ngroups) {
    const int64_t big = (int64_t)1 << 31;
    return d && d->hkv > 0 && d->b >= 0 && d->b < big && d->hq >= 0 && d->hq < 65536 && d->tk >= 0 &&
           d->tk <= (big >> 1) && d->d >= 0 && d->d <= 256 && ngroups >= 0 && ngroups < big &&
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
    if (p.wide && num_pages == 0) {  // (its kernel reads the first page in the place of one that is not there)
        fill_zero(o, rows * d->d * dtype_bytes(d->dtype), st);
        DM_LAUNCH_CHECK("attention_decode_shared: fill");
        return DM_OK;
    }
    SharedArgs a{};
    a.B = (int32_t)d->b, a.S = (int32_t)d->tk, a.left = (int32_t)left_of(d);
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
    a.nsp = p.nsp, a.nso = p.nso, a.ptiles = (int32_t)p.ptiles, a.otiles = p.otiles;
    const size_t parts = (size_t)rows * (p.nsp + p.nso);
    a.part_o = (float *)workspace;
    a.part_lse = (float *)((char *)workspace + align_up(parts * d->d * sizeof(float)));
    const int32_t items = (int32_t)p.items;
    // (the 16-bit kernel: a workgroup a prefix's item, a wavefront a row's, see decode_shared_mfma)
    const int64_t np = p.ptiles * p.nsp * d->hkv, waves = !mfma ? 1 : (p.wide && d->d != 256 ? 8 : 4);
    const unsigned g = (unsigned)(np + (p.items - np + waves - 1) / waves);
    // (8192 rows of 7 ranges: 10 us by wavefronts, 28 by workgroups; of more than 64, a workgroup)
    const bool few = p.nsp + p.nso <= 64 && d->d % 4 == 0 && aligned_16b(o);
#define SHARED_W(DT, D)                                                                            \
    if (p.wide)                                                                                    \
        decode_shared_mfma<DT, D, true><<<g, 64 * shared_waves<D, true>(), 0, st>>>(a, items, q, k_pages, v_pages); \
    else                                                                                           \
        decode_shared_mfma<DT, D, false><<<g, 64 * shared_waves<D, false>(), 0, st>>>(a, items, q, k_pages, v_pages)
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
    if (few)                                                                   \
        decode_shared_merge_few<DT><<<(unsigned)((rows + 3) / 4), 256, 0, st>>>(a, rows, o); \
    else if (d->d % 4 == 0)                                                    \
        decode_shared_merge<DT, 4><<<(unsigned)rows, 256, 0, st>>>(a, o);      \
    else                                                                       \
        decode_shared_merge<DT, 1><<<(unsigned)rows, 256, 0, st>>>(a, o)
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
