// The pages of a cache: reserved, forked, freed and compacted on the device, with nothing read back.
//
// A page is free where no row holds it (its count is 0). Whoever needs pages takes the free ones of
// the lowest indices, in the order of the rows or forks: a result that any implementation has, and
// one that keeps the pages in use together. The bookkeeping is a walk over the counts with prefix
// sums, by one workgroup (it is a few KB to a few hundred KB, and pages are handed out in order);
// copying pages is what costs bandwidth, and is spread over the card in 16 KB pieces.
//
// The walks are bound by latency: with 4096 pages and 128 rows, 64 forks are planned in 4.4 us and made
// (four layers' last pages, 16 MB at most) in 6.8, 128 rows' pages reserved in 4.6, 64 rows freed in 3.3,
// about 3 us of each a launch. Compaction is bound by its copies: 6000 pages of 32 KB in four pools half in use,
// 5.1 us of plan and 4.6 of counts in front of 68-80 us at 4.9 to 5.7 TB/s.
#include <algorithm>
#include <string>

#include "attention_kernels.h"
#include "dm_common.h"

namespace dm {

struct CacheArgs {
    int64_t rows, max_pages, num_pages, page_size;
    int32_t *table, *lengths, *counts;
};

constexpr int kPoolsPerLaunch = 32;
struct PoolArgs {
    int32_t n;
    struct {
        char *pages;
        int64_t bytes, stride;
    } at[kPoolsPerLaunch];
};

constexpr int kPlan = 1024;     // threads of a planning workgroup
constexpr int kPiece = 16384;   // bytes that a workgroup copies at a time

__device__ __forceinline__ int64_t keys_of(const CacheArgs &a, int64_t len) {
    const int64_t most = a.max_pages * a.page_size;
    return len < 0 ? 0 : (len > most ? most : len);
}
__device__ __forceinline__ int64_t pages_of(const CacheArgs &a, int64_t keys) {
    return (keys + a.page_size - 1) / a.page_size;
}

// The workgroup's exclusive prefix sums of x, and its total, in 32 bits (the host sees to it that the sums
// fit). For every thread of kPlan; `sums` is LDS, two turns of it, so that a scan costs one barrier.
struct PlanSums {
    int4 of[2][kPlan / 64 / 4];
};
__device__ __forceinline__ int32_t plan_scan(int32_t x, PlanSums &sums, int &turn, int32_t *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int32_t in = x;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int32_t y = __shfl_up(in, o, 64);
        if (lane >= o) in += y;
    }
    int4 *s = sums.of[turn];
    turn ^= 1;
    if (lane == 63) ((int32_t *)s)[wave] = in;
    __syncthreads();
    int32_t before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < kPlan / 64 / 4; i++) {
        const int4 v = s[i];
        const int32_t y[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int u = 0; u < 4; u++) {
            before += 4 * i + u < wave ? y[u] : 0;
            all += y[u];
        }
    }
    *total = all;
    return before + in - x;
}

// The counts of four pages from p on (1 past the last).
__device__ __forceinline__ int4 four_counts(const CacheArgs &a, int64_t p) {
    if (p + 4 <= a.num_pages && ((uintptr_t)a.counts & 15) == 0) return *(const int4 *)(a.counts + p);
    int4 x;
    x.x = p < a.num_pages ? a.counts[p] : 1, x.y = p + 1 < a.num_pages ? a.counts[p + 1] : 1;
    x.z = p + 2 < a.num_pages ? a.counts[p + 2] : 1, x.w = p + 3 < a.num_pages ? a.counts[p + 3] : 1;
    return x;
}

// Walks the counts from *cursor until `want` free pages are in `list` (lowest index first) or there
// are no more; *found and *cursor are the workgroup's. (`list` is written when the workgroup next meets.)
__device__ __forceinline__ void find_free(const CacheArgs &a, int64_t want, int32_t *list, int64_t *cursor,
                                          int32_t *found, PlanSums &sums, int &turn) {
    while (*found < want && *cursor < a.num_pages) {
        const int64_t i = *cursor + (int64_t)threadIdx.x * 4;
        const int4 c = four_counts(a, i);
        const bool is[4] = {c.x <= 0, c.y <= 0, c.z <= 0, c.w <= 0};
        int32_t total, at = *found + plan_scan(is[0] + is[1] + is[2] + is[3], sums, turn, &total);
#pragma unroll
        for (int u = 0; u < 4; u++)
            if (is[u]) list[at++] = (int32_t)(i + u);
        *found += total;
        *cursor += kPlan * 4;
    }
}

__global__ __launch_bounds__(kPlan) void cache_reserve_kernel(CacheArgs a, const int32_t *__restrict__ want,
                                                              uint8_t *__restrict__ granted, int32_t *list) {
    __shared__ PlanSums sums;
    __shared__ int32_t first[kPlan], need_of[kPlan], have_of[kPlan];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int turn = 0;
    int64_t cursor = 0, wanted = 0;
    int32_t found = 0;
    for (int64_t r0 = 0; r0 < a.rows; r0 += kPlan) {
        const int64_t r = r0 + tid;
        int64_t have = 0, need = 0, to = 0;
        bool fits = true, grows = false;
        if (r < a.rows) {
            const int64_t len = keys_of(a, a.lengths[r]);
            to = want[r];
            grows = to > len;
            fits = to <= a.max_pages * a.page_size;
            have = pages_of(a, len);
            need = grows && fits ? pages_of(a, to) - have : 0;
        }
        // (a need of more pages than there are is one of one more than there are: its sums fit)
        const int32_t asked = (int32_t)min(need, a.num_pages + 1);
        int32_t total;
        const int64_t at = wanted + plan_scan(asked, sums, turn, &total);
        wanted += total;
        find_free(a, min(wanted, a.num_pages), list, &cursor, &found, sums, turn);
        const bool ok = fits && (need == 0 || at + asked <= found);
        if (r < a.rows) {
            granted[r] = ok;
            if (ok && grows) a.lengths[r] = (int32_t)to;
        }
        first[tid] = (int32_t)min(at, (int64_t)INT32_MAX);
        need_of[tid] = ok ? (int32_t)need : 0;
        have_of[tid] = (int32_t)have;
        __syncthreads();
        // a wavefront the pages of 64 rows at a time: those of few by their lanes, long ones together
        for (int x0 = wave * 64; x0 < kPlan && r0 + x0 < a.rows; x0 += kPlan) {
            const int x = x0 + lane;
            const int mine = need_of[x];
            if (mine <= 8)
                for (int i = 0; i < mine; i++) {
                    const int32_t page = list[first[x] + i];
                    a.table[(r0 + x) * a.max_pages + have_of[x] + i] = page;
                    a.counts[page] = 1;
                }
            for (unsigned long long more = __ballot(mine > 8); more; more &= more - 1) {
                const int y = x0 + __builtin_ctzll(more), n = need_of[y];
                for (int i = lane; i < n; i += 64) {
                    const int32_t page = list[first[y] + i];
                    a.table[(r0 + y) * a.max_pages + have_of[y] + i] = page;
                    a.counts[page] = 1;
                }
            }
        }
        __syncthreads();
    }
}

// Which forks are made, and the pages of their own: held [n] is the keys that the child takes over, -1
// for a fork that is not made. The first fork that names a child has it: claim [rows], in LDS for tables
// of up to kClaims rows (its 16 KB; larger tables claim in the workspace, through the cache).
constexpr int kClaims = 4096;
template <bool LDS>
__global__ __launch_bounds__(kPlan) void cache_fork_plan(CacheArgs a, const int32_t *__restrict__ parents,
                                                         const int32_t *__restrict__ children, int64_t n,
                                                         int32_t *__restrict__ fresh, int32_t *__restrict__ held,
                                                         int32_t *claims, int32_t *list) {
    __shared__ PlanSums sums;
    __shared__ int32_t lds[LDS ? kClaims : 1];
    const int tid = threadIdx.x;
    int turn = 0;
    for (int64_t r = tid; r < a.rows; r += kPlan) {
        if constexpr (LDS)
            lds[r] = INT32_MAX;
        else
            __hip_atomic_store(claims + r, INT32_MAX, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    for (int64_t i = tid; i < n; i += kPlan) {
        const int64_t c = children[i];
        if (c >= 0 && c < a.rows) atomicMin(LDS ? lds + c : claims + c, (int32_t)i);
    }
    __syncthreads();
    int64_t cursor = 0, wanted = 0;
    int32_t found = 0;
    for (int64_t i0 = 0; i0 < n; i0 += kPlan) {
        const int64_t i = i0 + tid;
        int64_t keys = -1;
        if (i < n) {
            const int64_t p = parents[i], c = children[i];
            if (p >= 0 && p < a.rows && c >= 0 && c < a.rows && a.lengths[c] <= 0 &&
                (LDS ? lds[c] : __hip_atomic_load(claims + c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) == (int32_t)i)
                keys = keys_of(a, a.lengths[p]);
        }
        const bool part = keys > 0 && keys % a.page_size != 0;
        int32_t total;
        const int64_t at = wanted + plan_scan(part, sums, turn, &total);
        wanted += total;
        find_free(a, min(wanted, a.num_pages), list, &cursor, &found, sums, turn);
        __syncthreads();  // the list is written
        const bool ok = keys >= 0 && (!part || at < found);
        if (i < n) {
            held[i] = ok ? (int32_t)keys : -1;
            fresh[i] = ok ? (part ? list[at] : -1) : -2;
        }
    }
}

// One workgroup's copy of `bytes` from one place to another.
template <int VEC>
__device__ __forceinline__ void copy_bytes(char *__restrict__ to, const char *__restrict__ from, int64_t bytes) {
    if constexpr (VEC == 16) {
        const int n = (int)(bytes / 16);
        for (int i = threadIdx.x; i < n; i += 256 * 4) {
            // (four loads without conditions, the last piece again where there are fewer)
            const uint4 *f = (const uint4 *)from;
            uint4 *t = (uint4 *)to;
            const uint4 x0 = f[i], x1 = f[min(i + 256, n - 1)], x2 = f[min(i + 512, n - 1)], x3 = f[min(i + 768, n - 1)];
            t[i] = x0;
            if (i + 256 < n) t[i + 256] = x1;
            if (i + 512 < n) t[i + 512] = x2;
            if (i + 768 < n) t[i + 768] = x3;
        }
        for (int i = n * 16 + threadIdx.x; i < bytes; i += 256) to[i] = from[i];
    } else {
        for (int64_t i = threadIdx.x; i < bytes; i += 256) to[i] = from[i];
    }
}

// Block (i, 0, z): fork i's row of the table, its every gridDim.z-th share; block (i, 1 + x, z): the
// filled rows of the parent's last page in pool x, piece z.
template <int VEC>
__global__ __launch_bounds__(256) void cache_fork_apply(CacheArgs a, PoolArgs pools, bool tables,
                                                        const int32_t *__restrict__ parents,
                                                        const int32_t *__restrict__ children,
                                                        const int32_t *__restrict__ fresh,
                                                        const int32_t *__restrict__ held) {
    const int64_t i = blockIdx.x;
    const int64_t keys = held[i];
    if (keys < 0) return;
    const int64_t p = parents[i], c = children[i], whole = keys / a.page_size, rest = keys % a.page_size;
    const int32_t own = fresh[i];
    if (tables && blockIdx.y == 0) {
        const int32_t *src = a.table + p * a.max_pages;
        int32_t *dst = a.table + c * a.max_pages;
        for (int64_t j = (int64_t)blockIdx.z * 256 + threadIdx.x; j < whole; j += 256 * gridDim.z) {
            const int32_t page = src[j];
            dst[j] = page;
            if (page >= 0 && page < a.num_pages) atomicAdd(a.counts + page, 1);
        }
        if (blockIdx.z == 0 && threadIdx.x == 0) {
            if (own >= 0) {
                dst[whole] = own;
                a.counts[own] = 1;
            }
            a.lengths[c] = (int32_t)keys;
        }
        return;
    }
    if (own < 0) return;
    const int64_t from = a.table[p * a.max_pages + whole];
    if (from < 0 || from >= a.num_pages) return;
    const auto &pool = pools.at[blockIdx.y - tables];
    const int64_t bytes = rest * (pool.bytes / a.page_size);
    for (int64_t b = (int64_t)blockIdx.z * kPiece; b < bytes; b += (int64_t)gridDim.z * kPiece)
        copy_bytes<VEC>(pool.pages + own * pool.stride + b, pool.pages + from * pool.stride + b,
                        min((int64_t)kPiece, bytes - b));
}

// A workgroup a row. The length is taken in exchange for 0, so a row named twice is given up once.
__global__ __launch_bounds__(256) void cache_free_kernel(CacheArgs a, const int32_t *__restrict__ rows) {
    __shared__ int32_t len;
    const int64_t r = rows[blockIdx.x];
    if (r < 0 || r >= a.rows) return;
    if (threadIdx.x == 0) len = atomicExch(a.lengths + r, 0);
    __syncthreads();
    const int64_t n = pages_of(a, keys_of(a, len));
    int32_t *row = a.table + r * a.max_pages;
    for (int64_t j = threadIdx.x; j < n; j += 256) {
        const int32_t page = row[j];
        row[j] = -1;
        if (page >= 0 && page < a.num_pages) atomicSub(a.counts + page, 1);
    }
}

// Compaction in three launches (two for a single chunk): the pages in use counted by chunk; each chunk's holes and movers put
// in their places of the two lists (moved holds -2 - place for a mover until the last launch); the
// pages, counts and entries moved.
constexpr int kChunk = kPlan * 4;
struct CompactWork {
    int64_t nchunks;
    int32_t *movers_n;  // how many pages move
    int32_t *chunks;    // [nchunks] pages in use
    int32_t *holes, *movers;
};

__device__ __forceinline__ void uses(const CacheArgs &a, int64_t p, int32_t (&is)[4]) {
    const int4 c = four_counts(a, p);
    is[0] = p < a.num_pages && c.x > 0, is[1] = p + 1 < a.num_pages && c.y > 0;
    is[2] = p + 2 < a.num_pages && c.z > 0, is[3] = p + 3 < a.num_pages && c.w > 0;
}

__global__ __launch_bounds__(kPlan) void cache_compact_count(CacheArgs a, CompactWork w) {
    __shared__ PlanSums sums;
    int turn = 0;
    int32_t is[4], total;
    uses(a, (int64_t)blockIdx.x * kChunk + threadIdx.x * 4, is);
    plan_scan(is[0] + is[1] + is[2] + is[3], sums, turn, &total);
    if (threadIdx.x == 0) w.chunks[blockIdx.x] = total;
}

__global__ __launch_bounds__(kPlan) void cache_compact_plan(CacheArgs a, CompactWork w, int32_t *__restrict__ moved) {
    __shared__ PlanSums sums;
    int turn = 0;
    const int tid = threadIdx.x;
    const int64_t p0 = (int64_t)blockIdx.x * kChunk + tid * 4;
    int32_t is[4], total;
    uses(a, p0, is);
    int32_t before = 0, all = 0;  // the pages in use in front of this chunk, and altogether
    if (w.nchunks == 1) plan_scan(is[0] + is[1] + is[2] + is[3], sums, turn, &all);
    for (int64_t c0 = 0; w.nchunks > 1 && c0 < w.nchunks; c0 += kPlan) {
        const int64_t c = c0 + tid;
        const int32_t x = c < w.nchunks ? w.chunks[c] : 0;
        // (one scan: what lies in front of this chunk's place in it is the sum in front of it)
        __shared__ int32_t front;
        const int32_t sum = plan_scan(x, sums, turn, &total);
        if (c == (int64_t)blockIdx.x) front = all + sum;
        __syncthreads();
        if ((int64_t)blockIdx.x >= c0 && (int64_t)blockIdx.x < c0 + kPlan) before = front;
        all += total;
    }
    // the pages in use below index n = all: those stay
    const int64_t cn = all / kChunk;
    int32_t stay = 0;
    for (int64_t c0 = 0; c0 < cn; c0 += kPlan) {
        const int64_t c = c0 + tid;
        plan_scan(c < cn ? (w.nchunks > 1 ? w.chunks[c] : all) : 0, sums, turn, &total);
        stay += total;
    }
    int32_t last[4], mine = 0;
    const int64_t q0 = cn * kChunk + tid * 4;
    uses(a, q0, last);
#pragma unroll
    for (int u = 0; u < 4; u++) mine += q0 + u < all && last[u];
    plan_scan(mine, sums, turn, &total);
    stay += total;
    if (blockIdx.x == 0 && tid == 0) *w.movers_n = all - stay;
    int32_t live = before + plan_scan(is[0] + is[1] + is[2] + is[3], sums, turn, &total);  // pages in use below p
#pragma unroll
    for (int u = 0; u < 4; u++) {
        const int64_t p = p0 + u;
        if (p >= a.num_pages) break;
        int32_t to = -1;
        if (is[u]) {
            if (p < all) {
                to = (int32_t)p;
            } else {
                const int32_t k = live - stay;
                w.movers[k] = (int32_t)p;
                to = -2 - k;
            }
            live++;
        } else if (p < all) {
            w.holes[p - live] = (int32_t)p;
        }
        moved[p] = to;
    }
}

// Blocks 0 .. nchunks4 - 1: the new indices and counts (256 pages each); then nrows blocks: the rows'
// entries; the rest copy pages. (A row's entry is the same from a mover's place and from its final
// index, so those blocks need not wait for one another.)
template <int VEC>
__global__ __launch_bounds__(256) void cache_compact_apply(CacheArgs a, PoolArgs pools, CompactWork w, int64_t nindex,
                                                           int64_t nrows, int64_t pieces,
                                                           int32_t *moved) {
    int64_t block = blockIdx.x;
    if (block < nindex) {
        const int64_t p = block * 256 + threadIdx.x;
        if (p >= a.num_pages) return;
        const int32_t x = moved[p];
        if (x > -2) return;
        const int32_t to = w.holes[-2 - x];
        a.counts[to] = a.counts[p];
        a.counts[p] = 0;
        moved[p] = to;
        return;
    }
    block -= nindex;
    if (block < nrows) {
        for (int64_t r = block; r < a.rows; r += nrows) {
            const int64_t n = pages_of(a, keys_of(a, a.lengths[r]));
            for (int64_t j = threadIdx.x; j < n; j += 256) {
                const int32_t page = a.table[r * a.max_pages + j];
                if (page < 0 || page >= a.num_pages) continue;
                const int32_t x = __hip_atomic_load(moved + page, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                a.table[r * a.max_pages + j] = x > -2 ? x : w.holes[-2 - x];
            }
        }
        return;
    }
    block -= nrows;
    const int64_t blocks = gridDim.x - nindex - nrows;
    const int64_t n = (int64_t)*w.movers_n * pools.n * pieces;
    for (int64_t x = block; x < n; x += blocks) {
        const int64_t b = x % pieces * kPiece, k = x / pieces / pools.n;
        const auto &pool = pools.at[x / pieces % pools.n];
        if (b >= pool.bytes) continue;
        copy_bytes<VEC>(pool.pages + w.holes[k] * pool.stride + b, pool.pages + w.movers[k] * pool.stride + b,
                        min((int64_t)kPiece, pool.bytes - b));
    }
}

static const int64_t kI31 = (int64_t)1 << 31;
static const int64_t kMostPages = ((int64_t)1 << 21) - 1;  // a planning workgroup's sums of 1024 needs fit 32 bits
static const int64_t kMostRows = (int64_t)1 << 22;  // rows of a call: a workgroup each, under 2^32 threads

static bool table_sizes(const dm_cache_table *t) {
    return t && t->rows >= 0 && t->rows < kI31 && t->max_pages >= 0 && t->max_pages < kI31 && t->num_pages >= 0 &&
           t->num_pages < kMostPages && t->page_size >= 1 && t->page_size < kI31;
}

static int check_table(const std::string &op, const dm_cache_table *t) {
    if (!t) return refuse(op + ": null table");
    if (!table_sizes(t))
        return refuse(op + ": page_size must be positive, rows, max_pages and num_pages not negative, the pages "
                           "fewer than 2^21");
    if ((t->rows > 0 && !t->lengths) || (t->rows * t->max_pages > 0 && !t->block_table) ||
        (t->num_pages > 0 && !t->refcounts))
        return refuse(op + ": the block table, the lengths or the page counts are missing");
    return DM_OK;
}

static CacheArgs cache_args(const dm_cache_table *t) {
    return CacheArgs{t->rows, t->max_pages, t->num_pages, t->page_size, t->block_table, t->lengths, t->refcounts};
}

static int check_pools(const std::string &op, const dm_cache_table *t, const dm_cache_pool *pools, int64_t n) {
    if (n < 0 || (n > 0 && !pools)) return refuse(op + ": the pools are missing");
    for (int64_t i = 0; i < n; i++) {
        const dm_cache_pool &p = pools[i];
        if (p.page_bytes < 0 || p.page_bytes % t->page_size != 0 || p.page_stride < p.page_bytes ||
            p.page_bytes > ((int64_t)1 << 40) || (t->num_pages > 0 && p.page_stride > ((int64_t)1 << 60) / t->num_pages))
            return refuse(op + ": a pool's pages are page_size rows of as many bytes each, and apart");
        if (t->num_pages > 0 && p.page_bytes > 0 && !p.pages) return refuse(op + ": a pool's pages are missing");
    }
    return DM_OK;
}

// The pools from `at` on that one launch takes, whether every copy of theirs can be made in 16-byte
// pieces (a fork's begin at rows: only their starts need the alignment), and the pieces of the largest page.
static PoolArgs pools_of(const dm_cache_pool *pools, int64_t n, int64_t at, bool *wide, int64_t *pieces) {
    PoolArgs a{};
    a.n = (int32_t)std::min<int64_t>(kPoolsPerLaunch, n - at);
    *wide = true;
    *pieces = 1;
    for (int i = 0; i < a.n; i++) {
        const dm_cache_pool &p = pools[at + i];
        a.at[i].pages = (char *)p.pages, a.at[i].bytes = p.page_bytes, a.at[i].stride = p.page_stride;
        *wide = *wide && ((uintptr_t)p.pages | (uintptr_t)p.page_stride) % 16 == 0;
        *pieces = std::max(*pieces, (p.page_bytes + kPiece - 1) / kPiece);
    }
    return a;
}

}  // namespace dm

using namespace dm;

extern "C" {

size_t dm_cache_reserve_workspace(const dm_cache_table *t) {
    return table_sizes(t) ? align_up((size_t)t->num_pages * sizeof(int32_t)) : 0;
}

int dm_cache_reserve(const dm_cache_table *t, const int32_t *new_lengths, uint8_t *granted, void *workspace,
                     size_t workspace_bytes, void *stream) {
    const std::string op("cache_reserve");
    if (int rc = check_table(op, t)) return rc;
    if (workspace_bytes < dm_cache_reserve_workspace(t))
        return refuse(op + ": the workspace is smaller than dm_cache_reserve_workspace");
    if (t->rows == 0) return DM_OK;
    if (!new_lengths || !granted) return refuse(op + ": the new lengths or the results' place are missing");
    cache_reserve_kernel<<<1, kPlan, 0, (hipStream_t)stream>>>(cache_args(t), new_lengths, granted,
                                                               (int32_t *)workspace);
    probe_add(DM_PROBE_CACHE_RESERVE);
    DM_LAUNCH_CHECK("cache_reserve: launch");
    return DM_OK;
}

size_t dm_cache_fork_workspace(const dm_cache_table *t, int64_t n) {
    if (!table_sizes(t) || n < 0 || n > kMostRows) return 0;
    return align_up((size_t)n * 4) + align_up((size_t)t->rows * 4) + align_up((size_t)t->num_pages * 4);
}

int dm_cache_fork(const dm_cache_table *t, const dm_cache_pool *pools, int64_t npools, const int32_t *parents,
                  const int32_t *children, int64_t n, int32_t *fresh, void *workspace, size_t workspace_bytes,
                  void *stream) {
    const std::string op("cache_fork");
    if (int rc = check_table(op, t)) return rc;
    if (int rc = check_pools(op, t, pools, npools)) return rc;
    if (n < 0 || n > kMostRows) return refuse(op + ": the parents and children are [N], N at most 2^22");
    if (workspace_bytes < dm_cache_fork_workspace(t, n))
        return refuse(op + ": the workspace is smaller than dm_cache_fork_workspace");
    if (n == 0) return DM_OK;
    if (!parents || !children || !fresh)
        return refuse(op + ": the parents, the children or the results' place are missing");
    hipStream_t st = (hipStream_t)stream;
    const CacheArgs a = cache_args(t);
    int32_t *held = (int32_t *)workspace;
    int32_t *claim = (int32_t *)((char *)workspace + align_up((size_t)n * 4));
    int32_t *list = (int32_t *)((char *)claim + align_up((size_t)t->rows * 4));
    if (t->rows <= kClaims)
        cache_fork_plan<true><<<1, kPlan, 0, st>>>(a, parents, children, n, fresh, held, claim, list);
    else
        cache_fork_plan<false><<<1, kPlan, 0, st>>>(a, parents, children, n, fresh, held, claim, list);
    for (int64_t at = 0; at == 0 || at < npools; at += kPoolsPerLaunch) {
        bool wide;
        int64_t pieces;
        const PoolArgs pa = pools_of(pools, npools, at, &wide, &pieces);
        const dim3 grid((unsigned)n, (unsigned)(pa.n + (at == 0)), (unsigned)std::min<int64_t>(pieces, 64));
        if (wide)
            cache_fork_apply<16><<<grid, 256, 0, st>>>(a, pa, at == 0, parents, children, fresh, held);
        else
            cache_fork_apply<1><<<grid, 256, 0, st>>>(a, pa, at == 0, parents, children, fresh, held);
    }
    probe_add(DM_PROBE_CACHE_FORK);
    DM_LAUNCH_CHECK("cache_fork: launch");
    return DM_OK;
}

int dm_cache_free(const dm_cache_table *t, const int32_t *rows, int64_t n, void *stream) {
    const std::string op("cache_free");
    if (int rc = check_table(op, t)) return rc;
    if (n < 0 || n > kMostRows) return refuse(op + ": the rows are [N], N at most 2^22");
    if (n == 0) return DM_OK;
    if (!rows) return refuse(op + ": the rows are missing");
    cache_free_kernel<<<(unsigned)n, 256, 0, (hipStream_t)stream>>>(cache_args(t), rows);
    probe_add(DM_PROBE_CACHE_FREE);
    DM_LAUNCH_CHECK("cache_free: launch");
    return DM_OK;
}

size_t dm_cache_compact_workspace(const dm_cache_table *t) {
    if (!table_sizes(t)) return 0;
    const int64_t nchunks = (t->num_pages + kChunk - 1) / kChunk;
    return 256 + align_up((size_t)nchunks * 4) + 2 * align_up((size_t)t->num_pages * 4);
}

int dm_cache_compact(const dm_cache_table *t, const dm_cache_pool *pools, int64_t npools, int32_t *moved,
                     void *workspace, size_t workspace_bytes, void *stream) {
    const std::string op("cache_compact");
    if (int rc = check_table(op, t)) return rc;
    if (int rc = check_pools(op, t, pools, npools)) return rc;
    if (workspace_bytes < dm_cache_compact_workspace(t))
        return refuse(op + ": the workspace is smaller than dm_cache_compact_workspace");
    if (t->num_pages == 0) return DM_OK;
    if (!moved) return refuse(op + ": the results' place is missing");
    hipStream_t st = (hipStream_t)stream;
    const CacheArgs a = cache_args(t);
    CompactWork w{};
    w.nchunks = (t->num_pages + kChunk - 1) / kChunk;
    char *at = (char *)workspace;
    w.movers_n = (int32_t *)at;
    w.chunks = (int32_t *)(at += 256);
    w.holes = (int32_t *)(at += align_up((size_t)w.nchunks * 4));
    w.movers = (int32_t *)(at += align_up((size_t)t->num_pages * 4));
    if (w.nchunks > 1) cache_compact_count<<<(unsigned)w.nchunks, kPlan, 0, st>>>(a, w);  // (one: the plan counts it)
    cache_compact_plan<<<(unsigned)w.nchunks, kPlan, 0, st>>>(a, w, moved);
    for (int64_t i = 0; i == 0 || i < npools; i += kPoolsPerLaunch) {
        bool wide;
        int64_t pieces;
        const PoolArgs pa = pools_of(pools, npools, i, &wide, &pieces);
        const int64_t nindex = i == 0 ? (t->num_pages + 255) / 256 : 0;
        const int64_t nrows = i == 0 ? std::min<int64_t>(t->rows, 1024) : 0;
        const int64_t ncopy = pa.n > 0 ? std::min<int64_t>(2048, t->num_pages * pa.n * pieces) : 0;
        const unsigned grid = (unsigned)(nindex + nrows + ncopy);
        if (grid == 0) continue;
        if (wide)
            cache_compact_apply<16><<<grid, 256, 0, st>>>(a, pa, w, nindex, nrows, pieces, moved);
        else
            cache_compact_apply<1><<<grid, 256, 0, st>>>(a, pa, w, nindex, nrows, pieces, moved);
    }
    probe_add(DM_PROBE_CACHE_COMPACT);
    DM_LAUNCH_CHECK("cache_compact: launch");
    return DM_OK;
}

}  // extern "C"
