// The pages of a cache: reserved, forked, freed and compacted on the device, with nothing read back.
//
// A page is free where no row holds it (its count is 0). Whoever needs pages takes the free ones of
// the lowest indices, in the order of the rows or forks: a result that any implementation has, and
// one that keeps the pages in use together. The bookkeeping is a walk over the counts with prefix
// sums, by one workgroup (it is a few KB to a few hundred KB, and pages are handed out in order);
// copying pages is what costs bandwidth, and is spread over the card in 16 KB pieces.
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

// The workgroup's exclusive prefix sums of x, and its total. For every thread of kPlan; `sums` is LDS.
__device__ __forceinline__ int64_t plan_scan(int64_t x, int64_t *sums, int64_t *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t in = x;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t y = __shfl_up(in, o, 64);
        if (lane >= o) in += y;
    }
    __syncthreads();
    if (lane == 63) sums[wave] = in;
    __syncthreads();
    int64_t before = 0, all = 0;
    for (int w = 0; w < kPlan / 64; w++) {
        const int64_t s = sums[w];
        if (w < wave) before += s;
        all += s;
    }
    *total = all;
    return before + in - x;
}

// Walks the counts from *cursor until `want` free pages are in `list` (lowest index first) or there
// are no more; *found and *cursor are the workgroup's.
__device__ __forceinline__ void find_free(const CacheArgs &a, int64_t want, int32_t *list, int64_t *cursor,
                                          int64_t *found, int64_t *sums) {
    while (*found < want && *cursor < a.num_pages) {
        const int64_t i = *cursor + (int64_t)threadIdx.x * 4;
        bool is[4];
        int64_t mine = 0, total;
#pragma unroll
        for (int u = 0; u < 4; u++) {
            is[u] = i + u < a.num_pages && a.counts[i + u] <= 0;
            mine += is[u];
        }
        int64_t at = *found + plan_scan(mine, sums, &total);
#pragma unroll
        for (int u = 0; u < 4; u++)
            if (is[u]) list[at++] = (int32_t)(i + u);
        *found += total;
        *cursor += kPlan * 4;
    }
    __syncthreads();  // the list is written
}

__global__ __launch_bounds__(kPlan) void cache_reserve_kernel(CacheArgs a, const int32_t *__restrict__ want,
                                                              uint8_t *__restrict__ granted, int32_t *list) {
    __shared__ int64_t sums[kPlan / 64];
    __shared__ int32_t first[kPlan], need_of[kPlan], have_of[kPlan];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int64_t cursor = 0, found = 0, wanted = 0;
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
        int64_t total;
        const int64_t at = wanted + plan_scan(need, sums, &total);
        wanted += total;
        find_free(a, min(wanted, a.num_pages), list, &cursor, &found, sums);
        const bool ok = fits && (need == 0 || at + need <= found);
        if (r < a.rows) {
            granted[r] = ok;
            if (ok && grows) a.lengths[r] = (int32_t)to;
        }
        first[tid] = (int32_t)min(at, (int64_t)INT32_MAX);
        need_of[tid] = ok ? (int32_t)need : 0;
        have_of[tid] = (int32_t)have;
        __syncthreads();
        for (int x = wave; x < kPlan && r0 + x < a.rows; x += kPlan / 64)
            for (int i = lane; i < need_of[x]; i += 64) {
                const int32_t page = list[first[x] + i];
                a.table[(r0 + x) * a.max_pages + have_of[x] + i] = page;
                a.counts[page] = 1;
            }
        __syncthreads();
    }
}

// Which forks are made, and the pages of their own: held [n] is the keys that the child takes over, -1
// for a fork that is not made. claim [rows]: the first fork that names a child.
__global__ __launch_bounds__(kPlan) void cache_fork_plan(CacheArgs a, const int32_t *__restrict__ parents,
                                                         const int32_t *__restrict__ children, int64_t n,
                                                         int32_t *__restrict__ fresh, int32_t *__restrict__ held,
                                                         int32_t *claim, int32_t *list) {
    __shared__ int64_t sums[kPlan / 64];
    const int tid = threadIdx.x;
    for (int64_t r = tid; r < a.rows; r += kPlan)
        __hip_atomic_store(claim + r, INT32_MAX, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    for (int64_t i = tid; i < n; i += kPlan) {
        const int64_t c = children[i];
        if (c >= 0 && c < a.rows) atomicMin(claim + c, (int32_t)i);
    }
    __syncthreads();
    int64_t cursor = 0, found = 0, wanted = 0;
    for (int64_t i0 = 0; i0 < n; i0 += kPlan) {
        const int64_t i = i0 + tid;
        int64_t keys = -1;
        if (i < n) {
            const int64_t p = parents[i], c = children[i];
            if (p >= 0 && p < a.rows && c >= 0 && c < a.rows && a.lengths[c] <= 0 &&
                __hip_atomic_load(claim + c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (int32_t)i)
                keys = keys_of(a, a.lengths[p]);
        }
        const bool part = keys > 0 && keys % a.page_size != 0;
        int64_t total;
        const int64_t at = wanted + plan_scan(part, sums, &total);
        wanted += total;
        find_free(a, min(wanted, a.num_pages), list, &cursor, &found, sums);
        const bool ok = keys >= 0 && (!part || at < found);
        if (i < n) {
            held[i] = ok ? (int32_t)keys : -1;
            fresh[i] = ok ? (part ? list[at] : -1) : -2;
        }
        __syncthreads();
    }
}

// One workgroup's copy of `bytes` from one place to another.
template <int VEC>
__device__ __forceinline__ void copy_bytes(char *__restrict__ to, const char *__restrict__ from, int64_t bytes) {
    if constexpr (VEC == 16) {
        const int64_t n = bytes / 16;
        for (int64_t i = threadIdx.x; i < n; i += 256 * 4) {
            uint4 x[4];
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (i + 256 * u < n) x[u] = ((const uint4 *)from)[i + 256 * u];
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (i + 256 * u < n) ((uint4 *)to)[i + 256 * u] = x[u];
        }
        for (int64_t i = n * 16 + threadIdx.x; i < bytes; i += 256) to[i] = from[i];
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

// Compaction in three launches: the pages in use counted by chunk; each chunk's holes and movers put
// in their places of the two lists (moved holds -2 - place for a mover until the last launch); the
// pages, counts and entries moved.
constexpr int kChunk = kPlan * 4;
struct CompactWork {
    int64_t nchunks;
    int32_t *movers_n;  // how many pages move
    int32_t *chunks;    // [nchunks] pages in use
    int32_t *holes, *movers;
};

__device__ __forceinline__ int in_use(const CacheArgs &a, int64_t p) { return p < a.num_pages && a.counts[p] > 0; }

__global__ __launch_bounds__(kPlan) void cache_compact_count(CacheArgs a, CompactWork w) {
    __shared__ int64_t sums[kPlan / 64];
    const int64_t p = (int64_t)blockIdx.x * kChunk + threadIdx.x * 4;
    int64_t total;
    plan_scan(in_use(a, p) + in_use(a, p + 1) + in_use(a, p + 2) + in_use(a, p + 3), sums, &total);
    if (threadIdx.x == 0) w.chunks[blockIdx.x] = (int32_t)total;
}

__global__ __launch_bounds__(kPlan) void cache_compact_plan(CacheArgs a, CompactWork w, int32_t *__restrict__ moved) {
    __shared__ int64_t sums[kPlan / 64];
    const int tid = threadIdx.x;
    int64_t total, before = 0, all = 0;
    for (int64_t c0 = 0; c0 < w.nchunks; c0 += kPlan) {
        const int64_t c = c0 + tid, x = c < w.nchunks ? w.chunks[c] : 0;
        int64_t mine;
        plan_scan(c < (int64_t)blockIdx.x ? x : 0, sums, &mine);
        before += mine;
        plan_scan(x, sums, &total);
        all += total;
    }
    // the pages in use below index n = all: those stay
    const int64_t cn = all / kChunk;
    int64_t stay = 0;
    for (int64_t c0 = 0; c0 < cn; c0 += kPlan) {
        const int64_t c = c0 + tid;
        plan_scan(c < cn ? w.chunks[c] : 0, sums, &total);
        stay += total;
    }
    int64_t mine = 0;
    for (int u = 0; u < 4; u++) {
        const int64_t p = cn * kChunk + tid * 4 + u;
        mine += p < all && in_use(a, p);
    }
    plan_scan(mine, sums, &total);
    stay += total;
    if (blockIdx.x == 0 && tid == 0) *w.movers_n = (int32_t)(all - stay);
    const int64_t p0 = (int64_t)blockIdx.x * kChunk + tid * 4;
    int is[4];
    mine = 0;
    for (int u = 0; u < 4; u++) mine += is[u] = in_use(a, p0 + u);
    int64_t live = before + plan_scan(mine, sums, &total);  // pages in use below p
    for (int u = 0; u < 4; u++) {
        const int64_t p = p0 + u;
        if (p >= a.num_pages) break;
        int32_t to = -1;
        if (is[u]) {
            if (p < all) {
                to = (int32_t)p;
            } else {
                const int64_t k = live - stay;
                w.movers[k] = (int32_t)p;
                to = (int32_t)(-2 - k);
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
static const int64_t kMostRows = (int64_t)1 << 22;  // rows of a call: a workgroup each, under 2^32 threads

static bool table_sizes(const dm_cache_table *t) {
    return t && t->rows >= 0 && t->rows < kI31 && t->max_pages >= 0 && t->max_pages < kI31 && t->num_pages >= 0 &&
           t->num_pages < kI31 - 8192 && t->page_size >= 1 && t->page_size < kI31;
}

static int check_table(const std::string &op, const dm_cache_table *t) {
    if (!t) return refuse(op + ": null table");
    if (!table_sizes(t))
        return refuse(op + ": page_size must be positive, rows, max_pages and num_pages not negative");
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
    cache_fork_plan<<<1, kPlan, 0, st>>>(a, parents, children, n, fresh, held, claim, list);
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
    cache_compact_count<<<(unsigned)w.nchunks, kPlan, 0, st>>>(a, w);
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
