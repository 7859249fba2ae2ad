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
#include <new>
#include <string>
#include <utility>
#include <vector>

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

// ------------------------------------------------------------------------------------------
// Eviction
// ------------------------------------------------------------------------------------------
//
// Three launches. A workgroup a row finds what has to stay and the weight of the last key that stays of the others, by
// three counts of 11, 11 and 10 bits of the weights' order. Then a workgroup for every kPlan * 4 keys or more of a row
// gives the keys that stay their places, counting those in front of its own for itself (a walk by one workgroup was
// 27 us of 55 for 31000 keys, all of it instructions). At last the keys move down in every pool, a workgroup for a
// column of each: its loads of a step's keys have all arrived before it stores one of them, and what it stores to
// lies in front of all that it has yet to load, so that no order among workgroups is needed. Wide columns read memory
// in long runs, narrow ones are more workgroups with more keys a step.
//
// 16 rows of up to 4096 keys cut to 2048 in two layers' pools (537 MB): 8.4, 6.9 and 103 us, bound by the moves (5.2 TB/s).
// A row of 32768 keys cut to 4096: 18 (one workgroup reads it three times), 11 and 31 (a chain of steps).

// What the first launch leaves of a row, and the second for the copies: key j of [first, n) comes from page and row
// from[j] of the pool to to[j] (page kNoPage: one outside the pools), its weight is weight[j].
struct EvictRow {
    int32_t held, n, fixed, until;  // keys, those that stay; the keys [fixed, until) may go,
    uint32_t bar;                   // of which those above the bar stay and the first `ties` that equal it
    int32_t ties, first;
};
struct EvictWork {
    EvictRow *rows;
    uint2 *from, *to;  // [rows, max_pages * page_size]
    float *weight;
    int64_t cap;
};
constexpr uint32_t kNoPage = 0xffffffffu;
typedef uint32_t u32x2_vec __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_vec __attribute__((ext_vector_type(4)));
typedef float f32x4_unaligned __attribute__((ext_vector_type(4), aligned(4)));

// A float's place in the order of weights: -0 as 0, NaN above all.
__device__ __forceinline__ uint32_t weight_order(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ __launch_bounds__(kPlan) void cache_evict_select(CacheArgs a, const float *__restrict__ weights, int64_t stride,
                                                            const int32_t *__restrict__ budgets, int64_t recent,
                                                            EvictWork w) {
    __shared__ PlanSums sums;
    __shared__ int32_t hist[2048], shared_to, chosen, above;
    const int tid = threadIdx.x;
    const int64_t r = blockIdx.x;
    const int32_t held = (int32_t)keys_of(a, a.lengths[r]), budget = max(budgets[r], 0);
    const int32_t *row = a.table + r * a.max_pages;
    const float *wr = weights + r * stride;
    int turn = 0;
    if (tid == 0) shared_to = 0;
    __syncthreads();
    // the pages up to the last that another row holds stay
    const int32_t np = (int32_t)pages_of(a, held);
    int32_t most = 0;
    for (int32_t c = tid; c < np && held > budget; c += kPlan) {
        const int32_t page = row[c];
        if (page >= 0 && page < a.num_pages && a.counts[page] > 1) most = c + 1;
    }
    if (most) atomicMax(&shared_to, most);
    __syncthreads();
    const int32_t fixed = (int32_t)min((int64_t)held, shared_to * a.page_size);
    const int32_t until = max(fixed, held - (int32_t)min(recent, (int64_t)budget));
    const int32_t must = held - (until - fixed), n = min(held, max(budget, must));
    const int32_t need = n - must;
    uint32_t bar = 0xffffffffu;
    int32_t ties = 0;
    if (n < held && need > 0) {
        uint32_t prefix = 0, mask = 0;
        int32_t left = need;
        for (int pass = 0; pass < 3; pass++) {
            const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bins = pass == 2 ? 1024 : 2048;
            for (int i = tid; i < 2048; i += kPlan) hist[i] = 0;
            __syncthreads();
            auto count = [&](float y) {
                const uint32_t x = weight_order(y);
                if ((x & mask) == prefix) atomicAdd(&hist[(x >> shift) & (bins - 1)], 1);
            };
            const int32_t whole = fixed + (until - fixed) / (4 * kPlan) * (4 * kPlan);
#pragma unroll 4
            for (int32_t j = fixed; j < whole; j += 4 * kPlan) {
                const f32x4_unaligned y = *(const f32x4_unaligned *)(wr + j + 4 * tid);
                count(y[0]), count(y[1]), count(y[2]), count(y[3]);
            }
            for (int32_t j = whole + tid; j < until; j += kPlan) count(wr[j]);
            __syncthreads();
            // from the largest bin down: the one in which the count reaches `left`
            const int b1 = 2047 - 2 * tid, b0 = b1 - 1;
            const int32_t c1 = hist[b1], c0 = hist[b0];
            int32_t total;
            const int32_t before = plan_scan(c0 + c1, sums, turn, &total);
            if (before < left && before + c1 >= left) chosen = b1, above = before;
            if (before + c1 < left && before + c1 + c0 >= left) chosen = b0, above = before + c1;
            __syncthreads();
            prefix |= (uint32_t)chosen << shift;
            mask |= (uint32_t)(bins - 1) << shift;
            left -= above;
            __syncthreads();
        }
        bar = prefix, ties = left;
    }
    if (tid == 0) w.rows[r] = EvictRow{held, n, fixed, until, bar, ties, n};
}

// Workgroup (share, row): the keys of the row's share, a wavefront 256 of a step's 4096 in four rows of its lanes (so
// that the lanes' stores lie side by side). A key's place: the keys above the bar in front of it, and the ties taken.
constexpr int kEvictShares = 64;  // most shares of a row
__global__ __launch_bounds__(kPlan) void cache_evict_place(CacheArgs a, const float *__restrict__ weights, int64_t stride,
                                                           int32_t *__restrict__ kept, EvictWork w) {
    __shared__ int4 sums[2][kPlan / 64 / 4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t r = blockIdx.y;
    const EvictRow er = w.rows[r];
    const int32_t size = (int32_t)min(a.page_size, (int64_t)1 << 30);
    const int32_t steps = (er.held + 4 * kPlan - 1) / (4 * kPlan), share = (steps + gridDim.x - 1) / gridDim.x * 4 * kPlan;
    const int64_t from = (int64_t)blockIdx.x * share, cap = w.cap;
    int32_t *out = kept + r * cap;
    // behind the row, a part for each workgroup
    for (int64_t j = er.n + (int64_t)blockIdx.x * kPlan + tid; j < cap; j += (int64_t)gridDim.x * kPlan) out[j] = -1;
    if (from >= er.held) return;
    const int32_t begin = (int32_t)from, end = (int32_t)min((int64_t)er.held, from + share);
    if (er.n == er.held) {
        for (int32_t j = begin + tid; j < end; j += kPlan) out[j] = j;
        return;
    }
    const float *wr = weights + r * stride;
    const int32_t *row = a.table + r * a.max_pages;
    // the keys in front of the share: those that have to stay in closed form, the others counted
    int32_t over = min(begin, er.fixed) + max(0, begin - er.until), equal = 0;
    const bool takes = er.n > er.held - (er.until - er.fixed);  // some of those that may go stay
    int turn = 0;
    auto meet = [&](int32_t packed, int32_t *before, int32_t *total) __attribute__((always_inline)) {
        int32_t *all = (int32_t *)sums[turn];
        turn ^= 1;
        if (lane == 0) all[wave] = packed;
        __syncthreads();
        *before = *total = 0;
#pragma unroll
        for (int i = 0; i < kPlan / 64; i++) {
            *before += i < wave ? all[i] : 0;
            *total += all[i];
        }
    };
    if (takes && begin > er.fixed) {
        int32_t mine = 0, same = 0;
        const int32_t to = min(begin, er.until);
#pragma unroll 4
        for (int32_t j = er.fixed + tid; j < to; j += kPlan) {
            const uint32_t y = weight_order(wr[j]);
            mine += y > er.bar, same += y == er.bar;
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) mine += __shfl_xor(mine, o, 64), same += __shfl_xor(same, o, 64);
        int32_t before, total;
        meet(mine, &before, &total);
        over += total;
        meet(same, &before, &total);
        equal += total;
    }
    const unsigned long long below = ((unsigned long long)1 << lane) - 1;
    for (int32_t j0 = begin; j0 < end; j0 += kPlan * 4) {
        float x[4];
        unsigned long long is[4], eq[4];
        int32_t packed = 0, before, total;
#pragma unroll
        for (int u = 0; u < 4; u++) x[u] = wr[min(j0 + wave * 256 + u * 64 + lane, er.held - 1)];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int32_t j = j0 + wave * 256 + u * 64 + lane;
            const uint32_t y = weight_order(x[u]);
            const bool may = j >= er.fixed && j < er.until;
            is[u] = __ballot(may ? takes && y > er.bar : j < er.held);
            eq[u] = __ballot(may && takes && y == er.bar);
            packed += __popcll(is[u]) | __popcll(eq[u]) << 16;
        }
        meet(packed, &before, &total);
        int32_t o = over + (before & 0xffff), e = equal + (before >> 16);
        over += total & 0xffff, equal += total >> 16;
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int32_t j = j0 + wave * 256 + u * 64 + lane;
            const int32_t mine = e + __popcll(eq[u] & below), to = o + __popcll(is[u] & below) + min(mine, er.ties);
            if ((is[u] >> lane & 1) || ((eq[u] >> lane & 1) && mine < er.ties)) {
                out[to] = j;
                w.weight[r * cap + to] = x[u];
                const int32_t jc = j / size, tc = to / size, pf = row[jc], pt = row[tc];
                const bool ok = pf >= 0 && pf < a.num_pages && pt >= 0 && pt < a.num_pages;
                w.from[r * cap + to] = make_uint2(ok ? (uint32_t)pf : kNoPage, (uint32_t)(j - jc * size));
                w.to[r * cap + to] = make_uint2((uint32_t)pt, (uint32_t)(to - tc * size));
            } else if (j < er.held && j == to) {
                w.rows[r].first = j;  // (the first key that goes: no other has its own index for a place)
            }
            o += __popcll(is[u]), e += __popcll(eq[u]);
        }
    }
}

// What else changes of a row that gives up keys, a workgroup's: its weights, its length, its entries and the counts of the
// pages behind.
__device__ __forceinline__ void evict_finish(const CacheArgs &a, const EvictWork &w, float *weights, int64_t stride, int64_t r) {
    const EvictRow er = w.rows[r];
    if (er.n == er.held) return;
    float *wr = weights + r * stride;
    for (int32_t j = er.first + threadIdx.x; j < er.held; j += blockDim.x) wr[j] = j < er.n ? w.weight[r * w.cap + j] : 0.f;
    int32_t *row = a.table + r * a.max_pages;
    const int64_t np = pages_of(a, er.held);
    for (int64_t c = pages_of(a, er.n) + threadIdx.x; c < np; c += blockDim.x) {
        const int32_t page = row[c];
        row[c] = -1;
        if (page >= 0 && page < a.num_pages) atomicSub(a.counts + page, 1);
    }
    if (threadIdx.x == 0) a.lengths[r] = er.n;
}

// The first workgroups finish a row each (in the first launch of a call). Workgroup (row, pool, column): 2^shift threads
// a key, a T each. Two steps of kEvictLoads loads are in flight: a step's keys are stored while the next one's arrive.
constexpr int kEvictLoads = 8, kEvictThreads = 512;
template <class T>
__global__ __launch_bounds__(kEvictThreads) void cache_evict_move(CacheArgs a, EvictWork w, float *weights, int64_t weights_stride,
                                                                  int32_t finish, PoolArgs pools, int32_t columns,
                                                                  int32_t shift) {
    int64_t i = blockIdx.x;
    if (i < finish) {
        evict_finish(a, w, weights, weights_stride, i);
        return;
    }
    i -= finish;
    const int64_t page_size = a.page_size;
    const int32_t keys = kEvictThreads >> shift, step = keys * kEvictLoads, mine = threadIdx.x >> shift;
    const int32_t column = (int32_t)(i % columns);
    i /= columns;
    const int x = (int)(i % pools.n);
    const int64_t r = i / pools.n, bytes = pools.at[x].bytes / page_size, stride = pools.at[x].stride;
    const int64_t at = (((int64_t)column << shift) + (threadIdx.x & ((1 << shift) - 1))) * (int64_t)sizeof(T);
    const int32_t first = w.rows[r].first, count = w.rows[r].n;
    const uint2 *from = w.from + r * w.cap, *to = w.to + r * w.cap;
    if (first >= count || ((int64_t)column << shift) * (int64_t)sizeof(T) >= bytes) return;
    // (a thread past the row's end reads the row's first bytes, one without a key the pool's, and stores nothing)
    char *base = pools.at[x].pages + (at < bytes ? at : 0);
    auto place = [&](uint32_t page, uint32_t row) { return base + (int64_t)page * stride + (int64_t)row * bytes; };
    T even[kEvictLoads], odd[kEvictLoads];
    uint32_t page0[kEvictLoads], row0[kEvictLoads], page1[kEvictLoads], row1[kEvictLoads];
    uint2 f[kEvictLoads], t[kEvictLoads];
    auto look = [&](int32_t j0) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < kEvictLoads; u++) {
            const int32_t j = min(j0 + u * keys + mine, count - 1);
            f[u] = from[j], t[u] = to[j];
        }
    };
    auto load = [&](int32_t j0, T(&x)[kEvictLoads], uint32_t(&page)[kEvictLoads], uint32_t(&row)[kEvictLoads])
                    __attribute__((always_inline)) {  // and the places of the step behind
#pragma unroll
        for (int u = 0; u < kEvictLoads; u++) {
            const bool ok = f[u].x != kNoPage;
            x[u] = *(const T *)place(ok ? f[u].x : 0u, ok ? f[u].y : 0u);
            page[u] = ok && at < bytes && j0 + u * keys + mine < count ? t[u].x : kNoPage;
            row[u] = t[u].y;
        }
        look(j0 + step);
    };
    auto store = [&](T(&x)[kEvictLoads], uint32_t(&page)[kEvictLoads], uint32_t(&row)[kEvictLoads])
                     __attribute__((always_inline)) {
        // every load of the step has arrived before its first store: a key may lie where another of these comes from
#pragma unroll
        for (int u = 0; u < kEvictLoads; u++) {
            if constexpr (sizeof(T) > 4)
                asm volatile("" ::"v"(x[u][0]) : "memory");
            else
                asm volatile("" ::"v"((uint32_t)x[u]) : "memory");
        }
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
#pragma unroll
        for (int u = 0; u < kEvictLoads; u++)
            if (page[u] != kNoPage) *(T *)place(page[u], row[u]) = x[u];
    };
    look(first);
    load(first, even, page0, row0);
    for (int32_t j0 = first; j0 < count; j0 += 2 * step) {
        load(j0 + step, odd, page1, row1);
        store(even, page0, row0);
        if (j0 + step >= count) break;
        load(j0 + 2 * step, even, page0, row0);
        store(odd, page1, row1);
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

// Whether some byte is two pools' (whose keys would move twice): slices of one wider pool, alike in their strides,
// are told apart by their places in it, others by their ends.
static bool pools_overlap(const dm_cache_table *t, const dm_cache_pool *pools, int64_t n) {
    std::vector<std::pair<uintptr_t, int64_t>> at;
    for (int64_t i = 0; i < n; i++)
        if (t->num_pages > 0 && pools[i].page_bytes > 0) at.emplace_back((uintptr_t)pools[i].pages, i);
    std::sort(at.begin(), at.end());
    for (size_t i = 0; i < at.size(); i++) {
        const dm_cache_pool &p = pools[at[i].second];
        const uintptr_t end = at[i].first + (t->num_pages - 1) * p.page_stride + p.page_bytes;
        for (size_t j = i + 1; j < at.size() && at[j].first < end; j++) {
            const dm_cache_pool &q = pools[at[j].second];
            const int64_t off = (int64_t)((at[j].first - at[i].first) % p.page_stride);
            if (p.page_stride != q.page_stride || off < p.page_bytes || off + q.page_bytes > p.page_stride) return true;
        }
    }
    return false;
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

static EvictWork evict_work(const dm_cache_table *t, char *at, size_t *bytes) {
    EvictWork w{};
    w.cap = t->max_pages * t->page_size;
    const size_t rows = align_up((size_t)t->rows * sizeof(EvictRow)), keys = (size_t)(t->rows * w.cap);
    w.rows = (EvictRow *)at;
    w.from = (uint2 *)(at + rows);
    w.to = (uint2 *)(at + rows + align_up(keys * sizeof(uint2)));
    w.weight = (float *)(at + rows + 2 * align_up(keys * sizeof(uint2)));
    *bytes = rows + 2 * align_up(keys * sizeof(uint2)) + align_up(keys * sizeof(float));
    return w;
}
// Workgroups that a launch of the moves has at least, where the rows are wide enough: 16 rows cut to half 174, 131 and 135 us
// with 128, 256 and 512, a document to an eighth 84, 93 and 116 (before its places were shared out).
constexpr int64_t kEvictGroups = 256;
// How the pools from `at` on that one launch takes are cut: into columns of grain << shift bytes of a key.
struct EvictColumns {
    int64_t n, most, grain;  // pools, bytes of their widest key, bytes that all of their keys are whole numbers of
    int64_t of(int shift) const { return (most + (grain << shift) - 1) / (grain << shift); }
};
static EvictColumns evict_columns(const dm_cache_table *t, const dm_cache_pool *pools, int64_t npools, int64_t at) {
    EvictColumns c{std::min<int64_t>(kPoolsPerLaunch, npools - at), 0, 16};
    for (int64_t i = at; i < at + c.n; i++) {
        const int64_t row = pools[i].page_bytes / t->page_size;
        const uint64_t bits = (uint64_t)pools[i].pages | (uint64_t)pools[i].page_stride | (uint64_t)row;
        while (bits % c.grain) c.grain /= 2;
        c.most = std::max(c.most, row);
    }
    return c;
}
static bool evict_sizes(const dm_cache_table *t) {
    return table_sizes(t) && t->rows <= kMostRows && t->max_pages <= ((int64_t)1 << 30) / t->page_size &&
           t->rows * t->max_pages * t->page_size < kI31 * 16;
}

size_t dm_cache_evict_workspace(const dm_cache_table *t) {
    size_t bytes = 0;
    if (evict_sizes(t)) evict_work(t, nullptr, &bytes);
    return bytes;
}

int dm_cache_evict(const dm_cache_table *t, const dm_cache_pool *pools, int64_t npools, float *weights,
                   int64_t weights_stride, const int32_t *budgets, int64_t recent, int32_t *kept, void *workspace,
                   size_t workspace_bytes, void *stream) {
    const std::string op("cache_evict");
    if (int rc = check_table(op, t)) return rc;
    if (int rc = check_pools(op, t, pools, npools)) return rc;
    try {
        if (pools_overlap(t, pools, npools)) return refuse(op + ": a byte of the pools belongs to two of them");
    } catch (const std::bad_alloc &) {
        return refuse(op + ": out of host memory");
    }
    if (!evict_sizes(t))
        return refuse(op + ": a row holds at most 2^30 keys, the rows less than 2^35, rows are at most 2^22");
    if (recent < 0) return refuse(op + ": recent must not be negative");
    const int64_t cap = t->max_pages * t->page_size;
    if (t->rows > 1 && weights_stride < cap)
        return refuse(op + ": the weights are [R, max_pages * page_size], their rows apart");
    if (workspace_bytes < dm_cache_evict_workspace(t))
        return refuse(op + ": the workspace is smaller than dm_cache_evict_workspace");
    if (t->rows == 0 || cap == 0) return DM_OK;
    if (!weights || !budgets || !kept) return refuse(op + ": the weights, the budgets or the results' place are missing");
    for (int64_t i = 0; i < npools; i += kPoolsPerLaunch) {  // (workgroups of a launch: a row each, and columns of 512 bytes or more)
        const EvictColumns c = evict_columns(t, pools, npools, i);
        int64_t groups = t->rows;
        for (int64_t x = i; x < i + c.n; x++) groups += t->rows * (pools[x].page_bytes / t->page_size / 512 + 1);
        // (each pool has as many columns as the launch's widest one)
        if (std::max(groups, t->rows + t->rows * c.n * c.of(9)) >= ((int64_t)1 << 23))
            return refuse(op + ": more rows and bytes than one launch takes");
    }
    hipStream_t st = (hipStream_t)stream;
    size_t bytes;
    const EvictWork w = evict_work(t, (char *)workspace, &bytes);
    const CacheArgs ca = cache_args(t);
    const unsigned shares = (unsigned)std::min<int64_t>(kEvictShares, (cap + 4 * kPlan - 1) / (4 * kPlan));
    for (int64_t r = 0; r < t->rows; r += 65535) {  // (rows of a launch: 2^22 of them together would be 2^32 threads)
        const unsigned n = (unsigned)std::min<int64_t>(65535, t->rows - r);
        EvictWork part = w;
        part.rows += r, part.from += r * cap, part.to += r * cap, part.weight += r * cap;
        CacheArgs pa = ca;
        pa.table += r * t->max_pages, pa.lengths += r;
        float *at = weights + r * weights_stride;
        cache_evict_select<<<n, kPlan, 0, st>>>(pa, at, weights_stride, budgets + r, recent, part);
        cache_evict_place<<<dim3(shares, n), kPlan, 0, st>>>(pa, at, weights_stride, kept + r * cap, part);
    }
    for (int64_t i = 0; i == 0 || i < npools; i += kPoolsPerLaunch) {
        bool wide;
        int64_t pieces;
        const PoolArgs pa = pools_of(pools, npools, i, &wide, &pieces);
        const EvictColumns c = evict_columns(t, pools, npools, i);
        const int64_t grain = c.grain;
        // the widest columns that make kEvictGroups workgroups
        int shift = 9;
        while (shift > 0 && (t->rows * pa.n * c.of(shift) < kEvictGroups || (c.most <= grain << (shift - 1)))) shift--;
        const int64_t items = t->num_pages > 0 ? t->rows * pa.n * c.of(shift) : 0;  // (no page: nothing to load from)
        const int64_t finish = i == 0 ? t->rows : 0;
        if (finish + items == 0) continue;
#define EVICT_MOVE(T)                                                                                             \
    cache_evict_move<T><<<(unsigned)(finish + items), kEvictThreads, 0, st>>>(ca, w, weights, weights_stride,     \
                                                                              (int32_t)finish, pa, (int32_t)c.of(shift), shift)
        if (grain == 16)
            EVICT_MOVE(u32x4_vec);
        else if (grain == 8)
            EVICT_MOVE(u32x2_vec);
        else if (grain == 4)
            EVICT_MOVE(uint32_t);
        else if (grain == 2)
            EVICT_MOVE(uint16_t);
        else
            EVICT_MOVE(uint8_t);
#undef EVICT_MOVE
    }
    probe_add(DM_PROBE_CACHE_EVICT);
    DM_LAUNCH_CHECK("cache_evict: launch");
    return DM_OK;
}

}  // extern "C"
