// How a ragged batch of new tokens over a paged cache is shared out, worked out on the device.
//
// The query rows of a sequence (its new tokens x the query heads of one key-value head) lie in tiles, and a
// tile sweeps the keys that its rows see. All tiles laid one after another, each as long as its keys and a
// constant for its start, are a line; each of a fixed number of workers (workgroups or wavefronts) takes an
// equal part of it, wherever that begins and ends. So every worker has the same work whatever the lengths are, no
// length is needed on the host, and at most two of a worker's tiles are shared with others: a tile that a worker
// has whole is written at once, the pieces of a shared one go to the worker's two places in the workspace and are
// joined by a second launch. What a tile costs is linear in its number within the sequence, so a sequence's tiles are
// summed in closed form and a worker finds its part by a scan over the sequences and a search within one.
#pragma once

#include "dm_common.h"

namespace dm {

struct PagedArgs {
    int32_t S, N, cap, left;  // sequences, new tokens, keys that a table row holds, the window's left (-1: none)
    int32_t hq, hkv, d, rep;  // rep: query heads of a key-value head
    float scale;
    const int32_t *lengths, *cu, *table;  // cu: NULL for one token a sequence
    int64_t page_size, max_pages, num_pages;
    int64_t qt, qh, kb, kt, kh, vb, vt, vh;  // strides in elements
    void *o;
    float *lse;     // [N, Hq] or NULL
    float *scores;  // [S, Hkv, score_rows, cap]: the narrow tiles' scores (log2 units), or NULL
    int32_t score_rows;
};

// A shared tile's join: its rows, and the workers that have pieces of it. Of more than kJoinMany pieces each worker
// behind the first has some rows joined (one pass over a row's pieces a workgroup), of fewer the second one has all. (8 tokens
// of 2 heads of 128 against 60000 keys 182 us by one and 54 by all; a token of 8 heads against 100000 156 and 108.)
constexpr int kJoinMany = 48;
struct PagedJob {
    int32_t tok, head, per, rows, first, last;
};

// One line: which sequences' tiles lie on it, and its workers.
struct PagedLine {
    int32_t rt, pitch;  // most rows of a tile, and of this call's tiles
    int32_t m, hc, per; // tokens of a tile; tiles of a token (above rt heads); row r: token r / per, head r % per
    int32_t over, upto; // the sequences of over < n rep <= upto rows
    int32_t workers, unit;   // most workers; a piece's keys begin at multiples of unit (a power of 2) from the tile's first
    int32_t start, least;    // a tile's start in keys, and what a worker has at least
    float *o;           // [2 workers, pitch, D]: unnormalised outputs
    float2 *ml;         // [2 workers, pitch]: reference (log2 units) and sum
    PagedJob *jobs;     // [workers]
};

struct PagedSeq {
    int32_t first, n, len;  // first token, new tokens, keys with them
    bool ok;                // its offsets go up within the tokens
};

__device__ __forceinline__ PagedSeq paged_seq(const PagedArgs &a, int32_t s) {
    PagedSeq q;
    int32_t end = s + 1;
    q.first = s;
    if (a.cu) q.first = a.cu[s], end = a.cu[s + 1];
    q.len = min(max(a.lengths[s], 0), a.cap);
    q.ok = q.first >= 0 && q.first <= end && end <= a.N;
    q.n = q.ok ? end - q.first : 0;
    return q;
}

// sum over u < t of max(0, a + m u)
__device__ __forceinline__ int64_t ramp(int64_t a, int64_t m, int64_t t) {
    const int64_t u0 = a >= 0 ? 0 : min(t, (-a + m - 1) / m), c = t - u0;
    return c * (a + m * u0) + m * (c * (c - 1) / 2);
}

// sum over u < t of max(0, b - m u)
__device__ __forceinline__ int64_t slope(int64_t b, int64_t m, int64_t t) {
    const int64_t c = b <= 0 ? 0 : min(t, (b + m - 1) / m);
    return c * b - m * (c * (c - 1) / 2);
}

// What the first t token tiles of a sequence cost: of each its start, and the keys between the first that its
// first token sees and the last that its last one would see if the tile were full.
__device__ __forceinline__ int64_t tiles_cost(const PagedArgs &a, const PagedLine &l, const PagedSeq &q, int32_t t) {
    const int64_t p0 = (int64_t)q.len - q.n;
    int64_t x = (int64_t)t * l.start + ramp(p0 + l.m, l.m, t);
    if (a.left >= 0) x -= ramp(p0 - a.left, l.m, t);
    return x;
}
__device__ __forceinline__ int32_t tiles_of(const PagedArgs &a, const PagedLine &l, const PagedSeq &q) {
    return (q.n + l.m - 1) / l.m;
}
// how often the tiles of a sequence stand on the line
__device__ __forceinline__ int32_t turns_of(const PagedArgs &a, const PagedLine &l) { return a.hkv * l.hc; }
__device__ __forceinline__ bool on_line(const PagedArgs &a, const PagedLine &l, const PagedSeq &q) {
    const int64_t rows = (int64_t)q.n * a.rep;
    return q.n > 0 && rows > l.over && rows <= l.upto;
}

// The line of the weights that keys get: a tile is `keys` keys of a sequence, and costs, for each key-value head,
// its start and the rows that see any of them.
struct KeyLine {
    int32_t keys, workers, start, least, unit;
    int32_t over;     // the sequences of more than `over` rows
    float *sums;      // [2 workers, keys]
    PagedJob *jobs;   // [workers]: tok = sequence, head = tile
};
__device__ __forceinline__ int64_t tiles_cost(const PagedArgs &a, const KeyLine &l, const PagedSeq &q, int32_t t) {
    // tokens of tile u: those from max(0, keys u - p0) on and, with a window, in front of keys (u + 1) + left - p0
    const int64_t p0 = (int64_t)q.len - q.n;
    int64_t x = (int64_t)t * q.n - ramp(-p0, l.keys, t);
    if (a.left >= 0) {
        const int64_t y = p0 - l.keys - a.left;
        x -= slope(q.n + y, l.keys, t) - slope(y, l.keys, t);
    }
    return ((int64_t)t * l.start + x * a.rep) * a.hkv;
}
__device__ __forceinline__ int32_t tiles_of(const PagedArgs &a, const KeyLine &l, const PagedSeq &q) {
    return (q.len + l.keys - 1) / l.keys;
}
__device__ __forceinline__ int32_t turns_of(const PagedArgs &a, const KeyLine &l) { return 1; }
__device__ __forceinline__ bool on_line(const PagedArgs &a, const KeyLine &l, const PagedSeq &q) {
    return q.n > 0 && q.len > 0 && (int64_t)q.n * a.rep > l.over;
}

// The exclusive prefix sums of the workgroup's x on each of L lines, and their totals.
template <int NT, int L>
struct PlanSmem {
    int64_t pre[L][NT], waves[L][NT / 64];
};
template <int NT, int L, class Line>
__device__ __forceinline__ void plan_chunk(const PagedArgs &a, const Line (&l)[L], int32_t s0, PlanSmem<NT, L> &sm, bool *ok,
                                           int64_t (&all)[L]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int32_t s = s0 + (int32_t)threadIdx.x;
    int64_t x[L], in[L];
#pragma unroll
    for (int i = 0; i < L; i++) x[i] = 0;
    if (s < a.S) {
        const PagedSeq q = paged_seq(a, s);
        *ok = *ok && q.ok;
#pragma unroll
        for (int i = 0; i < L; i++)
            if (on_line(a, l[i], q)) x[i] = turns_of(a, l[i]) * tiles_cost(a, l[i], q, tiles_of(a, l[i], q));
    }
#pragma unroll
    for (int i = 0; i < L; i++) {
        in[i] = x[i];
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int64_t y = __shfl_up((long long)in[i], o, 64);
            if (lane >= o) in[i] += y;
        }
    }
    __syncthreads();  // (the last chunk's sums have been read)
#pragma unroll
    for (int i = 0; i < L; i++)
        if (lane == 63) sm.waves[i][wave] = in[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < L; i++) {
        int64_t before = 0;
        all[i] = 0;
#pragma unroll
        for (int w = 0; w < NT / 64; w++) {
            before += w < wave ? sm.waves[i][w] : 0;
            all[i] += sm.waves[i][w];
        }
        sm.pre[i][threadIdx.x] = before + in[i] - x[i];
    }
    __syncthreads();
}

// A worker's place on a line of length `total` with `workers` workers: worker w has [at(w), at(w + 1)).
struct PagedShare {
    int64_t total, each;
    int32_t workers, rest;  // total = each x workers + rest
    __device__ __forceinline__ int64_t at(int32_t w) const {
        return each * w + (int32_t)((uint32_t)(rest * w) / (uint32_t)workers);
    }
    // the last worker that begins in front of x > 0
    __device__ __forceinline__ int32_t last_before(int64_t x) const {
        int32_t w = (int32_t)min((int64_t)workers - 1, (x - 1) / each);
        while (w > 0 && at(w) >= x) w--;
        return w;
    }
};

// Where a worker stands: tile t of sequence s, in its u-th turn, which begins at `base` of the line.
struct PagedWalk {
    int32_t s, u, t;
    int32_t nt;  // tiles of the sequence
    PagedSeq q;
    int64_t base;
};

// The whole workgroup: the lines' lengths and shares; every line is of length 0 where the offsets do not go up (false).
template <int NT, int L, class Line>
__device__ __forceinline__ bool plan_lines(const PagedArgs &a, const Line (&l)[L], PlanSmem<NT, L> &sm, PagedShare (&sh)[L]) {
    bool ok = true;
#pragma unroll
    for (int i = 0; i < L; i++) sh[i].total = 0;
    for (int32_t s0 = 0; s0 < a.S; s0 += NT) {
        int64_t all[L];
        plan_chunk<NT, L>(a, l, s0, sm, &ok, all);
#pragma unroll
        for (int i = 0; i < L; i++) sh[i].total += all[i];
    }
    ok = __syncthreads_and(ok);
#pragma unroll
    for (int i = 0; i < L; i++) {
        if (!ok) sh[i].total = 0;
        sh[i].workers = (int32_t)max((int64_t)1, min((int64_t)l[i].workers, sh[i].total / l[i].least));
        sh[i].each = sh[i].total / sh[i].workers;
        sh[i].rest = (int32_t)(sh[i].total - sh[i].each * sh[i].workers);
    }
    return ok;
}

// The whole workgroup: the walk of the worker that begins at p of line I (wavefront-uniform, each wavefront its own; none:
// a p below zero).
template <int I, int NT, int L, class Line>
__device__ __forceinline__ void plan_find(const PagedArgs &a, const Line (&l)[L], PlanSmem<NT, L> &sm, const PagedShare &sh,
                                          int64_t p, PagedWalk *walk) {
    const int lane = threadIdx.x & 63;
    int64_t base = 0;
    for (int32_t s0 = 0; s0 < a.S && sh.total > 0; s0 += NT) {
        int64_t all[L];
        all[I] = sh.total;
        bool ok = true;
        if (a.S > NT) plan_chunk<NT, L>(a, l, s0, sm, &ok, all);
        if (p >= base && p < base + all[I]) {
            int n = 0;
#pragma unroll 1
            for (int i = 0; i < min(NT, a.S - s0); i += 64)
                n += __popcll(__ballot(i + lane < a.S - s0 && sm.pre[I][i + lane] <= p - base));
            walk->s = __builtin_amdgcn_readfirstlane(s0 + n - 1);
            walk->base = base + sm.pre[I][n - 1];
        }
        base += all[I];
    }
    __syncthreads();  // (the sums have been read)
    if (p < 0) return;
    walk->q = paged_seq(a, walk->s);
    walk->nt = tiles_of(a, l[I], walk->q);
    int64_t rem = p - walk->base;
    const int64_t turn = tiles_cost(a, l[I], walk->q, walk->nt), u = rem / turn;
    rem -= u * turn;
    // the last tile that begins at rem or in front of it: 64 probes at a time
    int32_t lo = 0, hi = walk->nt;  // it lies in [lo, hi)
    while (hi - lo > 1) {
        const int32_t step = (hi - lo + 63) / 64, t = lo + lane * step;
        const int n = __popcll(__ballot(t < hi && tiles_cost(a, l[I], walk->q, t) <= rem));
        lo += (n - 1) * step;
        hi = min(hi, lo + step);
    }
    walk->u = (int32_t)u, walk->t = lo;
    walk->base = p - rem + tiles_cost(a, l[I], walk->q, lo);
}

// A worker's next piece: rows of one tile, the keys [s0, s1) of those [lo, hi) that the tile sees.
struct PagedPiece {
    int32_t tok, head, per, rows;  // first token and query head; row r: token tok + r / per, head head + r % per
    int32_t pos, kh, s;            // the position of tok; key-value head, sequence
    int32_t row0;                  // the sequence's row of this head that r = 0 is
    int32_t s0, s1;
    bool whole;
    int32_t slot;                  // not whole: its place
    int32_t first;                 // the worker that the tile begins with, where another did
};

__device__ __forceinline__ PagedPiece piece_of(const PagedArgs &a, const PagedLine &l, const PagedWalk &w, const PagedShare &sh,
                                               int32_t worker, int64_t p, int64_t end, int64_t *next, int32_t *last) {
    PagedPiece x;
    const int32_t i0 = w.t * l.m, i1 = min(i0 + l.m, w.q.n);
    const int64_t cost = tiles_cost(a, l, w.q, w.t + 1) - tiles_cost(a, l, w.q, w.t);
    x.kh = w.u / l.hc;
    const int32_t c = w.u - x.kh * l.hc;  // which heads of a token
    x.tok = w.q.first + i0;
    x.head = x.kh * a.rep + c * l.rt;
    x.per = l.per;
    x.rows = l.hc > 1 ? min(l.rt, a.rep - c * l.rt) : (i1 - i0) * a.rep;
    x.pos = w.q.len - w.q.n + i0;
    x.s = w.s;
    x.row0 = i0 * a.rep + c * l.rt;
    const int32_t hi = max(0, w.q.len - w.q.n + i1);
    const int32_t lo = a.left >= 0 ? min(hi, max(0, x.pos - a.left)) : 0;
    auto key = [&](int64_t off) -> int32_t {  // the key at `off` of the tile's part of the line
        const int64_t k = (off - l.start) & -(int64_t)l.unit;
        return off >= cost ? hi : (k <= 0 ? lo : (int32_t)min((int64_t)hi, lo + k));
    };
    const int64_t o0 = p - w.base, o1 = min(end - w.base, cost);
    x.s0 = key(o0), x.s1 = key(o1);
    x.whole = o0 == 0 && o1 == cost;
    x.slot = 2 * worker + (o0 == 0 ? 1 : 0);
    *next = w.base + cost;
    // the worker that the tile's first border belongs to has it joined; where there are many pieces, all behind the first do
    *last = -1;
    x.first = worker - 1;
    if (o0 > 0) {
        const bool near = sh.at(worker - 1) <= w.base;
        if (!near) x.first = sh.last_before(w.base + 1);
        const int32_t end = sh.last_before(w.base + cost);
        if (near || end - x.first >= kJoinMany) *last = end;
    }
    return x;
}

// On to the next tile of the line (false: there is none).
template <class Line>
__device__ __forceinline__ bool walk_on(const PagedArgs &a, const Line &l, PagedWalk &w, int64_t base) {
    w.base = base;
    if (++w.t < w.nt) return true;
    w.t = 0;
    if (++w.u < turns_of(a, l)) return true;
    w.u = 0;
    // (64 sequences at a time: between two prompts may stand hundreds of single tokens. A prompt at each end of 1000 of
    // them 453 us one at a time and 149 so, of 62 107 and 89)
    const int lane = threadIdx.x & 63;
    for (int32_t s0 = w.s + 1; s0 < a.S; s0 += 64) {
        const int32_t s = s0 + lane;
        PagedSeq q{};
        if (s < a.S) q = paged_seq(a, s);
        const unsigned long long on = __ballot(s < a.S && on_line(a, l, q));
        if (!on) continue;
        const int n = __builtin_ctzll(on);
        w.s = s0 + n;
        w.q.first = __builtin_amdgcn_readlane(q.first, n), w.q.n = __builtin_amdgcn_readlane(q.n, n);
        w.q.len = __builtin_amdgcn_readlane(q.len, n), w.q.ok = true;
        w.nt = tiles_of(a, l, w.q);
        return true;
    }
    return false;
}

// A worker's next part of a tile of keys: its steps [r0, r1) of `unit` rows, counted through the key-value heads
// (each of them `steps`), rows from row `from` of a head on to `to`.
struct KeyPiece {
    int32_t s, k0;          // sequence, first key
    int32_t from, to, steps;
    int32_t r0, r1;
    bool whole;
    int32_t slot;
};
__device__ __forceinline__ KeyPiece key_piece(const PagedArgs &a, const KeyLine &l, const PagedWalk &w, const PagedShare &sh,
                                              int32_t worker, int64_t p, int64_t end, int64_t *next, int32_t *last) {
    KeyPiece x;
    const int64_t cost = tiles_cost(a, l, w.q, w.t + 1) - tiles_cost(a, l, w.q, w.t);
    const int32_t p0 = w.q.len - w.q.n;
    x.s = w.s, x.k0 = w.t * l.keys;
    const int32_t t0 = max(0, x.k0 - p0);
    const int32_t t1 = a.left >= 0 ? (int32_t)max((int64_t)t0, min((int64_t)w.q.n, (int64_t)x.k0 + l.keys + a.left - p0)) : w.q.n;
    x.from = t0 * a.rep, x.to = t1 * a.rep;
    x.steps = (x.to - x.from + l.unit - 1) / l.unit;
    const int64_t o0 = p - w.base, o1 = min(end - w.base, cost), all = (int64_t)x.steps * a.hkv;
    auto step = [&](int64_t off) { return off >= cost ? (int32_t)all : (int32_t)(off * all / cost); };
    x.r0 = step(o0), x.r1 = step(o1);
    x.whole = o0 == 0 && o1 == cost;
    x.slot = 2 * worker + (o0 == 0 ? 1 : 0);
    *next = w.base + cost;
    *last = -1;
    if (o0 > 0 && sh.at(worker - 1) <= w.base) *last = sh.last_before(w.base + cost);
    return x;
}

}  // namespace dm
