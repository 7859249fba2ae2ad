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
// Bandwidth-bound: every head is read once and written once. Measured in bf16 (a large copy on this card
// runs at 5.0 TB/s): 16384 tokens of 40 heads of 128 forward 63 us, 5.3 TB/s, backward 101 us, 5.0 TB/s, and
// 5 us for the weights' sums; 6144 tokens of 18 heads of 256 backward 36 us, 4.7 TB/s; 8192 tokens of 48
// heads of 128 into pages 42 us, 4.8 TB/s. A token for each of 64 sequences is a launch and a chain of
// loads (the length, its page, the heads): 7.7 us.
#include <algorithm>
#include <string>
#include <type_traits>

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

// place_paged, with the call's own positions where it has some.
__device__ __forceinline__ bool place_turned(const RopeArgs &a, const RopePages &pg, int64_t token, int64_t *p,
                                             int64_t *krow, int64_t *vrow) {
    const bool is = place_paged(pg, token, p, krow, vrow);
    if (a.positions && is) *p = place_plain(a, 0, token);
    return is;
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

// The simple forms, for any width, alignment and number of pairs: a workgroup takes a token, whose angles go
// to LDS, and a wavefront a head of it at a time (block (x, y): every gridDim.y-th four), four elements 64
// apart in a lane, a pair's other element found in the wavefront's row of LDS. Bound by the chain of a
// head (single elements loaded, their sum, the row, the result) that a wavefront goes through one at a time:
// 8192 tokens of 40 heads of 112 in bf16 take 125 us forward and 270 backward (with angles for every head 183
// and 377), where the kernels below take 27 and 41 for a width of 96.
template <int DT, int MODE>
__global__ __launch_bounds__(256) void rope_generic(RopeArgs a, RopePages pg, const void *__restrict__ q,
                                                    const void *__restrict__ k, const void *__restrict__ v,
                                                    void *__restrict__ qo, void *__restrict__ ko,
                                                    void *__restrict__ vo) {
    __shared__ float rows[4][256];
    __shared__ float2 angles[128];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float *row = rows[wave];
    const int heads = a.hq + a.hkv * (MODE == kRopePaged ? 2 : 1);
    for (int64_t token = blockIdx.x; token < a.tokens; token += gridDim.x) {
        const int64_t b = token / a.T, t = token - b * a.T;
        int64_t p, krow = -1, vrow = -1;
        bool is = true;
        if (MODE == kRopePaged)
            is = place_turned(a, pg, token, &p, &krow, &vrow);
        else
            p = place_plain(a, b, t);
        __syncthreads();  // (the last token's angles have been read)
        for (int j = threadIdx.x; j < a.n; j += 256) angles[j] = turn_of(p, a.inv_freq[j]);
        __syncthreads();
        for (int h = blockIdx.y * 4 + wave; h < heads; h += 4 * gridDim.y) {
            if (MODE == kRopePaged && h >= a.hq + a.hkv) {  // a value head: as it is
                const int hv = h - a.hq - a.hkv;
                if (is && vrow >= 0)
                    for (int e = lane; e < a.d; e += 64)
                        st<DT>(vo, vrow + hv * pg.v.h + e, ld<DT>(v, b * a.v.b + t * a.v.t + hv * a.v.h + e));
                continue;
            }
            const bool isq = h < a.hq;
            if (MODE == kRopePaged && !isq && krow < 0) continue;
            const int hh = isq ? h : h - a.hq;
            const void *src = isq ? q : k;
            const Strd sd = isq ? a.q : a.k;
            const void *wt = isq ? a.wq : a.wk;
            const int64_t from = b * sd.b + t * sd.t + hh * sd.h;
            float x[4], ss = 0.f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int e = lane + 64 * i;
                x[i] = e < a.d ? ld<DT>(src, from + e) : 0.f;
                ss += x[i] * x[i];
            }
            const float r = rsqrtf(wave_sum(ss) / a.d + a.eps);
            __builtin_amdgcn_wave_barrier();  // (a wavefront's LDS accesses complete in order)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int e = lane + 64 * i;
                const float wv = wt && e < a.d ? ld_any(a.weight_dtype, wt, e) + a.unit : 1.f;
                x[i] *= r * wv;
                row[e] = x[i];
            }
            __builtin_amdgcn_wave_barrier();
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
                    const float2 cs = angles[j];
                    y = first ? y * cs.x - row[other] * cs.y : row[other] * cs.y + y * cs.x;
                }
                st<DT>(dst, to + e, MODE == kRopePaged && !is ? 0.f : y);
            }
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
    __shared__ float2 angles[128];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float *row = rows[wave];
    const int heads = a.hq + a.hkv;
    float dw[2][4] = {};
    for (int64_t token = blockIdx.x; token < a.tokens; token += gridDim.x) {
        const int64_t b = token / a.T, t = token - b * a.T, p = place_plain(a, b, t);
        __syncthreads();  // (the last token's angles have been read)
        for (int j = threadIdx.x; j < a.n; j += 256) angles[j] = turn_of(p, a.inv_freq[j]);
        __syncthreads();
        for (int h = blockIdx.y * 4 + wave; h < heads; h += 4 * gridDim.y) {
            const bool isq = h < a.hq;
            const int hh = isq ? h : h - a.hq;
            const void *src = isq ? q : k, *grad = isq ? gq : gk, *wt = isq ? a.wq : a.wk;
            const Strd sd = isq ? a.q : a.k, sg = isq ? a.gq : a.gk;
            const int64_t from = b * sd.b + t * sd.t + hh * sd.h, gfrom = b * sg.b + t * sg.t + hh * sg.h;
            float x[4], z[4], ss = 0.f;
            __builtin_amdgcn_wave_barrier();  // (a wavefront's LDS accesses complete in order)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int e = lane + 64 * i;
                x[i] = e < a.d ? ld<DT>(src, from + e) : 0.f;
                z[i] = e < a.d ? ld<DT>(grad, gfrom + e) : 0.f;
                ss += x[i] * x[i];
                row[e] = z[i];
            }
            const float r = rsqrtf(wave_sum(ss) / a.d + a.eps);
            __builtin_amdgcn_wave_barrier();
            float gx = 0.f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int e = lane + 64 * i;
                if (e < 2 * a.n) {
                    int j, other;
                    bool first;
                    pair_of(e, a.n, a.interleaved, &j, &other, &first);
                    const float2 cs = angles[j];
                    z[i] = first ? z[i] * cs.x + row[other] * cs.y : z[i] * cs.x - row[other] * cs.y;
                }
                const float add = z[i] * (x[i] * r);
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
                if (e < a.d) st<DT>(dst, to + e, r * (z[i] - x[i] * r * mean));
            }
        }
    }
#pragma unroll
    for (int x = 0; x < 2; x++)
#pragma unroll
        for (int i = 0; i < 4; i++) sums[wave][x][lane + 64 * i] = dw[x][i];
    __syncthreads();
    const int64_t part = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    for (int e = threadIdx.x; e < 2 * a.d; e += 256) {
        const int x = e / a.d, c = e - x * a.d;
        parts[part * 2 * a.d + e] = (sums[0][x][c] + sums[1][x][c]) + (sums[2][x][c] + sums[3][x][c]);
    }
}

// The kernels for heads of 64, 80, 96, 128, 192 and 256 in 16-byte pieces of V values: D / (2 V) lanes take a
// head, each the pieces at V li and n + V li, the first and the second elements of its pairs (half style),
// or of adjacent ones (interleaved); past the rotated 2 n the rest of the head in the same manner. So a
// pair never leaves its lane, and a head's sums are moves within 16 lanes (32 in f32). Lanes come in powers
// of two: of a head of 96 two of eight are idle, with values of 0. (8192 tokens of 40 heads in bf16,
// replayed, forward and backward: 80 wide 27 and 39 us, 96 27 and 41, 192 51 and 85.)
//
// A workgroup takes `tile` tokens: the angles of all of them go to LDS first, one a thread, since every
// head of a token turns by the same ones, then its lanes go through the tokens' heads.
template <int DT>
constexpr int rope_v() { return DT == DM_F32 ? 4 : 8; }

// Lanes with pieces of a head, and lanes of a head.
template <int DT, int D>
constexpr int rope_pieces() { return D / (2 * rope_v<DT>()); }
constexpr int rope_lanes(int pieces) { return pieces <= 1 ? 1 : 2 * rope_lanes((pieces + 1) / 2); }

template <int DT>
__device__ __forceinline__ uint4 raw_piece(const void *p, int64_t at) {
    return *(const uint4 *)((const char *)p + at * (DT == DM_F32 ? 4 : 2));
}
template <int DT, int V>
__device__ __forceinline__ void unpack_piece(const uint4 &a, float (&x)[V]) {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
    if constexpr (DT == DM_F32) {
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) x[2 * i] = unpack_lo<DT>(w[i]), x[2 * i + 1] = unpack_hi<DT>(w[i]);
    }
}
template <int V>
__device__ __forceinline__ void zero_pieces(float (&a)[V], float (&b)[V]) {
#pragma unroll
    for (int i = 0; i < V; i++) a[i] = b[i] = 0.f;
}
template <int DT, int V>
__device__ __forceinline__ void put_piece(void *p, int64_t at, const float (&x)[V]) {
    if constexpr (DT == DM_F32)
        *(float4 *)((float *)p + at) = make_float4(x[0], x[1], x[2], x[3]);
    else
        *(uint4 *)((uint16_t *)p + at) =
            make_uint4(pack2<DT>(x[0], x[1]), pack2<DT>(x[2], x[3]), pack2<DT>(x[4], x[5]), pack2<DT>(x[6], x[7]));
}

// Sum over aligned groups of N lanes (4, 8, 16 or 32).
template <int N>
__device__ __forceinline__ float head_sum(float t) {
    if constexpr (N == 4) {
        t += __shfl_xor(t, 1, 64);
        return t + __shfl_xor(t, 2, 64);
    } else {
        return group_sum<N>(t);
    }
}

// What a lane holds of a head of D: its two pieces' places, and where its angles begin.
template <int D, int V, bool INTER>
struct HeadLane {
    int a, b;      // the pieces' first elements
    bool turns;    // they rotate
    int ja, jb;    // the first angle of each (half style: of both)
    __device__ __forceinline__ HeadLane(int li, int n) {
        turns = li * V < n;
        a = turns ? li * V : 2 * n + (li * V - n);
        b = turns ? n + li * V : 2 * n + (D - 2 * n) / 2 + (li * V - n);
        ja = INTER ? a / 2 : a;
        jb = INTER ? b / 2 : a;
    }
};

// The pieces turned by the angles c, s [n] of their token; BACK: back.
template <int V, bool INTER, bool BACK>
__device__ __forceinline__ void turn_pieces(float (&a)[V], float (&b)[V], const float *c, const float *s, int ja, int jb) {
    if constexpr (INTER) {
#pragma unroll
        for (int i = 0; i < V / 2; i++) {
            const float ca = c[ja + i], sa = BACK ? -s[ja + i] : s[ja + i];
            const float cb = c[jb + i], sb = BACK ? -s[jb + i] : s[jb + i];
            const float a0 = a[2 * i], a1 = a[2 * i + 1], b0 = b[2 * i], b1 = b[2 * i + 1];
            a[2 * i] = a0 * ca - a1 * sa, a[2 * i + 1] = a0 * sa + a1 * ca;
            b[2 * i] = b0 * cb - b1 * sb, b[2 * i + 1] = b0 * sb + b1 * cb;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) {
            const float ci = c[ja + i], si = BACK ? -s[ja + i] : s[ja + i];
            const float x = a[i], y = b[i];
            a[i] = x * ci - y * si, b[i] = x * si + y * ci;
        }
    }
}

// Goes through rows = tile x heads, `by` at a time, as (token of the tile, head).
struct RowWalk {
    int t, h, dt, dh, heads;
    __device__ __forceinline__ RowWalk(int from, int by, int heads_)
        : t(from / heads_), h(from % heads_), dt(by / heads_), dh(by % heads_), heads(heads_) {}
    __device__ __forceinline__ void next() {
        t += dt, h += dh;
        if (h >= heads) h -= heads, t++;
    }
};

constexpr int kRopeTile = 16;  // most tokens of a tile

// The weights, as they multiply, into LDS [2, D]: queries' and keys'.
template <int D>
__device__ __forceinline__ void fill_weights(const RopeArgs &a, float *w) {
    for (int e = threadIdx.x; e < 2 * D; e += 256) {
        const void *p = e < D ? a.wq : a.wk;
        w[e] = p ? ld_any(a.weight_dtype, p, e % D) + a.unit : 1.f;
    }
}
// The tile's positions in the pages (paged), and its angles: cos [tile, n] and sin [tile, n].
struct RopePlaces {
    int64_t at[kRopeTile], krow[kRopeTile], vrow[kRopeTile];
    int is[kRopeTile];
};
__device__ __forceinline__ void fill_places(const RopeArgs &a, const RopePages &pg, int64_t first, int tile, RopePlaces &o) {
    const int t = threadIdx.x;
    if (t < tile && first + t < a.tokens) {
        int64_t p, kr, vr;
        o.is[t] = place_turned(a, pg, first + t, &p, &kr, &vr);
        o.at[t] = p, o.krow[t] = kr, o.vrow[t] = vr;
    }
}
template <bool PAGED>
__device__ __forceinline__ void fill_angles(const RopeArgs &a, int64_t first, int tile, const RopePlaces *places,
                                            float *cs) {
    const int here = (int)max((int64_t)0, min((int64_t)tile, a.tokens - first));
    for (int i = threadIdx.x; i < here * a.n; i += 256) {
        const int t = i / a.n, j = i - t * a.n;
        int64_t p;
        if constexpr (PAGED) {
            p = places->at[t];
        } else {
            const int64_t b = (first + t) / a.T;
            p = place_plain(a, b, first + t - b * a.T);
        }
        const float2 x = turn_of(p, a.inv_freq[j]);
        cs[i] = x.x, cs[tile * a.n + i] = x.y;
    }
}

// A workgroup goes through tiles of tokens. Each round fills in the next tile's angles (paged: and the
// places of the one behind that) and begins the loads of its first heads, so that a tile costs one barrier and
// every part of the code stands once: the first rounds have a tile before the first token, which is empty.
// (With the angles first and all heads behind a barrier: 89 us, not 63, on 16384 tokens of 40 heads of 128, where
// a workgroup has an empty round and one tile: what it gains there is the loads begun in front of the barrier and
// the weights in LDS. Two heads a lane in flight, U: one and four measured the same or worse.)
template <int DT, int D, int MODE, bool INTER>
__global__ __launch_bounds__(256) void rope_fast(RopeArgs a, RopePages pg, int tile, const void *__restrict__ q,
                                                 const void *__restrict__ k, const void *__restrict__ v,
                                                 void *__restrict__ qo, void *__restrict__ ko, void *__restrict__ vo) {
    constexpr int V = rope_v<DT>(), PIECES = rope_pieces<DT, D>(), LPH = rope_lanes(PIECES), BY = 256 / LPH, U = 2;
    constexpr bool PAGED = MODE == kRopePaged;
    extern __shared__ __align__(16) float lds[];  // the weights [2, D], two tiles' angles
    __shared__ RopePlaces places[PAGED ? 3 : 1];
    const int tid = threadIdx.x, li = tid % LPH, r0 = tid / LPH, n = a.n;
    float *angles = lds + 2 * D;
    const int64_t step = (int64_t)gridDim.x * tile, start = (int64_t)blockIdx.x * tile;
    const bool part = PIECES == LPH || li < PIECES;  // (an idle lane reads the first pieces and holds zeros)
    const HeadLane<D, V, INTER> hl(part ? li : 0, n);
    uint4 ra[U], rb[U];
    auto load = [&](int64_t first, int r, RowWalk &w, int rows, const void *src, const Strd &sd) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (r + u * BY < rows) {
                const int64_t token = first + w.t, b = token / a.T;
                const int64_t from = b * sd.b + (token - b * a.T) * sd.t + w.h * sd.h;
                ra[u] = raw_piece<DT>(src, from + hl.a);
                rb[u] = raw_piece<DT>(src, from + hl.b);
            }
            w.next();
        }
    };
    // the heads whose first batch is loaded ahead: the queries', or the keys' where there are none
    const bool ahead_k = a.hq == 0;
    const int heads0 = max(ahead_k ? a.hkv : a.hq, 1);
    int buf = 0, pl = 0;
    for (int64_t first = start - (PAGED ? 2 : 1) * step; first < a.tokens; first += step) {
        const int64_t next = first + step;
        if constexpr (PAGED) {
            if (next + step >= start) fill_places(a, pg, next + step, tile, places[(pl + 2) % 3]);
        }
        if (next >= start)
            fill_angles<PAGED>(a, next, tile, &places[PAGED ? (pl + 1) % 3 : 0], angles + (buf ^ 1) * 2 * tile * n);
        if (first < start && next >= start) fill_weights<D>(a, lds);
        const int here = first < start ? 0 : (int)min((int64_t)tile, a.tokens - first);
        const float *cs = angles + buf * 2 * tile * n, *sn = cs + tile * n;
        const RopePlaces &place = places[PAGED ? pl : 0];
#pragma unroll 1
        for (int x = 0; x < 2; x++) {
            const int heads = x ? a.hkv : a.hq, rows = here * heads;
            if (rows == 0) continue;
            const void *src = x ? k : q;
            void *dst = x ? ko : qo;
            const Strd sd = x ? a.k : a.q;
            const float *wa = lds + x * D + hl.a, *wb = lds + x * D + hl.b;
            RowWalk w(r0, BY, heads), put(r0, BY, heads);
            for (int r = r0; r < rows; r += BY * U) {
                if (x == ahead_k && r == r0) {
#pragma unroll
                    for (int u = 0; u < U; u++) w.next();
                } else {
                    load(first, r, w, rows, src, sd);
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (r + u * BY < rows) {  // (a head's lanes agree)
                        float pa[V], pb[V], ss = 0.f;
                        unpack_piece<DT, V>(ra[u], pa);
                        unpack_piece<DT, V>(rb[u], pb);
                        if (!part) zero_pieces<V>(pa, pb);
#pragma unroll
                        for (int i = 0; i < V; i++) ss += pa[i] * pa[i] + pb[i] * pb[i];
                        const float rs = rsqrtf(head_sum<LPH>(ss) * (1.f / D) + a.eps);
#pragma unroll
                        for (int i = 0; i < V; i++) pa[i] *= rs * wa[i], pb[i] *= rs * wb[i];
                        if (hl.turns) turn_pieces<V, INTER, false>(pa, pb, cs + put.t * n, sn + put.t * n, hl.ja, hl.jb);
                        int64_t to;
                        bool on = true;
                        if (PAGED && x) {
                            to = place.krow[put.t] + put.h * pg.k.h;
                            on = place.krow[put.t] >= 0;
                        } else {
                            to = ((first + put.t) * heads + put.h) * D;
                            if (PAGED && !place.is[put.t]) {
#pragma unroll
                                for (int i = 0; i < V; i++) pa[i] = pb[i] = 0.f;
                            }
                        }
                        if (on && part) {
                            put_piece<DT, V>(dst, to + hl.a, pa);
                            put_piece<DT, V>(dst, to + hl.b, pb);
                        }
                    }
                    put.next();
                }
            }
        }
        if constexpr (PAGED) {
            constexpr int E = DT == DM_F32 ? 4 : 2;
            RowWalk w(r0, BY, max(a.hkv, 1));
            for (int r = r0; r < here * a.hkv; r += BY, w.next()) {
                if (place.vrow[w.t] < 0 || !part) continue;
                const uint4 *from = (const uint4 *)((const char *)v + ((first + w.t) * a.v.t + w.h * a.v.h) * E);
                uint4 *to = (uint4 *)((char *)vo + (place.vrow[w.t] + w.h * pg.v.h) * E);
                const uint4 y = from[li], z = from[li + PIECES];
                to[li] = y, to[li + PIECES] = z;
            }
        }
        if (next >= start && next < a.tokens) {
            RowWalk w(r0, BY, heads0);
            load(next, r0, w, (int)min((int64_t)tile, a.tokens - next) * (ahead_k ? a.hkv : a.hq), ahead_k ? k : q,
                 ahead_k ? a.k : a.q);
        }
        __syncthreads();
        buf ^= 1;
        pl = (pl + 1) % 3;
    }
}

// The gradients, the same rounds. A lane's weight gradients are of its own two pieces for every head that
// it takes, so they stay in registers over the workgroup's tiles (the queries' and the keys' in turn) and
// meet in LDS at the end.
template <int DT, int D, bool INTER>
__global__ __launch_bounds__(256) void rope_bwd_fast(RopeArgs a, int tile, const void *__restrict__ q,
                                                     const void *__restrict__ k, const void *__restrict__ gq,
                                                     const void *__restrict__ gk, void *__restrict__ dq,
                                                     void *__restrict__ dk, float *__restrict__ parts) {
    constexpr int V = rope_v<DT>(), PIECES = rope_pieces<DT, D>(), LPH = rope_lanes(PIECES), BY = 256 / LPH;
    extern __shared__ __align__(16) float lds[];  // the weights [2, D], two tiles' angles; at the end the lanes' sums [BY, D]
    const int tid = threadIdx.x, li = tid % LPH, r0 = tid / LPH, n = a.n;
    float *angles = lds + 2 * D;
    const bool part = PIECES == LPH || li < PIECES;
    const HeadLane<D, V, INTER> hl(part ? li : 0, n);
    float da[2][V] = {}, db[2][V] = {};  // of the heads that are gone through now, and of the others
    const int64_t step = (int64_t)gridDim.x * tile, start = (int64_t)blockIdx.x * tile;
    int buf = 0;
    for (int64_t first = start - step; first < a.tokens; first += step, buf ^= 1) {
        fill_angles<false>(a, first + step, tile, nullptr, angles + (buf ^ 1) * 2 * tile * n);
        if (first < start) fill_weights<D>(a, lds);
        const int here = first < start ? 0 : (int)min((int64_t)tile, a.tokens - first);
        const float *cs = angles + buf * 2 * tile * n, *sn = cs + tile * n;
#pragma unroll 1
        for (int x = 0; x < 2; x++) {
            const int heads = max(x ? a.hkv : a.hq, 1), rows = here * (x ? a.hkv : a.hq);
            const void *src = x ? k : q, *grad = x ? gk : gq;
            void *dst = x ? dk : dq;
            const Strd sd = x ? a.k : a.q, sg = x ? a.gk : a.gq;
            const float *wa = lds + x * D + hl.a, *wb = lds + x * D + hl.b;
            RowWalk w(r0, BY, heads);
            for (int r = r0; r < rows; r += BY, w.next()) {
                const int64_t token = first + w.t, b = token / a.T, t = token - b * a.T;
                const int64_t from = b * sd.b + t * sd.t + w.h * sd.h, g = b * sg.b + t * sg.t + w.h * sg.h;
                const uint4 rxa = raw_piece<DT>(src, from + hl.a), rxb = raw_piece<DT>(src, from + hl.b);
                const uint4 rza = raw_piece<DT>(grad, g + hl.a), rzb = raw_piece<DT>(grad, g + hl.b);
                float xa[V], xb[V], za[V], zb[V], ss = 0.f, gh = 0.f;
                unpack_piece<DT, V>(rxa, xa);
                unpack_piece<DT, V>(rxb, xb);
                if (!part) zero_pieces<V>(xa, xb);
#pragma unroll
                for (int i = 0; i < V; i++) ss += xa[i] * xa[i] + xb[i] * xb[i];
                const float rs = rsqrtf(head_sum<LPH>(ss) * (1.f / D) + a.eps);
                unpack_piece<DT, V>(rza, za);
                unpack_piece<DT, V>(rzb, zb);
                if (!part) zero_pieces<V>(za, zb);
                if (hl.turns) turn_pieces<V, INTER, true>(za, zb, cs + w.t * n, sn + w.t * n, hl.ja, hl.jb);
#pragma unroll
                for (int i = 0; i < V; i++) {
                    xa[i] *= rs, xb[i] *= rs;
                    da[0][i] += za[i] * xa[i], db[0][i] += zb[i] * xb[i];
                    za[i] *= wa[i], zb[i] *= wb[i];
                    gh += za[i] * xa[i] + zb[i] * xb[i];
                }
                const float mean = head_sum<LPH>(gh) * (1.f / D);
#pragma unroll
                for (int i = 0; i < V; i++) {
                    za[i] = rs * (za[i] - xa[i] * mean);
                    zb[i] = rs * (zb[i] - xb[i] * mean);
                }
                const int64_t to = ((first + w.t) * heads + w.h) * D;
                if (part) {
                    put_piece<DT, V>(dst, to + hl.a, za);
                    put_piece<DT, V>(dst, to + hl.b, zb);
                }
            }
#pragma unroll
            for (int i = 0; i < V; i++) {
                const float ta = da[0][i], tb = db[0][i];
                da[0][i] = da[1][i], db[0][i] = db[1][i];
                da[1][i] = ta, db[1][i] = tb;
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int x = 0; x < 2; x++) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; i++)
            if (part) lds[r0 * D + hl.a + i] = da[x][i], lds[r0 * D + hl.b + i] = db[x][i];
        __syncthreads();
        for (int e = tid; e < D; e += 256) {
            float t = 0.f;
            for (int i = 0; i < BY; i++) t += lds[i * D + e];
            parts[((int64_t)blockIdx.x * 2 + x) * D + e] = t;
        }
    }
}

// The workgroups' weight gradients added in order: a workgroup takes 16 columns, its 64 groups of
// threads every 64th part each.
__global__ __launch_bounds__(1024) void rope_weights(const float *__restrict__ parts, int64_t nparts, int d,
                                                     int weight_dtype, void *dwq, void *dwk) {
    __shared__ float sums[64][17];
    const int c = threadIdx.x & 15, g = threadIdx.x >> 4;
    const int64_t col = (int64_t)blockIdx.x * 16 + c;
    float s = 0.f;
    if (col < 2 * d) {
#pragma unroll 8
        for (int64_t i = g; i < nparts; i += 64) s += parts[i * 2 * d + col];
    }
    sums[g][c] = s;
    __syncthreads();
    if (g == 0 && col < 2 * d) {
        float t = 0.f;
#pragma unroll 8
        for (int i = 0; i < 64; i++) t += sums[i][c];
        void *to = col < d ? dwq : dwk;
        if (to) st_any(weight_dtype, to, col < d ? col : col - d, t);
    }
}

// Workgroups of the backward at most: three a compute unit, whose sums are rope_weights' work. (16384 tokens
// of 40 heads of 128 in bf16, replayed: 512 of them 111.5 us, 768 109.6, 2048 118.8; 6144 tokens of 18 heads
// of 256: 49.0, 49.0, 53.9.)
constexpr int64_t kRopeParts = 768;

// The simple kernels' grid: a workgroup a token up to `most`, and where those are few the tokens' heads, four a
// workgroup, shared out too.
static dim3 generic_grid(int64_t tokens, int64_t heads, int64_t most) {
    const int64_t x = std::max<int64_t>(1, std::min(tokens, most));
    return dim3((unsigned)x, (unsigned)std::max<int64_t>(1, std::min((heads + 3) / 4, most / x)));
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

// The fast kernels' calls: 16-byte pieces that no pair leaves.
static bool fast_takes(const dm_qk_norm_rope_desc *d, const RopeArgs &a, const void *const *ptrs, int n,
                       const Strd *strides, int ns) {
    const int v = d->dtype == DM_F32 ? 4 : 8;
    if ((d->d != 64 && d->d != 80 && d->d != 96 && d->d != 128 && d->d != 192 && d->d != 256) || d->n % v != 0)
        return false;
    for (int i = 0; i < n; i++)
        if (!aligned_16b(ptrs[i])) return false;
    for (int i = 0; i < ns; i++)
        if (strides[i].b % v || strides[i].t % v || strides[i].h % v) return false;
    return true;
}

// Tokens of a tile: enough heads for every lane of the workgroup to take four, while there are tiles
// for the compute units to share (at least 1024 workgroups), at most kRopeTile. (16384 tokens of 40 heads
// of 128 in bf16, replayed: two heads a lane 78 us, four 72.7, eight 74.6; 8192 tokens into pages 62, 53.2, 51;
// a tile of one token would leave most lanes of a small call idle, one of sixteen most compute units.)
static int rope_tile(const RopeArgs &a, int by) {
    const int64_t heads = std::max(1, a.hq + a.hkv);
    int64_t tile = 1;
    while (tile < kRopeTile && tile * heads < 4 * by && a.tokens >= 2048 * tile) tile *= 2;
    return (int)tile;
}
// Workgroups at most, as many as are resident and a few rounds more. (The same two: 1024 of them 75.7 and 52.2
// us; 4096 are one a tile there, 72.7 and 53.2. Calls of more tiles, replayed, 4096 workgroups and one a tile: 65536
// tokens of 40 heads of 128 263 and 242 us, 131072 of 10 134 and 130, of 5 heads of 64 49 and 52; into pages 65536 of
// 48 323 and 307, 131072 of 12 173 and 169.)
constexpr int64_t kRopeGrid = 4096;
static size_t rope_lds(const RopeArgs &a, int tile) { return ((size_t)2 * a.d + (size_t)4 * tile * a.n) * sizeof(float); }

// f(type, width, interleaved) as constants, for the fast kernels' widths.
template <int X>
using Int = std::integral_constant<int, X>;
template <typename F>
static void rope_dispatch(const dm_qk_norm_rope_desc *d, F f) {
    auto inter = [&](auto dt, auto width) {
        if (d->interleaved) f(dt, width, Int<1>{});
        else f(dt, width, Int<0>{});
    };
    auto of = [&](auto dt) {
        switch (d->d) {
            case 64: return inter(dt, Int<64>{});
            case 80: return inter(dt, Int<80>{});
            case 96: return inter(dt, Int<96>{});
            case 128: return inter(dt, Int<128>{});
            case 192: return inter(dt, Int<192>{});
            default: return inter(dt, Int<256>{});
        }
    };
    if (d->dtype == DM_F32) of(Int<DM_F32>{});
    else if (d->dtype == DM_BF16) of(Int<DM_BF16>{});
    else of(Int<DM_F16>{});
}

template <int MODE>
static int run_rope(const char *op, const dm_qk_norm_rope_desc *d, const RopeArgs &a, const RopePages &pg,
                    const void *q, const void *k, const void *v, void *qo, void *ko, void *vo,
                    hipStream_t st) {
    const void *ptrs[] = {q, k, qo, ko, v, vo};
    const Strd strides[] = {a.q, a.k, a.v, pg.k, pg.v};
    constexpr bool paged = MODE == kRopePaged;
    if (fast_takes(d, a, ptrs, paged ? 6 : 4, strides, paged ? 5 : 2)) {
        const int by = 256 / rope_lanes((int)(d->d / (d->dtype == DM_F32 ? 8 : 16))), tile = rope_tile(a, by);
        const unsigned grid = (unsigned)std::min((a.tokens + tile - 1) / tile, kRopeGrid);
        const size_t lds = rope_lds(a, tile);
        rope_dispatch(d, [&](auto dt, auto width, auto inter) {
            rope_fast<decltype(dt)::value, decltype(width)::value, MODE, decltype(inter)::value != 0>
                <<<grid, 256, lds, st>>>(a, pg, tile, q, k, v, qo, ko, vo);
        });
    } else {
        const dim3 grid = generic_grid(a.tokens, a.hq + a.hkv * (paged ? 2 : 1), kRopeGrid);
        if (d->dtype == DM_F32)
            rope_generic<DM_F32, MODE><<<grid, 256, 0, st>>>(a, pg, q, k, v, qo, ko, vo);
        else if (d->dtype == DM_BF16)
            rope_generic<DM_BF16, MODE><<<grid, 256, 0, st>>>(a, pg, q, k, v, qo, ko, vo);
        else
            rope_generic<DM_F16, MODE><<<grid, 256, 0, st>>>(a, pg, q, k, v, qo, ko, vo);
    }
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
    int64_t nparts = 0;
    if (a.tokens * (a.hq + a.hkv) > 0) {
        const void *ptrs[] = {q, k, grad_q, grad_k, dq, dk};
        const Strd strides[] = {a.q, a.k, a.gq, a.gk};
        if (fast_takes(d, a, ptrs, 6, strides, 4)) {
            const int by = 256 / rope_lanes((int)(d->d / (d->dtype == DM_F32 ? 8 : 16))), tile = rope_tile(a, by);
            nparts = std::min<int64_t>((a.tokens + tile - 1) / tile, kRopeParts);
            const unsigned grid = (unsigned)nparts;
            const size_t lds = std::max(rope_lds(a, tile), (size_t)by * d->d * sizeof(float));
            rope_dispatch(d, [&](auto dt, auto width, auto inter) {
                rope_bwd_fast<decltype(dt)::value, decltype(width)::value, decltype(inter)::value != 0>
                    <<<grid, 256, lds, st>>>(a, tile, q, k, grad_q, grad_k, dq, dk, parts);
            });
        } else {
            const dim3 grid = generic_grid(a.tokens, a.hq + a.hkv, kRopeParts);
            nparts = (int64_t)grid.x * grid.y;
            if (d->dtype == DM_F32)
                rope_bwd_generic<DM_F32><<<grid, 256, 0, st>>>(a, q, k, grad_q, grad_k, dq, dk, parts);
            else if (d->dtype == DM_BF16)
                rope_bwd_generic<DM_BF16><<<grid, 256, 0, st>>>(a, q, k, grad_q, grad_k, dq, dk, parts);
            else
                rope_bwd_generic<DM_F16><<<grid, 256, 0, st>>>(a, q, k, grad_q, grad_k, dq, dk, parts);
        }
    }
    if (dq_weight || dk_weight)
        rope_weights<<<(unsigned)((2 * a.d + 15) / 16), 1024, 0, st>>>(parts, nparts, a.d, a.weight_dtype,
                                                                      dq_weight, dk_weight);
    probe_add(DM_PROBE_QK_NORM_ROPE_BWD);
    DM_LAUNCH_CHECK((op + ": launch").c_str());
    return DM_OK;
}

// turned: by the descriptor's positions, where it has some.
static int rope_paged(const dm_qk_norm_rope_desc *d, bool turned, const dm_kv_pages *pages, const void *q,
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
    RopeArgs a = rope_args(d, q_weight, k_weight, inv_freq);
    if (!turned) a.positions = nullptr;
    return run_rope<kRopePaged>(op.c_str(), d, a, pg, q, k, v, q_out, k_pages, v_pages, (hipStream_t)stream);
}

int dm_qk_norm_rope_paged(const dm_qk_norm_rope_desc *d, const dm_kv_pages *pages, const void *q,
                          const void *k, const void *v, const void *q_weight, const void *k_weight,
                          const float *inv_freq, void *q_out, void *k_pages, void *v_pages, void *stream) {
    return rope_paged(d, false, pages, q, k, v, q_weight, k_weight, inv_freq, q_out, k_pages, v_pages, stream);
}

int dm_qk_norm_rope_paged_at(const dm_qk_norm_rope_desc *d, const dm_kv_pages *pages, const void *q,
                             const void *k, const void *v, const void *q_weight, const void *k_weight,
                             const float *inv_freq, void *q_out, void *k_pages, void *v_pages, void *stream) {
    return rope_paged(d, true, pages, q, k, v, q_weight, k_weight, inv_freq, q_out, k_pages, v_pages, stream);
}

}  // extern "C"
