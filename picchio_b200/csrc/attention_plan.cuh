// attention_plan.cuh - how the attention kernels over pages and packed
// prompts cut their work between thread blocks.
//
// The rows of one request that share a KV head (tokens x query heads of the
// group, token-major, so the causal edge of a block of rows is short) are cut
// into items of R rows; an item's keys are cut into tiles of KT.  The items
// of all (request, KV head) pairs stand on one line, each as long as its work
// (its keys, plus a constant for what an item costs besides), and every
// thread block takes an equal share of that line.  So ragged batches, causal
// triangles and single long rows all give balanced blocks, and the lengths
// are read on the device: the host needs none.  An item cut by a share's end
// is finished by several blocks: each leaves (O, m, l) in the workspace and
// the last to arrive adds them up in block order, so the result does not
// depend on who came last.
//
// The length of the first i items of a request has a closed form (causal: a
// triangle, with a window then a line), so a share's end is found by one scan
// over the requests and a bisection, without a list of items.
#pragma once
#include <cstdint>

#include "paged.h"

namespace pc {

// f / G for the flat row f = token * G + head of a group of G heads (f * G <
// 2^32, checked on the host)
__device__ __forceinline__ int div_g(const AttnOp &a, int f) {
    return a.G == 1 ? f : (int)__umulhi((unsigned)f, a.inv_g);
}

// A request's rows and keys as every kernel reads them, safe for any input.
struct SeqGeo {
    int q0, qlen, kv, p0, n_items;  // first row, rows, keys, first row's position (may be < 0), items
};

template <int R>
__device__ __forceinline__ SeqGeo seq_geo(const AttnOp &a, int b) {
    SeqGeo s;
    const int lo = min(max(a.cu[b], 0), a.T), hi = min(max(a.cu[b + 1], 0), a.T);
    s.q0 = lo;
    s.qlen = max(hi - lo, 0);
    const int rows = s.qlen * a.G;
    if (rows < a.min_q || rows > a.max_q) s.qlen = 0;
    s.kv = a.table ? (int)min((int64_t)max(a.kv_len[b], 0), (int64_t)a.max_pages * a.page_size) : s.qlen;
    s.p0 = s.kv - s.qlen;
    s.n_items = (s.qlen * a.G + R - 1) / R;
    return s;
}

// Whether a kernel that takes min_q <= rows <= max_q takes request b.
__device__ __forceinline__ bool takes(const int *cu, int b, int T, int G, int min_q, int max_q) {
    const int lo = min(max(__ldcg(cu + b), 0), T), hi = min(max(__ldcg(cu + b + 1), 0), T);
    const int rows = max(hi - lo, 0) * G;
    return rows >= min_q && rows <= max_q;
}

// Whether a launch beside another of the same call (min_q > 1) finds no request
// to take; every thread of the block calls it, before pdl_wait.  The launch
// before it lets this one start only after its own wait, so `cu` is written by
// then; the block must wait as well before it ends, since what comes next waits
// for this launch alone.
__device__ __forceinline__ bool nothing_to_take(const int *cu, int B, int T, int G, int min_q, int max_q) {
    bool any = false;
    for (int b = threadIdx.x; b < B; b += blockDim.x) any |= takes(cu, b, T, G, min_q, max_q);
    return !__syncthreads_or(any);
}

// The next request after b that a kernel takes, or one past `last`; a warp
// calls it, so that slots without a request cost little.
__device__ __forceinline__ int next_request(const int *cu, int b, int last, int T, int G, int min_q, int max_q) {
    for (int b0 = b + 1; b0 <= last; b0 += 32) {
        const int mine = b0 + (int)(threadIdx.x & 31);
        const unsigned m = __ballot_sync(0xffffffffu, mine <= last && takes(cu, mine, T, G, min_q, max_q));
        if (m) return b0 + __ffs(m) - 1;
    }
    return last + 1;
}

// Rows [r0, r1) of the request's tokens x group, keys [kb, ke), tiles of KT
// from tile t0 on (at least one, so that rows without keys are written).
struct ItemGeo {
    int r0, r1, pmin, pmax, kb, ke, t0, nt;
};

template <int R, int KT>
__device__ __forceinline__ ItemGeo item_geo(const AttnOp &a, const SeqGeo &s, int item) {
    ItemGeo g;
    g.r0 = item * R;
    g.r1 = min(g.r0 + R, s.qlen * a.G);
    g.pmin = s.p0 + div_g(a, g.r0);
    g.pmax = s.p0 + div_g(a, g.r1 - 1);
    g.kb = a.window > 0 ? max(0, g.pmin - a.window + 1) : 0;
    g.ke = max(g.pmax + 1, 0);
    g.t0 = g.kb / KT;
    g.nt = max(1, (g.ke + KT - 1) / KT - g.t0);
    return g;
}

// a / b of numbers that are not negative: the 64-bit division is a routine of
// its own, worth going round in the short calls, where the numbers are small
__device__ __forceinline__ int64_t div_len(int64_t a, int64_t b) {
    if (((a | b) >> 32) == 0) return (uint32_t)a / (uint32_t)b;
    return a / b;
}

// Length of the first i items of a request and one KV head, in keys x group.
template <int R, int KT, int OV>
__device__ __forceinline__ int64_t items_len(const AttnOp &a, const SeqGeo &s, int i) {
    const int64_t A = (int64_t)s.p0 * a.G;
    int64_t lo = A < 0 ? min((int64_t)i, div_len(-A, R)) : 0;  // items without keys
    int64_t hi = i;                                     // from here on the window's length
    const int64_t W = (int64_t)a.window * a.G + R;
    if (a.window > 0) hi = max(lo, min((int64_t)i, A >= W ? (int64_t)0 : div_len(W - A, R)));
    return (int64_t)i * OV * a.G + (hi - lo) * A + R * (hi * (hi + 1) - lo * (lo + 1)) / 2 + (i - hi) * W;
}

// A point on the line: tile `tile` of an item; len0, len: where the item
// starts and how long it is.
struct PlanPoint {
    int b, kvh, item, tile;
    int64_t len0, len;
};

struct PlanShare {
    PlanPoint s, e;  // first tile, one past the last
    int64_t total;
    int n;  // thread blocks that have a share
};

template <int THREADS>
struct PlanScratch {
    int64_t warp[THREADS / 32];
    int64_t base[2];  // where the requests of the two ends start
    int b[2];
    int64_t total;
    PlanShare share;
};

__device__ __forceinline__ int64_t share_start(int64_t total, int n, int k) { return div_len(total * k, n); }

template <int R, int KT, int OV>
__device__ __forceinline__ void plan_point(const AttnOp &a, int b, int64_t base, int64_t x, PlanPoint &p) {
    const SeqGeo s = seq_geo<R>(a, b);
    const int64_t per = items_len<R, KT, OV>(a, s, s.n_items);
    p.b = b;
    p.kvh = (int)div_len(x - base, per);
    const int64_t r = (x - base) - p.kvh * per;
    int lo = 0, hi = s.n_items;  // items_len(lo) <= r < items_len(hi)
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (items_len<R, KT, OV>(a, s, mid) <= r) lo = mid;
        else hi = mid;
    }
    p.item = lo;
    const int64_t c0 = items_len<R, KT, OV>(a, s, lo);
    p.len = items_len<R, KT, OV>(a, s, lo + 1) - c0;
    p.len0 = base + p.kvh * per + c0;
    const ItemGeo g = item_geo<R, KT>(a, s, lo);
    p.tile = (int)div_len((r - c0) * g.nt, p.len);
}

// The share of thread block `cta` of `ctas`; every thread of the block calls
// it.  MINK: keys that a share has at least (the whole batch has fewer blocks
// then).
template <int R, int KT, int OV, int MINK, int THREADS>
__device__ void plan_share(const AttnOp &a, int cta, int ctas, PlanScratch<THREADS> &sc) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int NW = THREADS / 32;
    int64_t mine = 0, sum = 0;
    for (int b = tid; b < a.B; b += THREADS) {
        const SeqGeo s = seq_geo<R>(a, b);
        mine = a.KVH * items_len<R, KT, OV>(a, s, s.n_items);
        sum += mine;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sc.warp[warp] = sum;
    if (tid < 2) sc.b[tid] = a.B;
    __syncthreads();
    int64_t total = 0;
    for (int w = 0; w < NW; ++w) total += sc.warp[w];
    // no share is shorter than an item's longest tile, so no share of an item
    // it touches is empty
    int64_t least = (int64_t)a.G * (max(KT, MINK) + OV + 1) + R + 1;
    const int n = (int)max((int64_t)1, min((int64_t)ctas, div_len(total, least)));
    if (cta >= n || total == 0) {
        if (tid == 0) sc.share.n = 0;
        __syncthreads();
        return;
    }
    const int64_t x0 = share_start(total, n, cta), x1 = share_start(total, n, cta + 1);
    if (a.B == 1 && tid < 2) {
        sc.b[tid] = (tid ? x1 : x0) < total ? 0 : 1;
        sc.base[tid] = 0;
    }
    int64_t carry = 0;
    for (int b0 = 0; b0 < (a.B == 1 ? 0 : a.B); b0 += THREADS) {
        const int b = b0 + tid;
        if (a.B > THREADS) {
            mine = 0;
            if (b < a.B) {
                const SeqGeo s = seq_geo<R>(a, b);
                mine = a.KVH * items_len<R, KT, OV>(a, s, s.n_items);
            }
        }
        int64_t inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        __syncthreads();  // sc.warp is free
        if (lane == 31) sc.warp[warp] = inc;
        __syncthreads();
        int64_t before = carry, all = 0;
        for (int w = 0; w < NW; ++w) {
            if (w < warp) before += sc.warp[w];
            all += sc.warp[w];
        }
        const int64_t end = before + inc, start = end - mine;
        if (x0 >= start && x0 < end) { sc.b[0] = b; sc.base[0] = start; }
        if (x1 >= start && x1 < end) { sc.b[1] = b; sc.base[1] = start; }
        carry += all;
    }
    __syncthreads();
    if (tid == 0) {
        sc.share.n = n;
        sc.share.total = total;
        plan_point<R, KT, OV>(a, sc.b[0], sc.base[0], x0, sc.share.s);
    }
    if (tid == 32) {
        if (sc.b[1] < a.B) {
            plan_point<R, KT, OV>(a, sc.b[1], sc.base[1], x1, sc.share.e);
        } else {
            sc.share.e.b = a.B;
            sc.share.e.kvh = sc.share.e.item = sc.share.e.tile = 0;
        }
    }
    __syncthreads();
}

// The walk over a share's items: the tiles [tl, th) of item `item` of (b,
// kvh) are this block's.
template <int R, int KT>
struct PlanWalk {
    const AttnOp &a;
    const PlanShare &sh;
    int b, kvh, item, tl, th;
    bool first;
    SeqGeo s;
    ItemGeo g;

    __device__ __forceinline__ PlanWalk(const AttnOp &a_, const PlanShare &sh_) : a(a_), sh(sh_) {
        b = sh.s.b;
        kvh = sh.s.kvh;
        item = sh.s.item;
        first = true;
    }
    // false: the share is done.  Sets tl, th, s, g for the item at hand.
    __device__ __forceinline__ bool load(bool request = true) {
        if (b >= a.B) return false;
        if (request) s = seq_geo<R>(a, b);
        if (s.n_items == 0) {
            b = next_request(a.cu, b, min(sh.e.b, a.B - 1), a.T, a.G, a.min_q, a.max_q);
            if (b >= a.B) return false;
            s = seq_geo<R>(a, b);
        }
        const bool at_end = b == sh.e.b && kvh == sh.e.kvh && item == sh.e.item;
        if (b > sh.e.b || (at_end && sh.e.tile == 0)) return false;
        g = item_geo<R, KT>(a, s, item);
        tl = first ? sh.s.tile : 0;
        th = at_end ? sh.e.tile : g.nt;
        return th > tl;
    }
    __device__ __forceinline__ bool next() {
        if (b == sh.e.b && kvh == sh.e.kvh && item == sh.e.item) return false;  // cut here
        first = false;
        bool request = false;
        if (++item == s.n_items) {
            item = 0;
            if (++kvh == a.KVH) {
                kvh = 0;
                ++b;
                request = true;
            }
        }
        return load(request);
    }
    __device__ __forceinline__ bool whole() const { return tl == 0 && th == g.nt; }
};

// Who finishes a cut item: thread blocks k0 .. k1; block k0 has its first
// tile and left its part in slot 1, the others in slot 0.
struct CutItem {
    int k0, k1;
};

template <int R, int KT>
__device__ __forceinline__ CutItem cut_item(const PlanWalk<R, KT> &w) {
    // an item that a share cuts is the share's first or its last
    const PlanPoint &p = w.first ? w.sh.s : w.sh.e;
    const int64_t total = w.sh.total;
    const int n = w.sh.n;
    CutItem c;
    c.k0 = (int)div_len((p.len0 + 1) * n - 1, total);
    c.k1 = (int)div_len((p.len0 + p.len) * n - 1, total);
    if (c.k0 < c.k1 && (share_start(total, n, c.k0 + 1) - p.len0) * w.g.nt < p.len) ++c.k0;
    return c;
}

}  // namespace pc
