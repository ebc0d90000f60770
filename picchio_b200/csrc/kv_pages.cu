// kv_pages.cu - the bookkeeping of a paged KV cache on the device: the tables
// of one serving step from the requests' lengths, and the store of new K and V
// rows to their slots.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "launch.cuh"
#include "paged.h"

namespace pc {

namespace {

constexpr int TAB_THREADS = 1024;

// Sums stop here (adding so stays associative): 1024 requests can ask for more
// than 32 bits hold, and whatever is above every capacity is refused alike.
// Capacities and single values are at most half of it.
constexpr int TAB_MOST = 1 << 29;
__device__ __forceinline__ int add_most(int a, int b) { return min(a + b, TAB_MOST); }

// Inclusive sums over the block of three values at once, none below zero.
__device__ __forceinline__ void block_scan3(int (&v)[3], int (&all)[3], int (*sh)[TAB_THREADS / 32]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int c = 0; c < 3; ++c)
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, v[c], o);
            if (lane >= o) v[c] = add_most(v[c], u);
        }
    __syncthreads();
    if (lane == 31)
#pragma unroll
        for (int c = 0; c < 3; ++c) sh[c][warp] = v[c];
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 3; ++c) {
        int inc = sh[c][lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc = add_most(inc, u);
        }
        all[c] = __shfl_sync(0xffffffffu, inc, 31);
        const int before = __shfl_sync(0xffffffffu, inc, (warp + 31) & 31);
        if (warp) v[c] = add_most(v[c], before);
    }
}

// Position and slot of the step's row t: its request by bisection of cu_new.
__device__ __forceinline__ void row_slot(const pc_kv_step &s, int t, int total) {
    if (t >= total) {
        s.pos_dev[t] = -1;
        s.slot_dev[t] = -1;
        return;
    }
    int lo = 0, hi = s.n_requests;  // cu_new[lo] <= t < cu_new[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s.cu_new_dev[mid] <= t) lo = mid;
        else hi = mid;
    }
    const int p = max(s.kv_len_dev[lo], 0) + t - s.cu_new_dev[lo], page = p / s.page_size;
    s.pos_dev[t] = p;
    s.slot_dev[t] = (int64_t)s.page_table_dev[(int64_t)lo * s.max_pages + page] * s.page_size + p % s.page_size;
}

// Up to how many rows the table block fills in itself, one a thread; more
// rows have a launch of their own, which is 2 us more for the smallest steps
// and saves 50 us at 16,000 rows.
constexpr int TAB_ROWS = TAB_THREADS;

// One block: the requests in chunks of 1024, each chunk a scan; a request's
// pages are moved by its thread if they are one or two, else by its warp.
// Bound by latency: a few dependent trips to L2 and the scans' barriers.
// Measured: 64 requests, one token each 4.1 us; 512 requests with 60 chunks of
// up to 512 and 25 ended, 16,384 rows 16 us (72 us with one thread filling each
// request's pages and rows).
__global__ void __launch_bounds__(TAB_THREADS) kv_tables_kernel(const pc_kv_step s) {
    __shared__ int sh[3][TAB_THREADS / 32];
    const int tid = threadIdx.x, lane = tid & 31, P = s.page_size;
    pdl_wait();
    pdl_trigger();
    const int n_free = min(max(*s.n_free_dev, 0), s.free_cap);
    // `move(b, j, at)` for the n things of request b that go to `at` on
    auto each = [&](int b, int n, int at, auto move) {
        if (n <= 2)
            for (int j = 0; j < n; ++j) move(b, j, at + j);
        for (unsigned more = __ballot_sync(0xffffffffu, n > 2); more; more &= more - 1) {
            const int src = __ffs(more) - 1;
            const int bb = __shfl_sync(0xffffffffu, b, src), nn = __shfl_sync(0xffffffffu, n, src),
                      aa = __shfl_sync(0xffffffffu, at, src);
            for (int j = lane; j < nn; j += 32) move(bb, j, aa + j);
        }
    };
    // pages of ended requests on top of the free ones
    int given = 0;
    for (int b0 = 0; b0 < s.n_requests; b0 += TAB_THREADS) {
        const int b = b0 + tid;
        int v[3] = {0, 0, 0}, all[3];
        if (b < s.n_requests && s.new_len_dev[b] < 0)
            v[0] = min((int)(((int64_t)max(s.kv_len_dev[b], 0) + P - 1) / P), s.max_pages);
        const int n = v[0];
        if (!__syncthreads_or(n)) continue;
        block_scan3(v, all, sh);
        each(b, n, n_free + given + v[0] - n, [&](int r, int j, int at) {
            if (at < s.free_cap) s.free_pages_dev[at] = s.page_table_dev[(int64_t)r * s.max_pages + j];
        });
        given = add_most(given, all[0]);
    }
    const int avail = min(n_free + given, s.free_cap);
    __syncthreads();
    int want0 = 0, add0 = 0, took0 = 0, used = 0;
    for (int b0 = 0; b0 < s.n_requests; b0 += TAB_THREADS) {
        const int b = b0 + tid;
        int v[3] = {0, 0, 0}, all[3];
        int kv = 0, add = 0, held = 0;
        bool fits = false, ended = false;
        if (b < s.n_requests) {
            kv = max(s.kv_len_dev[b], 0);
            add = s.new_len_dev[b];
            ended = add < 0;
            fits = !ended && (int64_t)kv + add <= (int64_t)s.max_pages * P;
            held = fits ? (kv + P - 1) / P : 0;
            v[0] = fits ? (kv + add + P - 1) / P - held : 0;
            v[1] = fits ? min(add, s.n_tokens + 1) : 0;
        }
        const int want = v[0];
        block_scan3(v, all, sh);
        const int upto = add_most(want0, v[0]), tokens = add_most(add0, v[1]);
        const bool ok = fits && (want == 0 || upto <= avail) && (add == 0 || tokens <= s.n_tokens);
        int u[3] = {ok ? add : 0, ok ? want : 0, 0}, uall[3];
        block_scan3(u, uall, sh);
        // request b's page held + j is the (upto - want + j)-th from the top of the free ones
        const int first = ok && want ? upto - want : 0;
        each(b, ok ? want : 0, first, [&](int r, int j, int nth) {
            const int kept = (max(s.kv_len_dev[r], 0) + P - 1) / P;
            s.page_table_dev[(int64_t)r * s.max_pages + kept + j] = s.free_pages_dev[avail - 1 - nth];
        });
        if (b < s.n_requests) {
            s.kv_end_dev[b] = ended ? 0 : ok ? kv + add : kv;
            s.served_dev[b] = ok;
            s.cu_new_dev[b + 1] = took0 + u[0];
        }
        want0 = add_most(want0, all[0]);
        add0 = add_most(add0, all[1]);
        took0 += uall[0];
        used += uall[1];
    }
    if (tid == 0) {
        s.cu_new_dev[0] = 0;
        *s.n_free_out_dev = avail - used;
    }
    if (s.n_tokens > TAB_ROWS) return;
    __syncthreads();
    if (tid < s.n_tokens) row_slot(s, tid, took0);
}

__global__ void __launch_bounds__(256) kv_slots_kernel(const pc_kv_step s) {
    pdl_wait();
    pdl_trigger();
    const int t = blockIdx.x * 256 + threadIdx.x;
    if (t < s.n_tokens) row_slot(s, t, s.cu_new_dev[s.n_requests]);
}

struct StoreOp {
    void *kc, *vc;
    const void *k, *v;
    int64_t kcs[3], vcs[3], ks[2], vs[2];
    const int64_t *slot;
    int64_t slots;
    int n, page, KVH, D;
};

template <typename S>
__device__ __forceinline__ float up(S v) { return (float)v; }
template <typename D>
__device__ __forceinline__ D down(float v);
template <> __device__ __forceinline__ float down<float>(float v) { return v; }
template <> __device__ __forceinline__ __half down<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 down<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 8 elements as loaded and stored: 16 or 32 bytes
template <typename T>
__device__ __forceinline__ void load8(const T *p, float (&f)[8]) {
    uint4 r[sizeof(T) / 2];
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) r[i] = __ldcs(reinterpret_cast<const uint4 *>(p) + i);
    const T *t = reinterpret_cast<const T *>(r);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = up(t[i]);
}
template <typename T>
__device__ __forceinline__ void store8(T *p, const float (&f)[8]) {
    uint4 r[sizeof(T) / 2];
    T *t = reinterpret_cast<T *>(r);
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = down<T>(f[i]);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4 *>(p)[i] = r[i];
}

// A block takes `rows` rows of the step, a thread 8 elements of K and the same
// of V at a time.  Bytes only: 16-byte loads and stores, all of a thread's
// loads before its stores.  Measured: 16,301 rows of 8 x 128 bf16 26 us, 5.1
// TB/s (79 % of the measured copy; element by element 57 us); 64 rows 1.6 us.
constexpr int ST_UNROLL = 2;
template <typename S, typename D>
__global__ void __launch_bounds__(256) kv_store_kernel(const StoreOp o, const int rows) {
    pdl_wait();
    pdl_trigger();
    const int per = o.D / 8, row = o.KVH * per;
    const int64_t t0 = (int64_t)blockIdx.x * rows;
    const int n = (int)min((int64_t)rows, o.n - t0) * row;
    for (int i0 = threadIdx.x; i0 < n; i0 += 256 * ST_UNROLL) {
        float k[ST_UNROLL][8], v[ST_UNROLL][8];
        int64_t kd[ST_UNROLL], vd[ST_UNROLL];
#pragma unroll
        for (int u = 0; u < ST_UNROLL; ++u) {
            const int i = i0 + 256 * u;
            kd[u] = -1;
            if (i >= n) continue;
            const int r = i / row, c = i - r * row, h = c / per, d = (c - h * per) * 8;
            const int64_t t = t0 + r, slot = o.slot[t];
            if (slot < 0 || slot >= o.slots) continue;
            int64_t page, at;
            if (slot >> 31 == 0) {
                page = (unsigned)slot / (unsigned)o.page;
                at = (unsigned)slot - (unsigned)page * (unsigned)o.page;
            } else {
                page = slot / o.page;
                at = slot - page * o.page;
            }
            kd[u] = page * o.kcs[0] + at * o.kcs[1] + h * o.kcs[2] + d;
            vd[u] = page * o.vcs[0] + at * o.vcs[1] + h * o.vcs[2] + d;
            load8(reinterpret_cast<const S *>(o.k) + t * o.ks[0] + h * o.ks[1] + d, k[u]);
            load8(reinterpret_cast<const S *>(o.v) + t * o.vs[0] + h * o.vs[1] + d, v[u]);
        }
#pragma unroll
        for (int u = 0; u < ST_UNROLL; ++u)
            if (kd[u] >= 0) {
                store8(reinterpret_cast<D *>(o.kc) + kd[u], k[u]);
                store8(reinterpret_cast<D *>(o.vc) + vd[u], v[u]);
            }
    }
}

template <typename S>
cudaError_t store_to(const StoreOp &o, int dtype, int nsm, cudaStream_t st) {
    // rows a block: two pieces a thread, fewer while that leaves SMs without a block
    const int row = o.KVH * (o.D / 8);
    int rows = std::max(1, 256 * ST_UNROLL / row);
    while (rows > 1 && (int64_t)o.n < (int64_t)rows * nsm) rows = (rows + 1) / 2;
    const int grid = (o.n + rows - 1) / rows;
    if (dtype == PC_DT_F32) return launch_k(kv_store_kernel<S, float>, dim3(grid), dim3(256), 0, st, o, rows);
    if (dtype == PC_DT_F16) return launch_k(kv_store_kernel<S, __half>, dim3(grid), dim3(256), 0, st, o, rows);
    return launch_k(kv_store_kernel<S, __nv_bfloat16>, dim3(grid), dim3(256), 0, st, o, rows);
}

}  // namespace

cudaError_t launch_kv_tables(const pc_kv_step &s, cudaStream_t st) {
    const cudaError_t e = launch_k(kv_tables_kernel, dim3(1), dim3(TAB_THREADS), 0, st, s);
    if (e != cudaSuccess || s.n_tokens <= TAB_ROWS) return e;
    return launch_k(kv_slots_kernel, dim3((s.n_tokens + 255) / 256), dim3(256), 0, st, s);
}

cudaError_t launch_kv_store(const pc_kv_pages &kv, const void *k, const int64_t *ks, const void *v, const int64_t *vs,
                            int src_dtype, const int64_t *slot, int n, int nsm, cudaStream_t st) {
    StoreOp o;
    o.kc = kv.k_dev;
    o.vc = kv.v_dev;
    o.k = k;
    o.v = v;
    for (int i = 0; i < 3; ++i) {
        o.kcs[i] = kv.k_stride[i];
        o.vcs[i] = kv.v_stride[i];
    }
    for (int i = 0; i < 2; ++i) {
        o.ks[i] = ks[i];
        o.vs[i] = vs[i];
    }
    o.slot = slot;
    o.slots = (int64_t)kv.n_pages * kv.page_size;
    o.n = n;
    o.page = kv.page_size;
    o.KVH = kv.n_kv_heads;
    o.D = kv.head_dim;
    if (src_dtype == PC_DT_F32) return store_to<float>(o, kv.dtype, nsm, st);
    if (src_dtype == PC_DT_F16) return store_to<__half>(o, kv.dtype, nsm, st);
    return store_to<__nv_bfloat16>(o, kv.dtype, nsm, st);
}

}  // namespace pc
