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

// Inclusive sums over the block of three values at once.
__device__ __forceinline__ void block_scan3(int (&v)[3], int (&all)[3], int (*sh)[TAB_THREADS / 32]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int c = 0; c < 3; ++c)
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, v[c], o);
            if (lane >= o) v[c] += u;
        }
    __syncthreads();
    if (lane == 31)
#pragma unroll
        for (int c = 0; c < 3; ++c) sh[c][warp] = v[c];
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 3; ++c) {
        const int x = sh[c][lane];
        int inc = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += u;
        }
        all[c] = __shfl_sync(0xffffffffu, inc, 31);
        v[c] += __shfl_sync(0xffffffffu, inc - x, warp);
    }
}

// One block: the requests in chunks of 1024, each chunk a scan.
__global__ void __launch_bounds__(TAB_THREADS) kv_tables_kernel(const pc_kv_step s) {
    __shared__ int sh[3][TAB_THREADS / 32];
    const int tid = threadIdx.x, P = s.page_size;
    pdl_wait();
    pdl_trigger();
    const int n_free = min(max(*s.n_free_dev, 0), s.free_cap);
    // pages of ended requests on top of the free ones
    int given = 0;
    for (int b0 = 0; b0 < s.n_requests; b0 += TAB_THREADS) {
        const int b = b0 + tid;
        int v[3] = {0, 0, 0}, all[3];
        if (b < s.n_requests && s.new_len_dev[b] < 0)
            v[0] = min((max(s.kv_len_dev[b], 0) + P - 1) / P, s.max_pages);
        const int n = v[0];
        block_scan3(v, all, sh);
        const int at = n_free + given + v[0] - n;
        for (int j = 0; j < n; ++j)
            if (at + j < s.free_cap) s.free_pages_dev[at + j] = s.page_table_dev[(int64_t)b * s.max_pages + j];
        given += all[0];
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
            held = (kv + P - 1) / P;
            v[0] = fits ? (kv + add + P - 1) / P - held : 0;
            v[1] = fits ? min(add, s.n_tokens + 1) : 0;
        }
        const int want = v[0];
        block_scan3(v, all, sh);
        const int64_t upto = (int64_t)want0 + v[0], tokens = (int64_t)add0 + v[1];
        const bool ok = fits && (want == 0 || upto <= avail) && (add == 0 || tokens <= s.n_tokens);
        int u[3] = {ok ? add : 0, ok ? want : 0, 0}, uall[3];
        block_scan3(u, uall, sh);
        if (b < s.n_requests) {
            int *row = s.page_table_dev + (int64_t)b * s.max_pages;
            if (ok)
                for (int j = 0; j < want; ++j) row[held + j] = s.free_pages_dev[avail - 1 - (int)(upto - want) - j];
            s.kv_end_dev[b] = ended ? 0 : ok ? kv + add : kv;
            s.served_dev[b] = ok;
            s.cu_new_dev[b + 1] = took0 + u[0];
            if (ok)
                for (int i = 0; i < add; ++i) {
                    const int p = kv + i, t = took0 + u[0] - add + i;
                    s.pos_dev[t] = p;
                    s.slot_dev[t] = (int64_t)row[p / P] * P + p % P;
                }
        }
        want0 = (int)min((int64_t)want0 + all[0], (int64_t)1 << 30);
        add0 = (int)min((int64_t)add0 + all[1], (int64_t)1 << 30);
        took0 += uall[0];
        used += uall[1];
    }
    for (int t = took0 + tid; t < s.n_tokens; t += TAB_THREADS) {
        s.pos_dev[t] = -1;
        s.slot_dev[t] = -1;
    }
    if (tid == 0) {
        s.cu_new_dev[0] = 0;
        *s.n_free_out_dev = avail - used;
    }
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

template <typename T>
struct alignas(sizeof(T) * 8) Vec8 {
    T v[8];
};

// A thread moves 8 elements of a K row and the same of the V row.
template <typename S, typename D>
__global__ void __launch_bounds__(256) kv_store_kernel(const StoreOp o) {
    pdl_wait();
    pdl_trigger();
    const int per = o.D / 8, row = o.KVH * per;
    const int64_t n = (int64_t)o.n * row;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
        const int t = (int)(i / row), c = (int)(i % row), h = c / per, d = (c % per) * 8;
        const int64_t slot = o.slot[t];
        if (slot < 0 || slot >= o.slots) continue;
        const int64_t page = slot / o.page, r = slot % o.page;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const S *src = reinterpret_cast<const S *>(w ? o.v : o.k) + t * (w ? o.vs : o.ks)[0] +
                           h * (w ? o.vs : o.ks)[1] + d;
            const int64_t *cs = w ? o.vcs : o.kcs;
            D *dst = reinterpret_cast<D *>(w ? o.vc : o.kc) + page * cs[0] + r * cs[1] + h * cs[2] + d;
            D y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = down<D>(up(src[j]));
#pragma unroll
            for (int j = 0; j < 8; ++j) dst[j] = y[j];
        }
    }
}

template <typename S>
cudaError_t store_to(const StoreOp &o, int dtype, int grid, cudaStream_t st) {
    if (dtype == PC_DT_F32) return launch_k(kv_store_kernel<S, float>, dim3(grid), dim3(256), 0, st, o);
    if (dtype == PC_DT_F16) return launch_k(kv_store_kernel<S, __half>, dim3(grid), dim3(256), 0, st, o);
    return launch_k(kv_store_kernel<S, __nv_bfloat16>, dim3(grid), dim3(256), 0, st, o);
}

}  // namespace

cudaError_t launch_kv_tables(const pc_kv_step &s, cudaStream_t st) {
    return launch_k(kv_tables_kernel, dim3(1), dim3(TAB_THREADS), 0, st, s);
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
    const int64_t work = (int64_t)n * o.KVH * (o.D / 8);
    const int grid = (int)std::min<int64_t>((work + 255) / 256, (int64_t)nsm * 8);
    if (src_dtype == PC_DT_F32) return store_to<float>(o, kv.dtype, grid, st);
    if (src_dtype == PC_DT_F16) return store_to<__half>(o, kv.dtype, grid, st);
    return store_to<__nv_bfloat16>(o, kv.dtype, grid, st);
}

}  // namespace pc
