// paged.cu - the C entry points of the paged KV cache operators: checks of
// their arguments, the attention workspace, and the choice of a kernel.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstring>
#include <string>

#include "context.h"
#include "paged.h"

struct pc_attn {
    int dev = 0, nsm = 148;
    float *part = nullptr;
    unsigned *ticket = nullptr;
    int *err = nullptr;
};

namespace {

using namespace pc;

// The device of a call, and the caller's again when it returns.
struct OnDevice {
    int old = -1;
    cudaError_t e;
    explicit OnDevice(int dev) {
        e = cudaGetDevice(&old);
        if (e == cudaSuccess && old != dev) e = cudaSetDevice(dev);
        else old = -1;
    }
    ~OnDevice() {
        if (old >= 0) cudaSetDevice(old);
    }
};

int dt_size(int dt) { return dt == PC_DT_F32 ? 4 : 2; }
bool dt_ok(int dt) { return dt == PC_DT_F32 || dt == PC_DT_F16 || dt == PC_DT_BF16; }

// Rows start on 16-byte boundaries (16-byte loads, tensor maps).
bool aligned(const void *p, const int64_t *s, int n, int esize) {
    if ((uintptr_t)p % 16) return false;
    for (int i = 0; i < n; ++i)
        if (s[i] < 0 || (s[i] * esize) % 16) return false;
    return true;
}

pc_status check_pages(const pc_kv_pages *kv) {
    if (!kv || !kv->k_dev || !kv->v_dev || kv->n_pages < 1 || kv->n_kv_heads < 1)
        return fail(PC_ERR_INVALID_ARG, "bad pc_kv_pages");
    if (!dt_ok(kv->dtype)) return fail(PC_ERR_FORMAT, "cache type must be PC_DT_F32, PC_DT_F16 or PC_DT_BF16");
    if (kv->head_dim < 8 || kv->head_dim > 128 || kv->head_dim % 8)
        return fail(PC_ERR_FORMAT, "head_dim must be a multiple of 8, at most 128");
    if (kv->page_size < 8 || kv->page_size % 8 || kv->page_size > (1 << 16))
        return fail(PC_ERR_FORMAT, "page_size must be a multiple of 8, at most 65536");
    const int es = dt_size(kv->dtype);
    if (!aligned(kv->k_dev, kv->k_stride, 3, es) || !aligned(kv->v_dev, kv->v_stride, 3, es))
        return fail(PC_ERR_FORMAT, "K and V pages need 16-byte aligned pointers and strides");
    return PC_OK;
}

pc_status check_call(const pc_attn_call *c) {
    if (!c || c->n_rows < 0 || c->n_requests < 0 || c->n_heads < 1 || c->n_kv_heads < 1 || c->window < 0 ||
        !(c->scale > 0.0f) || !std::isfinite(c->scale))
        return fail(PC_ERR_INVALID_ARG, "bad pc_attn_call");
    if (c->n_heads % c->n_kv_heads) return fail(PC_ERR_INVALID_ARG, "n_heads must be a multiple of n_kv_heads");
    if (c->n_heads / c->n_kv_heads > 128) return fail(PC_ERR_FORMAT, "at most 128 query heads per KV head");
    if (!dt_ok(c->dtype)) return fail(PC_ERR_FORMAT, "type must be PC_DT_F32, PC_DT_F16 or PC_DT_BF16");
    if (c->head_dim < 8 || c->head_dim > 128 || c->head_dim % 8)
        return fail(PC_ERR_FORMAT, "head_dim must be a multiple of 8, at most 128");
    const int64_t group = c->n_heads / c->n_kv_heads;
    if (c->n_rows * group * group >= (1ll << 32) || c->n_rows * group > (1 << 27) || c->n_requests > (1 << 24))
        return fail(PC_ERR_RANGE, "too many rows or requests");
    if (c->n_rows == 0 || c->n_requests == 0) return PC_OK;
    if (!c->q_dev || !c->out_dev || !c->cu_new_dev) return fail(PC_ERR_INVALID_ARG, "null tensor");
    const int es = dt_size(c->dtype);
    if (!aligned(c->q_dev, c->q_stride, 2, es) || !aligned(c->out_dev, c->out_stride, 2, es))
        return fail(PC_ERR_FORMAT, "q and out need 16-byte aligned pointers and strides");
    return PC_OK;
}

AttnOp op_of(const pc_attn *a, const pc_attn_call *c) {
    AttnOp o;
    memset(&o, 0, sizeof o);
    o.q = c->q_dev;
    o.out = c->out_dev;
    for (int i = 0; i < 2; ++i) {
        o.qs[i] = c->q_stride[i];
        o.os[i] = c->out_stride[i];
    }
    o.cu = c->cu_new_dev;
    o.sinks = c->sinks_dev;
    o.B = c->n_requests;
    o.T = c->n_rows;
    o.H = c->n_heads;
    o.KVH = c->n_kv_heads;
    o.G = c->n_heads / c->n_kv_heads;
    o.D = c->head_dim;
    o.inv_g = (unsigned)(((1ull << 32) + o.G - 1) / o.G);
    o.window = std::min(c->window, 1 << 30);  // positions are below it; position - window stays in 32 bits
    o.scale = c->scale;
    o.min_q = 1;
    o.max_q = INT_MAX;
    o.part = a->part;
    o.ticket = a->ticket;
    o.err = a->err;
    return o;
}

// f16 and bf16 have two kernels: one for few rows of a request and KV head
// (tokens x query heads of the group), bound by reading K and V, and one for
// many, bound by the products.  Which a request takes goes by its own rows,
// read on the device; over whole prompts only the second is launched.
//
// Up to FEW_ROWS rows, and up to FEW_GROUP where a token alone has that many,
// take the first.  It reads the keys once per 16 rows, the second once per 256.
// 64 requests over 2000 positions, first and second, us: 64-wide heads, 8 a
// group, 16 rows 62 and 127, 32 rows 106 and 127, 48 rows 149 and 127; 128-wide,
// 4 a group, 16 rows 101 and 175, 32 rows 181 and 176; single tokens of 64 heads
// a group 33 and 37, of 128 heads 51 and 37 (128-wide 83 and 53).
//
// The second is launched unless the whole batch has so few rows that one
// request of them all does not need it: the host does not know how the rows are
// shared out (slots without a request have none), and the average says
// nothing about the longest.  The launch costs 1 to 5 us where it finds nothing to
// do (64 single tokens over 500-8000 positions 111 -> 115, 16 over 2000 20 ->
// 21.5); without it 512 rows of one request over 32,768 positions take 263 us
// instead of 79, 1024 tokens of one among 511 slots without a request 169 instead
// of 45.  At 128 rows of one request: over 4096 positions 25 us without, 30 with
// it, over 32,768 79 and 65.
constexpr int FEW_ROWS = 16, FEW_GROUP = 64, FEW_ALONE = 128;

pc_status run_attention(pc_attn *a, const AttnOp &o, int dtype, cudaStream_t st) {
    cudaError_t e = cudaSuccess;
    if (dtype != PC_DT_F32) {
        if (!o.table) {
            if (launch_attn_rows(o, dtype, a->nsm, st, e)) {
                PC_CU(e);
                return PC_OK;
            }
        } else {
            AttnOp few = o, many = o;
            const bool all_few = (int64_t)o.T * o.G <= FEW_ALONE;
            if (!all_few) {
                few.max_q = o.G <= FEW_GROUP ? std::max(o.G, FEW_ROWS) : FEW_ROWS;
                many.min_q = few.max_q + 1;
            }
            if (launch_attn_few(few, dtype, a->nsm, st, e)) {
                if (e == cudaSuccess && !all_few && !launch_attn_rows(many, dtype, a->nsm, st, e))
                    e = launch_attn_simt(many, dtype, a->nsm, st);
                PC_CU(e);
                return PC_OK;
            }
        }
    }
    PC_CU(launch_attn_simt(o, dtype, a->nsm, st));
    return PC_OK;
}

}  // namespace

extern "C" {

pc_status pc_kv_tables(int device, const pc_kv_step *s, void *stream) {
    if (!s || s->n_requests < 0 || s->max_pages < 1 || s->n_tokens < 0 || s->free_cap < 0 || !s->n_free_dev ||
        !s->cu_new_dev || !s->n_free_out_dev || (s->free_cap > 0 && !s->free_pages_dev) ||
        (s->n_requests > 0 &&
         (!s->kv_len_dev || !s->new_len_dev || !s->page_table_dev || !s->kv_end_dev || !s->served_dev)) ||
        (s->n_tokens > 0 && (!s->pos_dev || !s->slot_dev)))
        return fail(PC_ERR_INVALID_ARG, "bad pc_kv_tables arguments");
    if (s->page_size < 8 || s->page_size % 8 || s->page_size > (1 << 16))
        return fail(PC_ERR_FORMAT, "page_size must be a multiple of 8, at most 65536");
    if (s->n_requests > (1 << 20) || s->n_tokens > (1 << 28) || s->free_cap > (1 << 28) ||
        (int64_t)s->max_pages * s->page_size > INT_MAX / 2)
        return fail(PC_ERR_RANGE, "too many requests, tokens, free pages or positions");
    if ((s->n_requests > 0 && s->kv_end_dev == s->kv_len_dev) || s->n_free_out_dev == s->n_free_dev)
        return fail(PC_ERR_INVALID_ARG, "kv_end and n_free_out must not overlap the inputs");
    OnDevice on(device);
    PC_CU(on.e);
    PC_CU(launch_kv_tables(*s, (cudaStream_t)stream));
    return PC_OK;
}

pc_status pc_kv_store(int device, const pc_kv_pages *kv, const void *k_dev, const int64_t *k_stride,
                      const void *v_dev, const int64_t *v_stride, int src_dtype, const int64_t *slot_dev, int n,
                      void *stream) {
    PC_TRY(check_pages(kv));
    if (n < 0) return fail(PC_ERR_INVALID_ARG, "bad pc_kv_store arguments");
    if (!dt_ok(src_dtype)) return fail(PC_ERR_FORMAT, "source type must be PC_DT_F32, PC_DT_F16 or PC_DT_BF16");
    if (n == 0) return PC_OK;
    if (!k_dev || !v_dev || !k_stride || !v_stride || !slot_dev)
        return fail(PC_ERR_INVALID_ARG, "bad pc_kv_store arguments");
    if (!aligned(k_dev, k_stride, 2, dt_size(src_dtype)) || !aligned(v_dev, v_stride, 2, dt_size(src_dtype)))
        return fail(PC_ERR_FORMAT, "k and v need 16-byte aligned pointers and strides");
    OnDevice on(device);
    PC_CU(on.e);
    constexpr int NSM = 148;  // only how small the blocks are cut hangs on it
    PC_CU(launch_kv_store(*kv, k_dev, k_stride, v_dev, v_stride, src_dtype, slot_dev, n, NSM, (cudaStream_t)stream));
    return PC_OK;
}

pc_status pc_attn_create(int device, pc_attn **out) {
    if (!out) return fail(PC_ERR_INVALID_ARG, "bad pc_attn_create arguments");
    OnDevice on(device);
    PC_CU(on.e);
    pc_attn *a = new pc_attn();
    a->dev = device;
    auto done = [&](pc_status s) {
        if (s != PC_OK) pc_attn_free(a);
        else *out = a;
        return s;
    };
    cudaError_t e = cudaDeviceGetAttribute(&a->nsm, cudaDevAttrMultiProcessorCount, device);
    if (e == cudaSuccess) e = attn_simt_configure();
    if (e == cudaSuccess) e = attn_rows_configure();
    if (e == cudaSuccess) e = attn_few_configure();
    const size_t part = std::max({attn_simt_part_floats(a->nsm), attn_rows_part_floats(a->nsm), attn_few_part_floats(a->nsm)});
    if (e == cudaSuccess) e = cudaMalloc(&a->part, part * sizeof(float));
    if (e == cudaSuccess) e = cudaMalloc(&a->ticket, ATTN_MAX_CTAS * sizeof(unsigned));
    if (e == cudaSuccess) e = cudaMalloc(&a->err, sizeof(int));
    if (e == cudaSuccess) e = cudaMemset(a->ticket, 0, ATTN_MAX_CTAS * sizeof(unsigned));
    if (e == cudaSuccess) e = cudaMemset(a->err, 0, sizeof(int));
    if (e == cudaSuccess) e = cudaDeviceSynchronize();
    return done(e == cudaSuccess ? PC_OK : cuda_fail(e, "pc_attn_create"));
}

void pc_attn_free(pc_attn *a) {
    if (!a) return;
    OnDevice on(a->dev);
    cudaDeviceSynchronize();
    cudaFree(a->part);
    cudaFree(a->ticket);
    cudaFree(a->err);
    delete a;
}

pc_status pc_attn_paged(pc_attn *a, const pc_attn_call *c, const pc_kv_pages *kv, const int *page_table_dev,
                        int max_pages, const int *kv_len_dev, void *stream) {
    if (!a) return fail(PC_ERR_INVALID_ARG, "null pc_attn");
    PC_TRY(check_call(c));
    PC_TRY(check_pages(kv));
    if (c->n_rows == 0 || c->n_requests == 0) return PC_OK;
    if (!page_table_dev || !kv_len_dev || max_pages < 1)
        return fail(PC_ERR_INVALID_ARG, "bad pc_attn_paged arguments");
    if (kv->dtype != c->dtype || kv->n_kv_heads != c->n_kv_heads || kv->head_dim != c->head_dim)
        return fail(PC_ERR_FORMAT, "q and the cache differ in type, KV heads or head_dim");
    if ((int64_t)max_pages * kv->page_size > INT_MAX / 2) return fail(PC_ERR_RANGE, "too many positions");
    OnDevice on(a->dev);
    PC_CU(on.e);
    AttnOp o = op_of(a, c);
    o.k = kv->k_dev;
    o.v = kv->v_dev;
    for (int i = 0; i < 3; ++i) {
        o.ks[i] = kv->k_stride[i];
        o.vs[i] = kv->v_stride[i];
    }
    o.table = page_table_dev;
    o.kv_len = kv_len_dev;
    o.max_pages = max_pages;
    o.page_size = kv->page_size;
    o.n_pages = kv->n_pages;
    return run_attention(a, o, c->dtype, (cudaStream_t)stream);
}

pc_status pc_attn_packed(pc_attn *a, const pc_attn_call *c, const void *k_dev, const int64_t *k_stride,
                         const void *v_dev, const int64_t *v_stride, void *stream) {
    if (!a) return fail(PC_ERR_INVALID_ARG, "null pc_attn");
    PC_TRY(check_call(c));
    if (c->n_rows == 0 || c->n_requests == 0) return PC_OK;
    if (!k_dev || !v_dev || !k_stride || !v_stride) return fail(PC_ERR_INVALID_ARG, "null tensor");
    const int es = dt_size(c->dtype);
    if (!aligned(k_dev, k_stride, 2, es) || !aligned(v_dev, v_stride, 2, es))
        return fail(PC_ERR_FORMAT, "k and v need 16-byte aligned pointers and strides");
    OnDevice on(a->dev);
    PC_CU(on.e);
    AttnOp o = op_of(a, c);
    o.k = k_dev;
    o.v = v_dev;
    for (int i = 0; i < 2; ++i) {
        o.ks[i + 1] = k_stride[i];
        o.vs[i + 1] = v_stride[i];
    }
    return run_attention(a, o, c->dtype, (cudaStream_t)stream);
}

pc_status pc_attn_check(pc_attn *a, void *stream) {
    if (!a) return fail(PC_ERR_INVALID_ARG, "null pc_attn");
    OnDevice on(a->dev);
    PC_CU(on.e);
    PC_CU(cudaStreamSynchronize((cudaStream_t)stream));
    int e = 0;
    PC_CU(cudaMemcpy(&e, a->err, sizeof e, cudaMemcpyDeviceToHost));
    if (!e) return PC_OK;
    PC_CU(cudaMemset(a->err, 0, sizeof e));
    PC_CU(cudaMemset(a->ticket, 0, ATTN_MAX_CTAS * sizeof(unsigned)));  // a kernel that gave up leaves them as they were
    PC_CU(cudaDeviceSynchronize());
    return fail(PC_ERR_TIMEOUT, "a bounded wait of an attention kernel gave up");
}

}  // extern "C"
