// paged.h - launch interface of the paged KV cache operators (tables, store,
// attention over pages and over packed prompts).
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/picchio_b200.h"

namespace pc {

// One attention call as its kernels see it.  K and V element (page or 0,
// position or row, KV head, i) sits at page * s[0] + position * s[1] + head *
// s[2] + i; packed prompts have table == nullptr and s[0] unused.
struct AttnOp {
    const void *q, *k, *v;
    void *out;
    int64_t qs[2], os[2], ks[3], vs[3];
    const int *cu, *kv_len, *table;  // kv_len, table: paged only
    const float *sinks;
    int max_pages, page_size, n_pages;
    int B, T, H, KVH, G, D, window;
    float scale;
    unsigned inv_g;        // 2^32 / G rounded up (G > 1)
    int min_q, max_q;      // the kernel takes requests with min_q <= rows * G <= max_q
    float *part;           // partial (O, m, l) of items cut between CTAs, two slots per CTA
    unsigned *ticket;      // one per CTA, zero between calls
    int *err;
};

constexpr int ATTN_MAX_CTAS = 148 * 8;

// Workspace floats that the kernel needs for `nsm` SMs.
size_t attn_simt_part_floats(int nsm);
cudaError_t attn_simt_configure();
cudaError_t launch_attn_simt(const AttnOp &a, int dtype, int nsm, cudaStream_t st);

// f16 and bf16 on the tensor cores; false (nothing launched) if K or V has
// strides that no tensor map describes.
size_t attn_rows_part_floats(int nsm);
cudaError_t attn_rows_configure();
bool launch_attn_rows(const AttnOp &a, int dtype, int nsm, cudaStream_t st, cudaError_t &e);

// The same for few rows a request.
size_t attn_few_part_floats(int nsm);
cudaError_t attn_few_configure();
bool launch_attn_few(const AttnOp &a, int dtype, int nsm, cudaStream_t st, cudaError_t &e);

cudaError_t launch_kv_tables(const pc_kv_step &s, cudaStream_t st);
cudaError_t launch_kv_store(const pc_kv_pages &kv, const void *k, const int64_t *ks, const void *v, const int64_t *vs,
                            int src_dtype, const int64_t *slot, int n, int nsm, cudaStream_t st);

}  // namespace pc
