// attention_simt.cu - attention over pages and packed prompts with fp32
// multiply-adds: every product and sum in fp32, for fp32 tensors (and any
// other type), head sizes up to 128.
//
// A thread block takes the items of its share (attention_plan.cuh).  R rows
// (tokens x query heads of one KV head) meet tiles of 64 keys: scores S = Q
// K^T from shared memory (4 rows x 64/TX keys per thread), the running maximum
// and sum of each row across the TX threads of its row group, then O += P V
// with O in registers (4 rows x HDP/TX columns per thread).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "attention_plan.cuh"
#include "launch.cuh"

namespace pc {

namespace {

constexpr int SIMT_KT = 64, SIMT_OV = 32;

template <int HDP, int R>
struct SimtCfg {
    static constexpr int TX = R == 64 ? 16 : 32;  // threads per group of 4 rows
    static constexpr int THREADS = R / 4 * TX;
    static constexpr int KPT = SIMT_KT / TX;      // keys per thread
    static constexpr int DPT = HDP / TX;          // output columns per thread
    static constexpr int LDK = HDP + 4, LDP = R + 4;
    static constexpr size_t SMEM = sizeof(float) * (R * HDP + SIMT_KT * LDK + SIMT_KT * HDP + SIMT_KT * LDP);
    static constexpr int PART = R * (HDP + 2);    // floats of one partial record: O, m, l
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f(float &d, float v) { d = v; }
__device__ __forceinline__ void from_f(__half &d, float v) { d = __float2half_rn(v); }
__device__ __forceinline__ void from_f(__nv_bfloat16 &d, float v) { d = __float2bfloat16_rn(v); }

// 16 bytes of a row as floats
template <typename T>
__device__ __forceinline__ void load16(const T *p, float (&f)[16 / sizeof(T)]) {
    const uint4 r = *reinterpret_cast<const uint4 *>(p);
    const T *t = reinterpret_cast<const T *>(&r);
#pragma unroll
    for (int i = 0; i < (int)(16 / sizeof(T)); ++i) f[i] = to_f(t[i]);
}

// Where position j of request b has its K or V row; null if its page is not one of the cache's.
template <typename T>
__device__ __forceinline__ const T *kv_row(const AttnOp &a, const void *base, const int64_t (&s)[3], int b, int q0,
                                           int kvh, int j) {
    const T *p = reinterpret_cast<const T *>(base) + kvh * s[2];
    if (!a.table) return p + (int64_t)(q0 + j) * s[1];
    const int page = a.table[(int64_t)b * a.max_pages + j / a.page_size];
    if (page < 0 || page >= a.n_pages) return nullptr;
    return p + page * s[0] + (int64_t)(j % a.page_size) * s[1];
}

template <typename T, int HDP, int R>
__global__ void __launch_bounds__(SimtCfg<HDP, R>::THREADS) attn_simt_kernel(const AttnOp a) {
    using C = SimtCfg<HDP, R>;
    constexpr int TX = C::TX, KPT = C::KPT, DPT = C::DPT, KT = SIMT_KT, VEC = 16 / sizeof(T);
    extern __shared__ __align__(16) float simt_smem[];
    float *Qs = simt_smem, *Ks = Qs + R * HDP, *Vs = Ks + KT * C::LDK, *Pt = Vs + KT * HDP;
    __shared__ PlanScratch<C::THREADS> sc;
    __shared__ int lastf;
    pdl_wait();
    pdl_trigger();
    plan_share<R, KT, SIMT_OV, 2 * KT, C::THREADS>(a, blockIdx.x, gridDim.x, sc);
    if (sc.share.n == 0) return;
    const int tid = threadIdx.x, tx = tid % TX, ty = tid / TX;
    PlanWalk<R, KT> w(a, sc.share);
    for (bool more = w.load(); more; more = w.next()) {
        const ItemGeo g = w.g;
        // Q, scaled; rows past the item and columns past head_dim are zeros
        __syncthreads();
        for (int c = tid; c < R * (HDP / VEC); c += C::THREADS) {
            const int r = c / (HDP / VEC), d = (c % (HDP / VEC)) * VEC, f = g.r0 + r;
            float x[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) x[i] = 0.0f;
            if (f < g.r1 && d < a.D)
                load16(reinterpret_cast<const T *>(a.q) + (int64_t)(w.s.q0 + f / a.G) * a.qs[0] +
                           (int64_t)(w.kvh * a.G + f % a.G) * a.qs[1] + d, x);
#pragma unroll
            for (int i = 0; i < VEC; ++i) Qs[r * HDP + d + i] = __fmul_rn(x[i], a.scale);
        }
        int pos[4];  // this thread's rows: 4 ty .. 4 ty + 3
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int f = g.r0 + 4 * ty + i;
            pos[i] = f < g.r1 ? w.s.p0 + f / a.G : -1;
        }
        float m[4], l[4], o[4][DPT];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            m[i] = -INFINITY;
            l[i] = 0.0f;
#pragma unroll
            for (int d = 0; d < DPT; ++d) o[i][d] = 0.0f;
        }
        for (int t = w.tl; t < w.th; ++t) {
            const int k0 = (g.t0 + t) * KT;
            __syncthreads();
            int odd = 0;  // a V element that is not finite
            for (int c = tid; c < KT * (HDP / VEC); c += C::THREADS) {
                const int r = c / (HDP / VEC), d = (c % (HDP / VEC)) * VEC, j = k0 + r;
                float x[VEC], y[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) x[i] = y[i] = 0.0f;
                if (j >= g.kb && j < g.ke && d < a.D) {
                    const T *kp = kv_row<T>(a, a.k, a.ks, w.b, w.s.q0, w.kvh, j);
                    const T *vp = kv_row<T>(a, a.v, a.vs, w.b, w.s.q0, w.kvh, j);
                    if (kp) {
                        load16(kp + d, x);
                        load16(vp + d, y);
                    }
                }
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    Ks[r * C::LDK + d + i] = x[i];
                    Vs[r * HDP + d + i] = y[i];
                    odd |= !isfinite(y[i]);
                }
            }
            odd = __syncthreads_or(odd);
            float s[4][KPT];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < KPT; ++j) s[i][j] = 0.0f;
#pragma unroll 4
            for (int d = 0; d < HDP; d += 4) {
                float4 q4[4], k4[KPT];
#pragma unroll
                for (int i = 0; i < 4; ++i) q4[i] = *reinterpret_cast<const float4 *>(Qs + (4 * ty + i) * HDP + d);
#pragma unroll
                for (int j = 0; j < KPT; ++j)
                    k4[j] = *reinterpret_cast<const float4 *>(Ks + (tx + TX * j) * C::LDK + d);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < KPT; ++j) {
                        s[i][j] = __fmaf_rn(q4[i].x, k4[j].x, s[i][j]);
                        s[i][j] = __fmaf_rn(q4[i].y, k4[j].y, s[i][j]);
                        s[i][j] = __fmaf_rn(q4[i].z, k4[j].z, s[i][j]);
                        s[i][j] = __fmaf_rn(q4[i].w, k4[j].w, s[i][j]);
                    }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int lo = a.window > 0 ? pos[i] - a.window : -1;
                float top = -INFINITY;
#pragma unroll
                for (int j = 0; j < KPT; ++j) {
                    const int key = k0 + tx + TX * j;
                    if (key > pos[i] || key <= lo) s[i][j] = -INFINITY;
                    top = fmaxf(top, s[i][j]);
                }
#pragma unroll
                for (int x = TX / 2; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                const float mn = fmaxf(m[i], top), ms = mn == -INFINITY ? 0.0f : mn;
                const float corr = expf(__fsub_rn(m[i], ms));
                float sum = 0.0f;
#pragma unroll
                for (int j = 0; j < KPT; ++j) {
                    const float p = expf(__fsub_rn(s[i][j], ms));
                    Pt[(tx + TX * j) * C::LDP + 4 * ty + i] = p;
                    sum = __fadd_rn(sum, p);
                }
#pragma unroll
                for (int x = TX / 2; x; x >>= 1) sum = __fadd_rn(sum, __shfl_xor_sync(0xffffffffu, sum, x));
                l[i] = __fmaf_rn(l[i], corr, sum);
                m[i] = mn;
#pragma unroll
                for (int d = 0; d < DPT; ++d) o[i][d] = __fmul_rn(o[i][d], corr);
            }
            __syncthreads();
            if (!odd) {
#pragma unroll 4
                for (int j = 0; j < KT; ++j) {
                    const float4 p4 = *reinterpret_cast<const float4 *>(Pt + j * C::LDP + 4 * ty);
                    const float p[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
                    for (int d = 0; d < DPT; ++d) {
                        const float v = Vs[j * HDP + tx + TX * d];
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[i][d] = __fmaf_rn(p[i], v, o[i][d]);
                    }
                }
            } else {  // 0 x inf: a key meets only the rows that see it
                for (int j = 0; j < KT; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = k0 + j;
                        if (key > pos[i] || (a.window > 0 && key <= pos[i] - a.window)) continue;
                        const float p = Pt[j * C::LDP + 4 * ty + i];
#pragma unroll
                        for (int d = 0; d < DPT; ++d) o[i][d] = __fmaf_rn(p, Vs[j * HDP + tx + TX * d], o[i][d]);
                    }
            }
        }
        if (!w.whole()) {
            const CutItem c = cut_item(w);
            float *mine = a.part + ((int64_t)blockIdx.x * 2 + (w.tl == 0)) * C::PART;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 4 * ty + i;
#pragma unroll
                for (int d = 0; d < DPT; ++d) mine[r * HDP + tx + TX * d] = o[i][d];
                if (tx == 0) {
                    mine[R * HDP + r] = m[i];
                    mine[R * HDP + R + r] = l[i];
                }
            }
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                lastf = atomicAdd(a.ticket + c.k0, 1u) == (unsigned)(c.k1 - c.k0);
                if (lastf) a.ticket[c.k0] = 0u;
            }
            __syncthreads();
            if (!lastf) continue;
            __threadfence();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 4 * ty + i;
                float mm = -INFINITY, ll = 0.0f, oo[DPT];
                for (int k = c.k0; k <= c.k1; ++k)
                    mm = fmaxf(mm, __ldcg(a.part + ((int64_t)k * 2 + (k == c.k0)) * C::PART + R * HDP + r));
                const float ms = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
                for (int d = 0; d < DPT; ++d) oo[d] = 0.0f;
                for (int k = c.k0; k <= c.k1; ++k) {
                    const float *p = a.part + ((int64_t)k * 2 + (k == c.k0)) * C::PART;
                    const float f = expf(__fsub_rn(__ldcg(p + R * HDP + r), ms));
                    ll = __fmaf_rn(__ldcg(p + R * HDP + R + r), f, ll);
#pragma unroll
                    for (int d = 0; d < DPT; ++d) oo[d] = __fmaf_rn(__ldcg(p + r * HDP + tx + TX * d), f, oo[d]);
                }
                m[i] = mm;
                l[i] = ll;
#pragma unroll
                for (int d = 0; d < DPT; ++d) o[i][d] = oo[d];
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int f = g.r0 + 4 * ty + i;
            if (f >= g.r1) continue;
            const int h = w.kvh * a.G + f % a.G;
            const bool none = m[i] == -INFINITY && l[i] == 0.0f;  // no key seen
            float corr = 1.0f, total = l[i];
            if (a.sinks) {
                const float sk = a.sinks[h], mm = fmaxf(m[i], sk);
                corr = m[i] == -INFINITY ? 0.0f : expf(__fsub_rn(m[i], mm));
                total = __fmaf_rn(l[i], corr, expf(__fsub_rn(sk, mm)));
            }
            const float inv = none ? 0.0f : __fdiv_rn(corr, total);
            T *out = reinterpret_cast<T *>(a.out) + (int64_t)(w.s.q0 + f / a.G) * a.os[0] + (int64_t)h * a.os[1];
#pragma unroll
            for (int d = 0; d < DPT; ++d)
                if (tx + TX * d < a.D) from_f(out[tx + TX * d], none ? 0.0f : __fmul_rn(o[i][d], inv));
        }
    }
}

template <typename T, int HDP, int R>
cudaError_t simt_set() {
    return cudaFuncSetAttribute(attn_simt_kernel<T, HDP, R>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)SimtCfg<HDP, R>::SMEM);
}

template <typename T, int HDP, int R>
cudaError_t simt_run(const AttnOp &a, int nsm, cudaStream_t st) {
    const int per = R == 64 ? (HDP == 64 ? 3 : 2) : (HDP == 64 ? 5 : 3);  // blocks that fit an SM
    return launch_k(attn_simt_kernel<T, HDP, R>, dim3(nsm * per), dim3(SimtCfg<HDP, R>::THREADS),
                    SimtCfg<HDP, R>::SMEM, st, a);
}

template <typename T>
cudaError_t simt_pick(const AttnOp &a, int nsm, cudaStream_t st) {
    const bool few = (int64_t)a.T * a.G <= (int64_t)16 * a.B;
    if (a.D <= 64) return few ? simt_run<T, 64, 16>(a, nsm, st) : simt_run<T, 64, 64>(a, nsm, st);
    return few ? simt_run<T, 128, 16>(a, nsm, st) : simt_run<T, 128, 64>(a, nsm, st);
}

template <typename T>
cudaError_t simt_set_all() {
    cudaError_t e = simt_set<T, 64, 16>();
    if (e == cudaSuccess) e = simt_set<T, 64, 64>();
    if (e == cudaSuccess) e = simt_set<T, 128, 16>();
    if (e == cudaSuccess) e = simt_set<T, 128, 64>();
    return e;
}

}  // namespace

size_t attn_simt_part_floats(int nsm) {
    return (size_t)nsm * 2 * 3 * SimtCfg<128, 64>::PART;
}

cudaError_t attn_simt_configure() {
    cudaError_t e = simt_set_all<float>();
    if (e == cudaSuccess) e = simt_set_all<__half>();
    if (e == cudaSuccess) e = simt_set_all<__nv_bfloat16>();
    return e;
}

cudaError_t launch_attn_simt(const AttnOp &a, int dtype, int nsm, cudaStream_t st) {
    if (dtype == PC_DT_F32) return simt_pick<float>(a, nsm, st);
    if (dtype == PC_DT_F16) return simt_pick<__half>(a, nsm, st);
    return simt_pick<__nv_bfloat16>(a, nsm, st);
}

}  // namespace pc
