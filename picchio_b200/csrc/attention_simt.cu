// attention_simt.cu - attention over pages and packed prompts with fp32
// multiply-adds: every product and sum in fp32, for fp32 tensors (and f16 and
// bf16 ones whose strides no tensor map describes), head sizes up to 128.
//
// A thread block takes the items of its share (attention_plan.cuh).  R rows
// (tokens x query heads of one KV head; 16, 32 or 64 of them, see simt_rows)
// meet tiles of 64 keys: scores S = Q K^T from shared
// memory (4 rows x 64/TX keys per thread: 8 16-byte loads for 64
// multiply-adds), the running maximum and sum of each row across the TX
// threads of its row group, then O += P V with O in registers (4 rows x HDP/TX
// columns per thread).  The next tile is copied (cp.async) while one is
// worked on.  Bound by the multiply-adds (128 a cycle and SM) and, at few
// rows, by the waits of a tile's steps for one another.  Measured, fp32, 64
// query over 8 KV heads of 64: prompts of 154, 259 and 287 tokens 80 us (the
// multiply-adds alone 19 us, 25 with the masked ones), three tokens each of 15
// requests of 173-1430 positions 47 us.  What an item costs beside its keys counts
// as 48 of them in the shares (24, 96, 160: the prompts 85, 83, 87 us, 64 single
// tokens to 2000 174, 166, 167 where it is 161; four chunks of 500 over 1500 within
// 1 %, the three tokens alike).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "attention_plan.cuh"
#include "launch.cuh"
#include "sm100.cuh"

namespace pc {

namespace {

constexpr int SIMT_KT = 64, SIMT_OV = 48;

template <int HDP, int R>
struct SimtCfg {
    static constexpr int TX = R == 16 ? 32 : 16;  // threads per group of 4 rows
    static constexpr int THREADS = R / 4 * TX;
    static constexpr int KPT = SIMT_KT / TX;      // keys per thread
    static constexpr int DPT = HDP / TX;          // output columns per thread: CV at a time, CV * TX apart
    static constexpr int CV = DPT < 4 ? DPT : 4;
    // O goes to memory four columns at a time (short prompts 81.6 -> 80.0 us); with fewer rows it does not pay (three
    // tokens of 15 requests: 47.8 us instead of 46.3)
    static constexpr bool WIDE = R == 64;
    static constexpr int LDK = HDP + 4, LDP = R + 4;
    static constexpr int STAGE = SIMT_KT * (LDK + HDP);  // floats of a K and a V tile
    static constexpr size_t SMEM = sizeof(float) * (R * HDP + 2 * STAGE + SIMT_KT * LDP);
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

// Four consecutive elements, aligned as such
template <typename T>
__device__ __forceinline__ void store4(T *p, float a, float b, float c, float d) {
    struct alignas(4 * sizeof(T)) {
        T t[4];
    } x;
    from_f(x.t[0], a);
    from_f(x.t[1], b);
    from_f(x.t[2], c);
    from_f(x.t[3], d);
    if constexpr (sizeof x == 16) *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<uint4 *>(&x);
    else *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<uint2 *>(&x);
}

__device__ __forceinline__ void copy16(void *dst, const void *src, int bytes) {  // zeros past `bytes`
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}

// Where position j of request b has its K and V rows; null if its page is not one of the cache's.
template <typename T>
__device__ __forceinline__ void kv_rows(const AttnOp &a, int b, int q0, int kvh, int j, const T *&kp, const T *&vp) {
    int64_t page = 0, row = q0 + j;
    if (a.table) {
        const unsigned pg = (unsigned)j / (unsigned)a.page_size;
        page = a.table[(int64_t)b * a.max_pages + pg];
        row = j - (int)pg * a.page_size;
        if (page < 0 || page >= a.n_pages) return;
    }
    kp = reinterpret_cast<const T *>(a.k) + page * a.ks[0] + row * a.ks[1] + kvh * a.ks[2];
    vp = reinterpret_cast<const T *>(a.v) + page * a.vs[0] + row * a.vs[1] + kvh * a.vs[2];
}

template <typename T, int HDP, int R>
__global__ void __launch_bounds__(SimtCfg<HDP, R>::THREADS) attn_simt_kernel(const AttnOp a) {
    using C = SimtCfg<HDP, R>;
    constexpr int TX = C::TX, KPT = C::KPT, DPT = C::DPT, KT = SIMT_KT, VEC = 16 / sizeof(T);
    extern __shared__ __align__(16) float simt_smem[];
    float *Qs = simt_smem, *ring = Qs + R * HDP, *Pt = ring + 2 * C::STAGE;
    __shared__ PlanScratch<C::THREADS> sc;
    __shared__ int lastf;
    if (a.min_q > 1 && nothing_to_take(a.cu, a.B, a.T, a.G, a.min_q, a.max_q)) {
        pdl_trigger();
        pdl_wait();
        return;
    }
    pdl_wait();
    pdl_trigger();
    plan_share<R, KT, SIMT_OV, 2 * KT, C::THREADS>(a, blockIdx.x, gridDim.x, sc);
    if (sc.share.n == 0) return;
    const int tid = threadIdx.x, tx = tid % TX, ty = tid / TX;
    auto col = [&](int d) { return d / C::CV * (C::CV * TX) + tx * C::CV + d % C::CV; };  // of o[.][d]
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
                load16(reinterpret_cast<const T *>(a.q) + (int64_t)(w.s.q0 + div_g(a, f)) * a.qs[0] +
                           (int64_t)(w.kvh * a.G + f - div_g(a, f) * a.G) * a.qs[1] + d, x);
#pragma unroll
            for (int i = 0; i < VEC; ++i) Qs[r * HDP + d + i] = __fmul_rn(x[i], a.scale);
        }
        int pos[4];  // this thread's rows: 4 ty .. 4 ty + 3
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int f = g.r0 + 4 * ty + i;
            pos[i] = f < g.r1 ? w.s.p0 + div_g(a, f) : -1;
        }
        float m[4], l[4], o[4][DPT];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            m[i] = -INFINITY;
            l[i] = 0.0f;
#pragma unroll
            for (int d = 0; d < DPT; ++d) o[i][d] = 0.0f;
        }
        // K and V rows of tile t into stage t % 2, zeros outside the item's keys
        auto copy = [&](int t) {
            const int k0 = (g.t0 + t) * KT;
            float *Ks = ring + (t & 1) * C::STAGE, *Vs = Ks + KT * C::LDK;
            for (int c = tid; c < KT * (HDP / VEC); c += C::THREADS) {
                const int r = c / (HDP / VEC), d = (c % (HDP / VEC)) * VEC, j = k0 + r;
                const T *kp = nullptr, *vp = nullptr;
                if (j >= g.kb && j < g.ke && d < a.D) kv_rows<T>(a, w.b, w.s.q0, w.kvh, j, kp, vp);
                if constexpr (sizeof(T) == 4) {
                    copy16(Ks + r * C::LDK + d, kp ? kp + d : reinterpret_cast<const T *>(a.q), kp ? 16 : 0);
                    copy16(Vs + r * HDP + d, vp ? vp + d : reinterpret_cast<const T *>(a.q), vp ? 16 : 0);
                } else {
                    float x[VEC], y[VEC];
#pragma unroll
                    for (int i = 0; i < VEC; ++i) x[i] = y[i] = 0.0f;
                    if (kp) {
                        load16(kp + d, x);
                        load16(vp + d, y);
                    }
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        Ks[r * C::LDK + d + i] = x[i];
                        Vs[r * HDP + d + i] = y[i];
                    }
                }
            }
            cp_async_commit();
        };
        copy(w.tl);
        for (int t = w.tl; t < w.th; ++t) {
            const int k0 = (g.t0 + t) * KT;
            float *Ks = ring + (t & 1) * C::STAGE, *Vs = Ks + KT * C::LDK;
            if (t + 1 < w.th) {
                copy(t + 1);
                cp_async_wait<1>();
            } else {
                cp_async_wait<0>();
            }
            __syncthreads();
            // in a tile that some row does not see whole: is there a V element that is not finite
            int odd = 0;
            if (k0 + KT - 1 > g.pmin || (a.window > 0 && k0 < g.pmax - a.window + 1)) {
                for (int c = tid; c < KT * HDP; c += C::THREADS) odd |= !isfinite(Vs[c]);
                odd = __syncthreads_or(odd);
            }
            // two multiply-adds an instruction: even and odd dimensions apart
            uint64_t s2[4][KPT];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < KPT; ++j) s2[i][j] = 0;
#pragma unroll 4
            for (int d = 0; d < HDP; d += 4) {
                ulonglong2 q4[4], k4[KPT];
#pragma unroll
                for (int i = 0; i < 4; ++i) q4[i] = *reinterpret_cast<const ulonglong2 *>(Qs + (4 * ty + i) * HDP + d);
#pragma unroll
                for (int j = 0; j < KPT; ++j)
                    k4[j] = *reinterpret_cast<const ulonglong2 *>(Ks + (tx + TX * j) * C::LDK + d);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < KPT; ++j) {
                        s2[i][j] = f2_fma(q4[i].x, k4[j].x, s2[i][j]);
                        s2[i][j] = f2_fma(q4[i].y, k4[j].y, s2[i][j]);
                    }
            }
            float s[4][KPT];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < KPT; ++j) s[i][j] = __fadd_rn(f2_lo(s2[i][j]), f2_hi(s2[i][j]));
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
                uint64_t o2[4][DPT / 2];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int d = 0; d < DPT; d += 2) o2[i][d / 2] = f2_pack(o[i][d], o[i][d + 1]);
#pragma unroll 4
                for (int j = 0; j < KT; ++j) {
                    const float4 p4 = *reinterpret_cast<const float4 *>(Pt + j * C::LDP + 4 * ty);
                    const uint64_t p[4] = {f2_pack(p4.x, p4.x), f2_pack(p4.y, p4.y), f2_pack(p4.z, p4.z),
                                           f2_pack(p4.w, p4.w)};
#pragma unroll
                    for (int d = 0; d < DPT; d += C::CV) {
                        uint64_t v[C::CV / 2];
                        const float *vr = Vs + j * HDP + col(d);
                        if constexpr (C::CV == 4) {
                            const ulonglong2 x = *reinterpret_cast<const ulonglong2 *>(vr);
                            v[0] = x.x, v[1] = x.y;
                        } else {
                            v[0] = *reinterpret_cast<const uint64_t *>(vr);
                        }
#pragma unroll
                        for (int e = 0; e < C::CV / 2; ++e)
#pragma unroll
                            for (int i = 0; i < 4; ++i) o2[i][d / 2 + e] = f2_fma(p[i], v[e], o2[i][d / 2 + e]);
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int d = 0; d < DPT; d += 2) {
                        o[i][d] = f2_lo(o2[i][d / 2]);
                        o[i][d + 1] = f2_hi(o2[i][d / 2]);
                    }
            } else {  // 0 x inf: a key meets only the rows that see it
                for (int j = 0; j < KT; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = k0 + j;
                        if (key > pos[i] || (a.window > 0 && key <= pos[i] - a.window)) continue;
                        const float p = Pt[j * C::LDP + 4 * ty + i];
#pragma unroll
                        for (int d = 0; d < DPT; ++d) o[i][d] = __fmaf_rn(p, Vs[j * HDP + col(d)], o[i][d]);
                    }
            }
            __syncthreads();  // the stage and P may be written again
        }
        if (!w.whole()) {
            const CutItem c = cut_item(w);
            float *mine = a.part + ((int64_t)blockIdx.x * 2 + (w.tl == 0)) * C::PART;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 4 * ty + i;
                if constexpr (C::WIDE) {
#pragma unroll
                    for (int d = 0; d < DPT; d += 4)
                        store4(mine + r * HDP + col(d), o[i][d], o[i][d + 1], o[i][d + 2], o[i][d + 3]);
                } else {
#pragma unroll
                    for (int d = 0; d < DPT; ++d) mine[r * HDP + col(d)] = o[i][d];
                }
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
            // the parts in block order; a part's loads for all four rows go together
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                m[i] = -INFINITY;
                l[i] = 0.0f;
#pragma unroll
                for (int d = 0; d < DPT; ++d) o[i][d] = 0.0f;
            }
#pragma unroll 2
            for (int k = c.k0; k <= c.k1; ++k) {
                const float *p = a.part + ((int64_t)k * 2 + (k == c.k0)) * C::PART;
                float pm[4], pl[4], po[4][DPT];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = 4 * ty + i;
                    pm[i] = __ldcg(p + R * HDP + r);
                    pl[i] = __ldcg(p + R * HDP + R + r);
                    if constexpr (C::WIDE) {
#pragma unroll
                        for (int d = 0; d < DPT; d += 4) {
                            const float4 x = __ldcg(reinterpret_cast<const float4 *>(p + r * HDP + col(d)));
                            po[i][d] = x.x;
                            po[i][d + 1] = x.y;
                            po[i][d + 2] = x.z;
                            po[i][d + 3] = x.w;
                        }
                    } else {
#pragma unroll
                        for (int d = 0; d < DPT; ++d) po[i][d] = __ldcg(p + r * HDP + col(d));
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float mn = fmaxf(m[i], pm[i]), ms = mn == -INFINITY ? 0.0f : mn;
                    const float old = expf(__fsub_rn(m[i], ms)), e = expf(__fsub_rn(pm[i], ms));
                    m[i] = mn;
                    l[i] = __fmaf_rn(pl[i], e, __fmul_rn(l[i], old));
#pragma unroll
                    for (int d = 0; d < DPT; ++d) o[i][d] = __fmaf_rn(po[i][d], e, __fmul_rn(o[i][d], old));
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int f = g.r0 + 4 * ty + i;
            if (f >= g.r1) continue;
            const int tok = div_g(a, f), h = w.kvh * a.G + f - tok * a.G;
            const bool none = m[i] == -INFINITY && l[i] == 0.0f;  // no key seen
            float corr = 1.0f, total = l[i];
            if (a.sinks) {
                const float sk = a.sinks[h], mm = fmaxf(m[i], sk);
                corr = m[i] == -INFINITY ? 0.0f : expf(__fsub_rn(m[i], mm));
                total = __fmaf_rn(l[i], corr, expf(__fsub_rn(sk, mm)));
            }
            const float inv = none ? 0.0f : __fdiv_rn(corr, total);
            T *out = reinterpret_cast<T *>(a.out) + (int64_t)(w.s.q0 + tok) * a.os[0] + (int64_t)h * a.os[1];
            auto value = [&](int d) -> float { return none ? 0.0f : __fmul_rn(o[i][d], inv); };
            if constexpr (C::WIDE) {
#pragma unroll
                for (int d = 0; d < DPT; d += 4)
                    if (col(d) < a.D) store4(out + col(d), value(d), value(d + 1), value(d + 2), value(d + 3));
            } else {
#pragma unroll
                for (int d = 0; d < DPT; ++d)
                    if (col(d) < a.D) from_f(out[col(d)], value(d));
            }
        }
    }
}

template <typename T, int HDP, int R>
cudaError_t simt_set() {
    return cudaFuncSetAttribute(attn_simt_kernel<T, HDP, R>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)SimtCfg<HDP, R>::SMEM);
}

// Blocks that fit an SM (shared memory, registers)
template <int HDP, int R>
constexpr int simt_per_sm() {
    return (int)std::min<size_t>(R == 64 ? 2 : 4, 227 * 1024 / (SimtCfg<HDP, R>::SMEM + 2048));
}

template <typename T, int HDP, int R>
cudaError_t simt_run(const AttnOp &a, int nsm, cudaStream_t st) {
    return launch_k(attn_simt_kernel<T, HDP, R>, dim3(nsm * simt_per_sm<HDP, R>()), dim3(SimtCfg<HDP, R>::THREADS),
                    SimtCfg<HDP, R>::SMEM, st, a);
}

// The least rows an item that hold the batch's rows a request (and KV head) on
// average: at fewer rows the products of rows that do not exist cost most (64
// single tokens over 1000 positions, 8 query heads a group: 16 rows 156 us, 32
// 205, 64 288).  Requests of more than 32 rows have a launch of their own with 64
// (the average says nothing about the longest: 1024 tokens of one among 511 slots
// without a request 620 us with 16 rows, 322 with this), unless there are so few
// rows in all that one request of them all can do without (over 4096 positions,
// 64- and 128-wide heads: 64 rows by 16 48 and 104 us, by 64 49 and 63; 512 rows
// by 32 200 and 477, by 64 152 and 324).  The launch costs 1 to 3 us where it
// finds nothing to do (three tokens of 15 requests 47 -> 50).
constexpr int SIMT_FEW = 32, SIMT_ALONE16 = 64, SIMT_ALONE32 = 512;

template <typename T, int HDP>
cudaError_t simt_rows(const AttnOp &a, int nsm, cudaStream_t st) {
    const int64_t rows = (int64_t)a.T * a.G;
    if (rows > (int64_t)SIMT_FEW * a.B) return simt_run<T, HDP, 64>(a, nsm, st);
    const bool r16 = rows <= (int64_t)16 * a.B, alone = rows <= (r16 ? SIMT_ALONE16 : SIMT_ALONE32);
    AttnOp few = a, many = a;
    if (!alone) {
        few.max_q = std::min(a.max_q, SIMT_FEW);
        many.min_q = std::max(a.min_q, SIMT_FEW + 1);
    }
    const cudaError_t e = r16 ? simt_run<T, HDP, 16>(few, nsm, st) : simt_run<T, HDP, 32>(few, nsm, st);
    return e == cudaSuccess && !alone ? simt_run<T, HDP, 64>(many, nsm, st) : e;
}

template <typename T>
cudaError_t simt_pick(const AttnOp &a, int nsm, cudaStream_t st) {
    return a.D <= 64 ? simt_rows<T, 64>(a, nsm, st) : simt_rows<T, 128>(a, nsm, st);
}

template <typename T>
cudaError_t simt_set_all() {
    cudaError_t e = simt_set<T, 64, 16>();
    if (e == cudaSuccess) e = simt_set<T, 64, 32>();
    if (e == cudaSuccess) e = simt_set<T, 64, 64>();
    if (e == cudaSuccess) e = simt_set<T, 128, 16>();
    if (e == cudaSuccess) e = simt_set<T, 128, 32>();
    if (e == cudaSuccess) e = simt_set<T, 128, 64>();
    return e;
}

}  // namespace

size_t attn_simt_part_floats(int nsm) {
    return (size_t)nsm * 2 * 4 * SimtCfg<128, 64>::PART;
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
