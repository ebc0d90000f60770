// attention_few.cu - attention of few rows a request (single tokens, a few
// guessed ones) over pages, for f16 and bf16 tensors: bound by reading K and
// V once.
//
// A thread block (two per SM) takes the items of its share
// (attention_plan.cuh): up to 16 rows (tokens x query heads of one KV head)
// against all their keys, in tiles of 16 KB of K and V (64 keys at head sizes
// to 64, 32 at 128).  Warp 4 fetches the tiles by TMA into a ring, across
// items, so the memory system does not see where one ends; warps 0-3 take the
// tiles in turn, each with its own running maximum, sum and O in registers:
// S = Q K^T and O += P V as mma.sync m16n8k16 (16 rows are all there are: the
// products are far below the legacy path's rate while the tiles arrive).  At
// the end of an item the four warps' parts are joined in shared memory, and
// those of several blocks (a row cut between shares) in the workspace.
#include <algorithm>

#include "attention_half.cuh"
#include "launch.cuh"

namespace pc {

namespace {

constexpr int FW_R = 16, FW_WARPS = 4, FW_THREADS = (FW_WARPS + 1) * 32, FW_OV = 128, FW_MINK = 256;
constexpr int FW_PER_SM = 2;

template <int HD>
struct FewCfg {
    static constexpr int KT = 4096 / HD, PANELS = HD / 64;
    // a multiple of the warps: a stage is always the same warp's, which so sees
    // every phase of its barrier (one that skips phases takes an older one of
    // the same parity for its own)
    static constexpr int STAGES = FW_WARPS;
    static constexpr int PANEL = KT * 128, TILE = PANELS * PANEL;  // 8 KB of K, and of V
    static constexpr int LDR = HD + 4;                             // floats of a row of a warp's record
    static constexpr int REC = FW_R * LDR;
    static constexpr size_t SMEM = 1024 + (size_t)STAGES * 2 * TILE + FW_WARPS * REC * 4;
    static constexpr int PART = FW_R * (HD + 2);  // floats of a block's record: O, m, l
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

template <typename T>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (Half16<T>::FMT)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T, int HD>
__global__ void __launch_bounds__(FW_THREADS, FW_PER_SM)
    attn_few_kernel(const AttnOp a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                    const int box) {
    using C = FewCfg<HD>;
    using E = Half16<T>;
    constexpr int KT = C::KT, NS = C::STAGES;
    extern __shared__ uint8_t few_smem_raw[];
    uint8_t *ring = few_smem_raw + (1024 - (smem_u32(few_smem_raw) & 1023)) % 1024;
    float *recs = reinterpret_cast<float *>(ring + NS * 2 * C::TILE);
    __shared__ PlanScratch<FW_THREADS> sc;
    __shared__ uint64_t full[NS], free_[NS], meet_bar;
    __shared__ volatile int dead;
    __shared__ int lastf;
    __shared__ float wm[FW_WARPS][FW_R], wl[FW_WARPS][FW_R];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < NS; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&free_[s], 1);
        }
        mbar_init(&meet_bar, FW_WARPS);
        fence_mbar_init();
        dead = 0;
    }
    pdl_wait();
    pdl_trigger();
    plan_share<FW_R, KT, FW_OV, FW_MINK, FW_THREADS>(a, blockIdx.x, gridDim.x, sc);
    if (sc.share.n == 0) return;
    auto wait_all = [&](uint64_t *b, uint32_t parity) -> bool {
        return __all_sync(0xffffffffu, bounded_wait(b, parity, &dead, a.err));
    };

    PlanWalk<FW_R, KT> w(a, sc.share);
    if (warp == FW_WARPS) {
        int it = 0;
        bool ok = true;
        for (bool more = w.load(); more && ok; more = w.next())
            for (int t = w.tl; t < w.th; ++t, ++it) {
                const int s = it % NS;
                if (!(ok = wait_all(&free_[s], ((it / NS) & 1) ^ 1))) break;
                const int k0 = (w.g.t0 + t) * KT;
                // boxes that hold keys of the item
                const int lo = max(w.g.kb - k0, 0) / box, hi = (min(w.g.ke - k0, KT) + box - 1) / box;
                const int nb = max(hi - lo, 0);
                if (lane == 0) {
                    if (nb) mbar_arrive_expect_tx(&full[s], (uint32_t)nb * box * 256 * C::PANELS);
                    else mbar_arrive(&full[s]);
                }
                __syncwarp();
                for (int i = lane; i < nb * C::PANELS * 2; i += 32) {
                    const int row = (lo + i % nb) * box, p = i / nb % C::PANELS, v = i / nb / C::PANELS, key = k0 + row;
                    uint8_t *d = ring + (s * 2 + v) * C::TILE + p * C::PANEL + row * 128;
                    const CUtensorMap *map = v ? &vmap : &kmap;
                    if (a.table) {
                        const int pg = key / a.page_size, page = a.table[(int64_t)w.b * a.max_pages + pg];
                        tma_load_4d(d, map, &full[s], p * 64, key - pg * a.page_size, w.kvh, page);
                    } else {
                        tma_load_3d(d, map, &full[s], p * 64, w.s.q0 + key, w.kvh);
                    }
                }
                __syncwarp();
            }
        if (!ok && lane == 0)  // copies in flight land before the block ends
            for (int s = 0; s < NS; ++s) {
                const int n = (it - s + NS - 1) / NS;
                const long long t0 = clock64();
                if (n > 0)
                    while (!mbar_try_wait(&full[s], (n - 1) & 1))
                        if (clock64() - t0 > ATTN_WAIT_CLOCKS) break;
            }
        return;
    }

    const int g8 = lane >> 2, t4 = lane & 3;
    const float c = __fmul_rn(a.scale, 1.4426950408889634f);
    int it = 0;
    uint32_t meets = 0;
    auto meet = [&]() -> bool {  // the four warps
        __syncwarp();
        if (lane == 0) mbar_arrive(&meet_bar);
        return wait_all(&meet_bar, meets++ & 1);
    };
    for (bool more = w.load(); more; more = w.next()) {
        const ItemGeo g = w.g;
        // Q: rows g8 and g8 + 8 of the item, zeros past it and past head_dim
        uint32_t qf[HD / 16][4];
        int pos[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int f = g.r0 + g8 + 8 * i;
            const bool in = f < g.r1;
            const int tok = in ? div_g(a, f) : 0;
            pos[i] = in ? w.s.p0 + tok : -1;
            const T *q = reinterpret_cast<const T *>(a.q) + (int64_t)(w.s.q0 + tok) * a.qs[0] +
                         (int64_t)(w.kvh * a.G + (in ? f - tok * a.G : 0)) * a.qs[1];
#pragma unroll
            for (int k = 0; k < HD / 16; ++k)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int d = k * 16 + x * 8 + 2 * t4;
                    qf[k][2 * x + i] = in && d < a.D ? *reinterpret_cast<const uint32_t *>(q + d) : 0u;
                }
        }
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, o[HD / 8][4];
#pragma unroll
        for (int n = 0; n < HD / 8; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[n][x] = 0.0f;
        bool ok = true;
        const int mine = w.tl + (warp - it % FW_WARPS + FW_WARPS) % FW_WARPS;  // tile it % 4 is this warp's
        for (int t = mine; t < w.th; t += FW_WARPS) {
            const int n = it + t - w.tl, s = n % NS;
            if (!(ok = wait_all(&full[s], (n / NS) & 1))) break;
            const int k0 = (g.t0 + t) * KT;
            const uint32_t kt = smem_u32(ring + s * 2 * C::TILE), vt = kt + C::TILE;
            float sc4[KT / 8][4];
#pragma unroll
            for (int nt = 0; nt < KT / 8; ++nt) {
#pragma unroll
                for (int x = 0; x < 4; ++x) sc4[nt][x] = 0.0f;
#pragma unroll
                for (int kp = 0; kp < HD / 32; ++kp) {  // 32 columns: two steps of 16
                    uint32_t b[4];
                    const int row = nt * 8 + (lane & 7), ch = kp * 4 + (lane >> 3);
                    ldsm4(b, kt + (ch >> 3) * C::PANEL + row * 128 + (((ch & 7) ^ (row & 7)) << 4));
                    mma16<T>(sc4[nt], qf[2 * kp], b[0], b[1]);
                    mma16<T>(sc4[nt], qf[2 * kp + 1], b[2], b[3]);
                }
            }
            const bool masked = k0 + KT - 1 > g.pmin || (a.window > 0 && k0 < g.pmax - a.window + 1);
            if (masked) {
#pragma unroll
                for (int nt = 0; nt < KT / 8; ++nt)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int key = k0 + nt * 8 + 2 * t4 + (x & 1), p = pos[x >> 1];
                        if (key > p || (a.window > 0 && key <= p - a.window)) sc4[nt][x] = -INFINITY;
                    }
                // V rows outside the item's keys hold anything: zeros.  Non-finite V that only some rows see is
                // added to those and taken out.
                uint8_t *v = ring + (s * 2 + 1) * C::TILE;
                bool bad = false;
                for (int i = lane; i < KT * C::PANELS * 8; i += 32) {
                    const int r = i / 8 % KT, key = k0 + r;
                    if (key >= max(g.kb, a.window > 0 ? g.pmax - a.window + 1 : 0) && key <= g.pmin) continue;
                    uint4 *q = reinterpret_cast<uint4 *>(v) + i;
                    if (key < g.kb || key >= g.ke) {
                        *q = make_uint4(0, 0, 0, 0);
                        continue;
                    }
                    const uint4 x = *q;
                    const uint32_t e[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                    for (int y = 0; y < 4; ++y) bad |= (e[y] & E::EXP) == E::EXP || (e[y] >> 16 & E::EXP) == E::EXP;
                }
                __syncwarp();
                if (__any_sync(0xffffffffu, bad)) {
#pragma unroll 1
                    for (int r = 0; r < KT; ++r) {
                        const int key = k0 + r;
                        if (key < g.kb || key >= g.ke) continue;
#pragma unroll
                        for (int nt = 0; nt < HD / 8; ++nt) {
                            const uint32_t x = *reinterpret_cast<const uint32_t *>(
                                v + (nt >> 3) * C::PANEL + r * 128 + (((nt & 7) ^ (r & 7)) << 4) + 4 * t4);
#pragma unroll
                            for (int y = 0; y < 4; ++y) {
                                const int p = pos[y >> 1];
                                const float f = E::up(y & 1 ? x >> 16 : x & 0xFFFFu);
                                if (!isfinite(f) && key <= p && !(a.window > 0 && key <= p - a.window))
                                    o[nt][y] = __fadd_rn(o[nt][y], f);
                            }
                        }
                    }
                    __syncwarp();
                    for (int i = lane; i < KT * C::PANELS * 32; i += 32) {
                        uint32_t *q = reinterpret_cast<uint32_t *>(v) + i;
                        uint32_t x = *q;
                        if ((x & E::EXP) == E::EXP) x &= 0xFFFF0000u;
                        if ((x >> 16 & E::EXP) == E::EXP) x &= 0x0000FFFFu;
                        *q = x;
                    }
                    __syncwarp();
                }
            }
            uint32_t pf[KT / 16][4];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float top = -INFINITY;
#pragma unroll
                for (int nt = 0; nt < KT / 8; ++nt) top = fmaxf(top, fmaxf(sc4[nt][2 * i], sc4[nt][2 * i + 1]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float mn = fmaxf(m[i], top), mc = mn == -INFINITY ? 0.0f : __fmul_rn(mn, c);
                const float corr = ex2(__fmaf_rn(m[i], c, -mc)), nmc = __fsub_rn(E::BIAS, mc);
                m[i] = mn;
                float sum = 0.0f;
#pragma unroll
                for (int nt = 0; nt < KT / 8; ++nt) {
                    const float p0 = ex2(__fmaf_rn(sc4[nt][2 * i], c, nmc));
                    const float p1 = ex2(__fmaf_rn(sc4[nt][2 * i + 1], c, nmc));
                    sum = __fadd_rn(sum, __fadd_rn(p0, p1));
                    pf[nt / 2][(nt & 1) * 2 + i] = E::pack(p0, p1);
                }
                sum = __fadd_rn(sum, __shfl_xor_sync(0xffffffffu, sum, 1));
                sum = __fadd_rn(sum, __shfl_xor_sync(0xffffffffu, sum, 2));
                l[i] = __fmaf_rn(l[i], corr, sum);
#pragma unroll
                for (int nt = 0; nt < HD / 8; ++nt) {
                    o[nt][2 * i] = __fmul_rn(o[nt][2 * i], corr);
                    o[nt][2 * i + 1] = __fmul_rn(o[nt][2 * i + 1], corr);
                }
            }
#pragma unroll
            for (int kk = 0; kk < KT / 16; ++kk)
#pragma unroll
                for (int nn = 0; nn < HD / 16; ++nn) {
                    uint32_t b[4];
                    const int j = lane >> 3, row = 16 * kk + (lane & 7) + 8 * (j & 1), ch = 2 * nn + (j >> 1);
                    ldsm4_t(b, vt + (ch >> 3) * C::PANEL + row * 128 + (((ch & 7) ^ (row & 7)) << 4));
                    mma16<T>(o[2 * nn], pf[kk], b[0], b[1]);
                    mma16<T>(o[2 * nn + 1], pf[kk], b[2], b[3]);
                }
            if (masked) fence_async_smem();  // V rows written here, and by TMA next
            __syncwarp();
            if (lane == 0) mbar_arrive(&free_[s]);
        }
        it += w.th - w.tl;
        if (!ok) return;

        // the four warps' parts in shared memory; thread: row tid / 8, HD / 8 columns
        float *rec = recs + warp * C::REC;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int nt = 0; nt < HD / 8; ++nt)
                *reinterpret_cast<float2 *>(rec + (g8 + 8 * i) * C::LDR + nt * 8 + 2 * t4) =
                    make_float2(o[nt][2 * i], o[nt][2 * i + 1]);
            if (t4 == 0) {
                wm[warp][g8 + 8 * i] = m[i] == -INFINITY ? m[i] : __fmul_rn(m[i], c);  // in powers of two
                wl[warp][g8 + 8 * i] = l[i];
            }
        }
        if (!meet()) return;
        constexpr int CW = HD / 8;
        const int row = tid >> 3, col = (tid & 7) * CW;
        float mm = -INFINITY, ll = 0.0f, acc[CW];
#pragma unroll
        for (int x = 0; x < FW_WARPS; ++x) mm = fmaxf(mm, wm[x][row]);
#pragma unroll
        for (int d = 0; d < CW; ++d) acc[d] = 0.0f;
        float ms = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
        for (int x = 0; x < FW_WARPS; ++x) {
            const float e = ex2(__fsub_rn(wm[x][row], ms));
            ll = __fmaf_rn(wl[x][row], e, ll);
#pragma unroll
            for (int d = 0; d < CW; d += 4) {
                const float4 v = *reinterpret_cast<const float4 *>(recs + x * C::REC + row * C::LDR + col + d);
                acc[d] = __fmaf_rn(v.x, e, acc[d]);
                acc[d + 1] = __fmaf_rn(v.y, e, acc[d + 1]);
                acc[d + 2] = __fmaf_rn(v.z, e, acc[d + 2]);
                acc[d + 3] = __fmaf_rn(v.w, e, acc[d + 3]);
            }
        }
        if (!w.whole()) {
            const CutItem ci = cut_item(w);
            float *p = a.part + ((int64_t)blockIdx.x * 2 + (w.tl == 0)) * C::PART;
#pragma unroll
            for (int d = 0; d < CW; d += 4)
                __stcg(reinterpret_cast<float4 *>(p + row * HD + col + d),
                       make_float4(acc[d], acc[d + 1], acc[d + 2], acc[d + 3]));
            if ((tid & 7) == 0) {
                __stcg(p + FW_R * HD + row, mm);
                __stcg(p + FW_R * (HD + 1) + row, ll);
            }
            __threadfence();
            if (!meet()) return;
            if (tid == 0) {
                lastf = atomicAdd(a.ticket + ci.k0, 1u) == (unsigned)(ci.k1 - ci.k0);
                if (lastf) a.ticket[ci.k0] = 0u;
            }
            if (!meet()) return;
            if (!lastf) continue;
            __threadfence();
            mm = -INFINITY;
            ll = 0.0f;
#pragma unroll
            for (int d = 0; d < CW; ++d) acc[d] = 0.0f;
            auto part = [&](int k) { return a.part + ((int64_t)k * 2 + (k == ci.k0)) * C::PART; };
#pragma unroll 4
            for (int k = ci.k0; k <= ci.k1; ++k) mm = fmaxf(mm, __ldcg(part(k) + FW_R * HD + row));
            ms = mm == -INFINITY ? 0.0f : mm;
#pragma unroll 4
            for (int k = ci.k0; k <= ci.k1; ++k) {
                const float *q = part(k);
                const float e = ex2(__fsub_rn(__ldcg(q + FW_R * HD + row), ms));
                ll = __fmaf_rn(__ldcg(q + FW_R * (HD + 1) + row), e, ll);
#pragma unroll
                for (int d = 0; d < CW; d += 4) {
                    const float4 v = __ldcg(reinterpret_cast<const float4 *>(q + row * HD + col + d));
                    acc[d] = __fmaf_rn(v.x, e, acc[d]);
                    acc[d + 1] = __fmaf_rn(v.y, e, acc[d + 1]);
                    acc[d + 2] = __fmaf_rn(v.z, e, acc[d + 2]);
                    acc[d + 3] = __fmaf_rn(v.w, e, acc[d + 3]);
                }
            }
        }
        const int f = g.r0 + row;
        if (f < g.r1 && col < a.D) {
            const int tok = div_g(a, f), h = w.kvh * a.G + f - tok * a.G;
            const float sink = a.sinks ? __fmul_rn(a.sinks[h], 1.4426950408889634f) : 0.0f;
            const float inv = row_factor<E>(mm, ll, a.sinks != nullptr, sink);
            const bool none = mm == -INFINITY && ll == 0.0f;
            T *out = reinterpret_cast<T *>(a.out) + (int64_t)(w.s.q0 + tok) * a.os[0] + (int64_t)h * a.os[1] + col;
#pragma unroll
            for (int d = 0; d < CW; d += 8) {
                uint32_t e[4];
#pragma unroll
                for (int y = 0; y < 4; ++y)
                    e[y] = none ? 0u : E::pack(__fmul_rn(acc[d + 2 * y], inv), __fmul_rn(acc[d + 2 * y + 1], inv));
                if (col + d < a.D) *reinterpret_cast<uint4 *>(out + d) = make_uint4(e[0], e[1], e[2], e[3]);
            }
        }
        if (!meet()) return;  // the records may be written again
    }
}

template <typename T, int HD>
cudaError_t few_set() {
    return cudaFuncSetAttribute(attn_few_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)FewCfg<HD>::SMEM);
}

template <typename T, int HD>
cudaError_t few_run(const AttnOp &a, int dtype, int nsm, cudaStream_t st, bool &can) {
    const int box = std::min(a.table ? a.page_size & -a.page_size : 128, FewCfg<HD>::KT);
    CUtensorMap k, v;
    can = kv_tensor_map(a, false, dtype, box, k) && kv_tensor_map(a, true, dtype, box, v);
    if (!can) return cudaSuccess;
    return launch_k(attn_few_kernel<T, HD>, dim3(nsm * FW_PER_SM), dim3(FW_THREADS), FewCfg<HD>::SMEM, st, a, k, v, box);
}

}  // namespace

size_t attn_few_part_floats(int nsm) { return (size_t)nsm * FW_PER_SM * 2 * FewCfg<128>::PART; }

cudaError_t attn_few_configure() {
    cudaError_t e = few_set<__half, 64>();
    if (e == cudaSuccess) e = few_set<__half, 128>();
    if (e == cudaSuccess) e = few_set<__nv_bfloat16, 64>();
    if (e == cudaSuccess) e = few_set<__nv_bfloat16, 128>();
    return e;
}

bool launch_attn_few(const AttnOp &a, int dtype, int nsm, cudaStream_t st, cudaError_t &e) {
    bool can;
    if (dtype == PC_DT_F16)
        e = a.D <= 64 ? few_run<__half, 64>(a, dtype, nsm, st, can) : few_run<__half, 128>(a, dtype, nsm, st, can);
    else
        e = a.D <= 64 ? few_run<__nv_bfloat16, 64>(a, dtype, nsm, st, can)
                      : few_run<__nv_bfloat16, 128>(a, dtype, nsm, st, can);
    return can;
}

}  // namespace pc
