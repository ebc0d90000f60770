// attention_rows.cu - attention of many rows over pages and packed prompts on
// the 5th-generation tensor cores, for f16 and bf16 tensors.
//
// A thread block (one per SM) takes the items of its share
// (attention_plan.cuh): 256 rows (tokens x query heads of one KV head) as two
// tiles of 128, against key tiles of 128.  Roles:
//   warps 0-3, 4-7  one row tile each, one row per thread: scores from TMEM,
//                   running maximum and sum, weights back to TMEM, and at the
//                   end of an item the output
//   warp 8          K and V tiles by TMA into a ring (one box per page piece)
//   warp 9          tcgen05.mma: S = Q K^T (both from shared memory), O += P V
//                   (P from TMEM, V from shared memory as it lies: keys are
//                   the strided, head columns the contiguous dimension)
//   warps 10, 11    Q rows of the next item; V rows of masked tiles put in
//                   order (below)
// With two row tiles one is in the softmax while the other's products run.
// At head sizes to 64, S, P and O of both tiles fit TMEM's 512 columns side
// by side, so the next S is computed while a row group is still in its
// exponentials; at 128, P takes the place of its S.
//
// The maximum that weights are taken against is moved only when a row's
// maximum has grown by more than 2^8 (any reference within the exponent
// range gives the same quotient), so O is hardly ever rescaled.
//
// A key that a row does not see has weight 0, but 0 x NaN is NaN: in tiles
// that some row does not see whole, V rows outside the item's keys (stale
// pages) are zeroed and non-finite V elements of the others taken out before
// the product; if there were any, the rows that see them get them added back
// from global memory at the end of the item.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "attention_plan.cuh"
#include "launch.cuh"
#include "sm100.cuh"

namespace pc {

namespace {

constexpr int RW_R = 256, RW_KT = 128, RW_OV = 128, RW_MINK = 256, RW_THREADS = 384;
constexpr long long RW_WAIT_CLOCKS = 2000000000ll;  // about a second
constexpr float RW_GROW = 8.0f;                     // log2 of the growth that moves the reference

template <int HD>
struct RowsCfg {
    static constexpr int PANELS = HD / 64;        // 64-column (128-byte) panels of a row
    static constexpr int TILE = PANELS * 16384;   // bytes of 128 rows
    static constexpr int STAGES = HD == 64 ? 3 : 2;
    static constexpr bool ALIAS = HD == 128;      // P in the place of S
    static constexpr int S0 = 0, P0 = ALIAS ? 0 : 256, PSTEP = ALIAS ? 128 : 64, O0 = ALIAS ? 256 : 384;
    static constexpr size_t SMEM = 1024 + (size_t)TILE * (2 + 2 * STAGES);
    static constexpr int PART = RW_R * (HD + 2);
};

struct RowsBars {
    uint64_t q_full[2], q_free[2], s_full[2], s_free[2], p_full[2], o_full[2];
    uint64_t k_full[3], k_free[3], v_full[3], v_free[3], v_fixed[3], both, drain;
};

__device__ __forceinline__ void tma_load_3d(void *dst, const CUtensorMap *map, uint64_t *bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
        "[%5];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void tma_load_4d(void *dst, const CUtensorMap *map, uint64_t *bar, int x, int y, int z,
                                            int w) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, "
        "%5}], [%6];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void cp_async16_fill(uint32_t dst, const void *src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// 32 consecutive TMEM columns of this thread's lane
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t *v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
          "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
          "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t *v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// D[tmem] (+)= A[tmem] x B[smem], 16-bit operands, fp32 sums
__device__ __forceinline__ void tc_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                          bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
}

// Descriptor of a B operand whose N dimension is contiguous (128-byte
// swizzled rows of 64 elements, one row per k): 8-row groups 1024 bytes
// apart, further 64-column panels `panel` bytes apart.
__device__ __forceinline__ uint64_t sw128_desc_n(uint32_t saddr, int panel) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(panel >> 4) << 16) | ((1024ull >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Element types: instruction-descriptor code, packing, the bits of a
// non-finite exponent, and the power of two that weights are stored at (f16
// weights keep 7 binary orders more before they underflow; the sums carry
// the same factor, so the quotient does not change).
template <typename T>
struct Half16;
template <>
struct Half16<__nv_bfloat16> {
    static constexpr uint32_t FMT = 1, EXP = 0x7F80u;
    static constexpr float BIAS = 0.0f;
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        uint32_t r;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
        return r;
    }
    static __device__ __forceinline__ float up(uint32_t h) { return __uint_as_float(h << 16); }
};
template <>
struct Half16<__half> {
    static constexpr uint32_t FMT = 0, EXP = 0x7C00u;
    static constexpr float BIAS = 7.0f;
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        uint32_t r;
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
        return r;
    }
    static __device__ __forceinline__ float up(uint32_t h) { return __half2float(__ushort_as_half((unsigned short)h)); }
};

template <typename T, int HD>
__global__ void __launch_bounds__(RW_THREADS, 1)
    attn_rows_kernel(const AttnOp a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                     const int box) {
    using C = RowsCfg<HD>;
    using E = Half16<T>;
    constexpr int NS = C::STAGES;
    extern __shared__ uint8_t rows_smem_raw[];
    uint8_t *smem = rows_smem_raw + (1024 - (smem_u32(rows_smem_raw) & 1023)) % 1024;
    uint8_t *qs = smem, *ks = qs + 2 * C::TILE, *vs = ks + NS * C::TILE;
    __shared__ PlanScratch<RW_THREADS> sc;
    __shared__ RowsBars bar;
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int dead;
    __shared__ int lastf;
    __shared__ volatile int odd[4];  // [i % 4] = i + 1: non-finite V in a masked tile of the block's item i
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        for (int t = 0; t < 2; ++t) {
            mbar_init(&bar.q_full[t], 64);
            mbar_init(&bar.q_free[t], 1);
            mbar_init(&bar.s_full[t], 1);
            mbar_init(&bar.s_free[t], 128);
            mbar_init(&bar.p_full[t], 128);
            mbar_init(&bar.o_full[t], 1);
        }
        for (int s = 0; s < NS; ++s) {
            mbar_init(&bar.k_full[s], 1);
            mbar_init(&bar.k_free[s], 1);
            mbar_init(&bar.v_full[s], 1);
            mbar_init(&bar.v_free[s], 1);
            mbar_init(&bar.v_fixed[s], 64);
        }
        mbar_init(&bar.both, 256);
        mbar_init(&bar.drain, 1);
        fence_mbar_init();
        dead = 0;
        for (int i = 0; i < 4; ++i) odd[i] = 0;
    }
    if (warp == 9) {
        tmem_alloc(&tmem_slot, 512);
        tmem_relinquish();
    }
    pdl_wait();
    pdl_trigger();
    plan_share<RW_R, RW_KT, RW_OV, RW_MINK, RW_THREADS>(a, blockIdx.x, gridDim.x, sc);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tm = tmem_slot;

    // A bounded wait: false once it, or any other wait of the block, gave up.
    auto wait = [&](uint64_t *b, uint32_t parity) -> bool {
        if (mbar_try_wait(b, parity)) return true;
        const long long t0 = clock64();
        while (!mbar_try_wait(b, parity)) {
            if (dead) return false;
            if (clock64() - t0 > RW_WAIT_CLOCKS) {
                dead = 1;
                atomicExch(a.err, 1);
                return false;
            }
        }
        return true;
    };
    // a tile of keys that some row of the item does not see whole
    auto masked = [&](const ItemGeo &g, int t) -> bool {
        const int k0 = (g.t0 + t) * RW_KT;
        return k0 + RW_KT - 1 > g.pmin || (a.window > 0 && k0 < g.pmax - a.window + 1);
    };

    if (sc.share.n == 0) {
        // no share
    } else if (warp == 8) {
        // ---- K and V tiles ----
        PlanWalk<RW_R, RW_KT> w(a, sc.share);
        int it = 0, fills[2] = {0, 0};
        bool ok = true;
        for (bool more = w.load(); more && ok; more = w.next()) {
            for (int t = w.tl; t < w.th && ok; ++t, ++it) {
                const int s = it % NS;
                const uint32_t ph = (it / NS) & 1;
                const int k0 = (w.g.t0 + t) * RW_KT;
                // boxes that hold keys of the item
                const int lo = max(w.g.kb - k0, 0) / box, hi = (min(w.g.ke - k0, RW_KT) + box - 1) / box;
                const int nb = max(hi - lo, 0);
                for (int kv = 0; kv < 2 && ok; ++kv) {
                    uint64_t *full = kv ? &bar.v_full[s] : &bar.k_full[s];
                    ok = wait(kv ? &bar.v_free[s] : &bar.k_free[s], ph ^ 1);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    uint8_t *dst = (kv ? vs : ks) + s * C::TILE;
                    const CUtensorMap *map = kv ? &vmap : &kmap;
                    if (lane == 0) {
                        if (nb) mbar_arrive_expect_tx(full, (uint32_t)nb * box * 128 * C::PANELS);
                        else mbar_arrive(full);
                    }
                    ++fills[kv];
                    __syncwarp();
                    for (int i = lane; i < nb * C::PANELS; i += 32) {
                        const int p = i / nb, row = (lo + i % nb) * box, key = k0 + row;
                        uint8_t *d = dst + p * 16384 + row * 128;
                        if (a.table) {
                            const int page = __ldg(a.table + (int64_t)w.b * a.max_pages + key / a.page_size);
                            tma_load_4d(d, map, full, p * 64, key % a.page_size, w.kvh, page);
                        } else {
                            tma_load_3d(d, map, full, p * 64, w.s.q0 + key, w.kvh);
                        }
                    }
                    __syncwarp();
                }
            }
        }
        if (!ok && lane == 0)  // copies in flight land before the block ends
            for (int s = 0; s < NS; ++s)
                for (int kv = 0; kv < 2; ++kv) {
                    const int n = (fills[kv] - s + NS - 1) / NS;  // fills of this stage
                    const long long t0 = clock64();
                    if (n > 0)
                        while (!mbar_try_wait(kv ? &bar.v_full[s] : &bar.k_full[s], (n - 1) & 1))
                            if (clock64() - t0 > RW_WAIT_CLOCKS) break;
                }
    } else if (warp == 9) {
        // ---- products ----
        if (lane == 0) {
            constexpr uint32_t ID_QK = (1u << 4) | (E::FMT << 7) | (E::FMT << 10) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
            constexpr uint32_t ID_PV = (1u << 4) | (E::FMT << 7) | (E::FMT << 10) | (1u << 16) | (((uint32_t)HD >> 3) << 17) |
                                       ((128u >> 4) << 24);
            PlanWalk<RW_R, RW_KT> w(a, sc.share);
            int kit = 0, vit = 0, n = 0, item = 0;  // n: tiles begun (S of both row tiles)
            bool ok = true;
            auto qk = [&](int t, int s) {  // S[t] = Q[t] K^T
                const uint64_t qd = sw128_desc(qs + t * C::TILE), kd = sw128_desc(ks + s * C::TILE);
#pragma unroll
                for (int k = 0; k < HD / 16; ++k) {
                    const int off = (k / 4) * (16384 >> 4) + (k % 4) * 2;
                    tc_mma_f16(tm + C::S0 + t * 128, qd + off, kd + off, ID_QK, k > 0);
                }
                tc_commit(&bar.s_full[t]);
            };
            auto pv = [&](int t, int s, bool acc) {  // O[t] (+)= P[t] V
#pragma unroll
                for (int k = 0; k < RW_KT / 16; ++k)
                    tc_mma_ts(tm + C::O0 + t * HD, tm + C::P0 + t * C::PSTEP + k * 8,
                              sw128_desc_n(smem_u32(vs + s * C::TILE) + k * 2048, 16384), ID_PV, acc || k > 0);
                tc_commit(&bar.o_full[t]);
            };
            for (bool more = w.load(); more && ok; more = w.next(), ++item) {
                for (int j = w.tl - 1; j < w.th && ok; ++j) {
                    // S of tile j + 1
                    auto next_s = [&](int t) -> bool {
                        if (j + 1 >= w.th) return true;
                        if (j + 1 == w.tl && !wait(&bar.q_full[t], item & 1)) return false;
                        if (t == 0 && !wait(&bar.k_full[kit % NS], (kit / NS) & 1)) return false;
                        if (!C::ALIAS && n > 0 && !wait(&bar.s_free[t], (n - 1) & 1)) return false;
                        tc_fence_after();
                        qk(t, kit % NS);
                        if (j + 2 == w.th) tc_commit(&bar.q_free[t]);
                        if (t == 1) {
                            tc_commit(&bar.k_free[kit % NS]);
                            ++kit;
                            ++n;
                        }
                        return true;
                    };
                    auto this_o = [&](int t) -> bool {
                        if (j < w.tl) return true;
                        const int s = vit % NS;
                        if (t == 0 && !wait(&bar.v_full[s], (vit / NS) & 1)) return false;
                        if (t == 0 && !wait(&bar.v_fixed[s], (vit / NS) & 1)) return false;
                        if (!wait(&bar.p_full[t], vit & 1)) return false;
                        tc_fence_after();
                        pv(t, s, j > w.tl);
                        if (t == 1) {
                            tc_commit(&bar.v_free[s]);
                            ++vit;
                        }
                        return true;
                    };
                    if (C::ALIAS) ok = this_o(0) && next_s(0) && this_o(1) && next_s(1);
                    else ok = next_s(0) && next_s(1) && this_o(0) && this_o(1);
                }
            }
            if (!ok) {  // products in flight end before TMEM is freed
                tc_commit(&bar.drain);
                const long long t0 = clock64();
                while (!mbar_try_wait(&bar.drain, 0))
                    if (clock64() - t0 > RW_WAIT_CLOCKS) break;
            }
        }
        __syncwarp();
    } else if (warp >= 10) {
        // ---- Q rows, V rows of masked tiles ----
        const int ht = tid - 320;
        PlanWalk<RW_R, RW_KT> w(a, sc.share);
        int it = 0, item = 0;
        bool ok = true;
        for (bool more = w.load(); more && ok; more = w.next(), ++item) {
            const T *q = reinterpret_cast<const T *>(a.q) + (int64_t)w.s.q0 * a.qs[0] + (int64_t)w.kvh * a.G * a.qs[1];
            for (int t = 0; t < 2 && ok; ++t) {
                ok = item == 0 || wait(&bar.q_free[t], (item - 1) & 1);
                if (!ok) break;
                const uint32_t dst = smem_u32(qs + t * C::TILE);
                for (int i = ht; i < 128 * C::PANELS * 8; i += 64) {
                    const int r = i / (C::PANELS * 8), c = i % (C::PANELS * 8), f = w.g.r0 + t * 128 + r;
                    const bool in = f < w.g.r1 && c * 8 < a.D;
                    const int fc = in ? f : 0, cc = in ? c : 0;
                    cp_async16_fill(dst + (c / 8) * 16384 + r * 128 + (((c % 8) ^ (r & 7)) << 4),
                                    q + (int64_t)(fc / a.G) * a.qs[0] + (int64_t)(fc % a.G) * a.qs[1] + cc * 8,
                                    in ? 16 : 0);
                }
                cp_async_commit();
                cp_async_wait<0>();
                fence_async_smem();
                mbar_arrive(&bar.q_full[t]);
            }
            for (int t = w.tl; t < w.th && ok; ++t, ++it) {
                const int s = it % NS;
                ok = wait(&bar.v_full[s], (it / NS) & 1);
                if (!ok) break;
                if (masked(w.g, t)) {
                    const int k0 = (w.g.t0 + t) * RW_KT;
                    uint8_t *v = vs + s * C::TILE;
                    bool bad = false;
                    for (int i = ht; i < 128 * C::PANELS * 8; i += 64) {
                        const int r = (i / 8) % 128, key = k0 + r;
                        uint4 *p = reinterpret_cast<uint4 *>(v) + i;  // 16 bytes of row r, wherever the swizzle puts them
                        if (key < w.g.kb || key >= w.g.ke) {
                            *p = make_uint4(0, 0, 0, 0);
                        } else {
                            uint4 x = *p;
                            uint32_t *e = reinterpret_cast<uint32_t *>(&x);
                            bool hit = false;
#pragma unroll
                            for (int m = 0; m < 4; ++m) {
                                if ((e[m] & E::EXP) == E::EXP) e[m] &= 0xFFFF0000u, hit = true;
                                if ((e[m] >> 16 & E::EXP) == E::EXP) e[m] &= 0x0000FFFFu, hit = true;
                            }
                            if (hit) {
                                *p = x;
                                bad = true;
                            }
                        }
                    }
                    if (bad) odd[item & 3] = item + 1;
                    fence_async_smem();
                }
                mbar_arrive(&bar.v_fixed[s]);
            }
        }
    } else {
        // ---- softmax and output of row tile t ----
        const int t = warp >> 2, r = tid & 127;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;
        const uint32_t sc_t = tm + lanes + C::S0 + t * 128, pt_t = tm + lanes + C::P0 + t * C::PSTEP,
                       ot_t = tm + lanes + C::O0 + t * HD;
        const float c = __fmul_rn(a.scale, 1.4426950408889634f);
        PlanWalk<RW_R, RW_KT> w(a, sc.share);
        int it = 0, item = 0;
        uint32_t both_n = 0;
        bool ok = true;
        auto both = [&]() -> bool {  // the two row tiles' threads meet
            mbar_arrive(&bar.both);
            return __all_sync(0xffffffffu, wait(&bar.both, both_n++ & 1));
        };
        for (bool more = w.load(); more && ok; more = w.next(), ++item) {
            const ItemGeo g = w.g;
            const int f = g.r0 + t * 128 + r;
            const int pos = f < g.r1 ? w.s.p0 + f / a.G : -1;
            float m = -INFINITY, l = 0.0f;  // reference (of the scores as they are), sum
            for (int j = w.tl; j < w.th && ok; ++j, ++it) {
                ok = wait(&bar.s_full[t], it & 1);
                if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                tc_fence_after();
                uint32_t sv[128];
#pragma unroll
                for (int x = 0; x < 4; ++x) tmem_ld32(sc_t + 32 * x, sv + 32 * x);
                tmem_ld_wait();
                if (!C::ALIAS) {
                    tc_fence_before();
                    mbar_arrive(&bar.s_free[t]);
                }
                if (masked(g, j)) {
                    const int k0 = (g.t0 + j) * RW_KT, hi = pos - k0, lo = a.window > 0 ? hi - a.window : -1;
#pragma unroll
                    for (int x = 0; x < 128; ++x)
                        if (x > hi || x <= lo) sv[x] = 0xFF800000u;
                }
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int x = 0; x < 128; ++x) top[x & 3] = fmaxf(top[x & 3], __uint_as_float(sv[x]));
                const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                // move the reference of rows whose maximum has grown
                const bool first = m == -INFINITY;
                const bool grow = !first && __fmul_rn(__fsub_rn(mx, m), c) > RW_GROW;
                float corr = 1.0f;
                if (grow) corr = ex2(__fmul_rn(__fsub_rn(m, mx), c));
                if (first || grow) m = mx;
                l = __fmul_rn(l, corr);
                if (j > w.tl) {  // P and O are this thread's again
                    ok = wait(&bar.o_full[t], (it - 1) & 1);
                    if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                    tc_fence_after();
                    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                        for (int x = 0; x < HD / 16; ++x) {
                            uint32_t ov[16];
                            tmem_ld16(ot_t + 16 * x, ov);
                            tmem_ld_wait();
#pragma unroll
                            for (int y = 0; y < 16; ++y) ov[y] = __float_as_uint(__fmul_rn(__uint_as_float(ov[y]), corr));
                            tmem_st16(ot_t + 16 * x, ov);
                        }
                    }
                }
                const float mc = m == -INFINITY ? 0.0f : __fsub_rn(__fmul_rn(m, c), E::BIAS);
                float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    uint32_t pk[16];
#pragma unroll
                    for (int y = 0; y < 16; ++y) {
                        const float p0 = ex2(__fmaf_rn(__uint_as_float(sv[32 * x + 2 * y]), c, -mc));
                        const float p1 = ex2(__fmaf_rn(__uint_as_float(sv[32 * x + 2 * y + 1]), c, -mc));
                        sum[(2 * y) & 3] = __fadd_rn(sum[(2 * y) & 3], p0);
                        sum[(2 * y + 1) & 3] = __fadd_rn(sum[(2 * y + 1) & 3], p1);
                        pk[y] = E::pack(p0, p1);
                    }
                    tmem_st16(pt_t + 16 * x, pk);
                }
                tmem_st_wait();
                tc_fence_before();
                mbar_arrive(&bar.p_full[t]);
                l = __fadd_rn(l, __fadd_rn(__fadd_rn(sum[0], sum[1]), __fadd_rn(sum[2], sum[3])));
            }
            if (!ok) break;
            ok = wait(&bar.o_full[t], (it - 1) & 1);
            if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            tc_fence_after();
            float o[HD];
#pragma unroll
            for (int x = 0; x < HD / 32; ++x) tmem_ld32(ot_t + 32 * x, reinterpret_cast<uint32_t *>(o) + 32 * x);
            tmem_ld_wait();
            if (odd[item & 3] == item + 1) {  // non-finite V of masked tiles, for the rows that see it
                for (int j = w.tl; j < w.th; ++j) {
                    if (!masked(g, j)) continue;
                    const int k0 = (g.t0 + j) * RW_KT;
                    for (int key = max(max(k0, g.kb), a.window > 0 ? pos - a.window + 1 : 0);
                         key <= min(min(k0 + RW_KT, g.ke) - 1, pos); ++key) {
                        const T *vp = reinterpret_cast<const T *>(a.v) + (int64_t)w.kvh * a.vs[2];
                        if (a.table) {
                            const int page = a.table[(int64_t)w.b * a.max_pages + key / a.page_size];
                            if (page < 0 || page >= a.n_pages) continue;
                            vp += page * a.vs[0] + (int64_t)(key % a.page_size) * a.vs[1];
                        } else {
                            vp += (int64_t)(w.s.q0 + key) * a.vs[1];
                        }
#pragma unroll
                        for (int d = 0; d < HD; ++d)
                            if (d < a.D) {
                                const float v = E::up(reinterpret_cast<const unsigned short *>(vp)[d]);
                                if (!isfinite(v)) o[d] = __fadd_rn(o[d], v);
                            }
                    }
                }
            }
            float mref = m == -INFINITY ? m : __fmul_rn(m, c);  // in powers of two
            if (!w.whole()) {
                const CutItem cut = cut_item(w);
                float *mine = a.part + ((int64_t)blockIdx.x * 2 + (w.tl == 0)) * C::PART;
#pragma unroll
                for (int d = 0; d < HD; ++d) __stcg(mine + d * RW_R + tid, o[d]);
                __stcg(mine + HD * RW_R + tid, mref);
                __stcg(mine + (HD + 1) * RW_R + tid, l);
                __threadfence();
                if (!(ok = both())) break;
                if (tid == 0) {
                    lastf = atomicAdd(a.ticket + cut.k0, 1u) == (unsigned)(cut.k1 - cut.k0);
                    if (lastf) a.ticket[cut.k0] = 0u;
                }
                if (!(ok = both())) break;
                if (!lastf) continue;
                __threadfence();
                float mm = -INFINITY;
                for (int k = cut.k0; k <= cut.k1; ++k)
                    mm = fmaxf(mm, __ldcg(a.part + ((int64_t)k * 2 + (k == cut.k0)) * C::PART + HD * RW_R + tid));
                const float ms = mm == -INFINITY ? 0.0f : mm;
                l = 0.0f;
#pragma unroll
                for (int d = 0; d < HD; ++d) o[d] = 0.0f;
                for (int k = cut.k0; k <= cut.k1; ++k) {
                    const float *p = a.part + ((int64_t)k * 2 + (k == cut.k0)) * C::PART + tid;
                    const float e = ex2(__fsub_rn(__ldcg(p + HD * RW_R), ms));
                    l = __fmaf_rn(__ldcg(p + (HD + 1) * RW_R), e, l);
#pragma unroll
                    for (int d = 0; d < HD; ++d) o[d] = __fmaf_rn(__ldcg(p + d * RW_R), e, o[d]);
                }
                mref = mm;
            }
            if (f < g.r1) {
                const int h = w.kvh * a.G + f % a.G;
                const bool none = mref == -INFINITY && l == 0.0f;  // no key seen
                float inv = 0.0f;
                if (!none) {
                    float den = l;
                    if (a.sinks) {
                        // both on the larger of the two references; E::BIAS is in l and o
                        const float sk = __fmul_rn(a.sinks[h], 1.4426950408889634f), mm = fmaxf(mref, sk);
                        const float e = ex2(__fsub_rn(mref, mm));
                        den = __fmaf_rn(l, e, ex2(__fadd_rn(__fsub_rn(sk, mm), E::BIAS)));
                        inv = __fdiv_rn(e, den);
                    } else {
                        inv = __fdiv_rn(1.0f, den);
                    }
                }
                T *out = reinterpret_cast<T *>(a.out) + (int64_t)(w.s.q0 + f / a.G) * a.os[0] + (int64_t)h * a.os[1];
#pragma unroll
                for (int d = 0; d < HD; d += 8)
                    if (d < a.D) {
                        uint4 v;
                        uint32_t *e = reinterpret_cast<uint32_t *>(&v);
#pragma unroll
                        for (int y = 0; y < 4; ++y)
                            e[y] = none ? 0u : E::pack(__fmul_rn(o[d + 2 * y], inv), __fmul_rn(o[d + 2 * y + 1], inv));
                        *reinterpret_cast<uint4 *>(out + d) = v;
                    }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tm, 512);
    }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                  const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn rows_encode_fn() {
    static EncodeTiledFn fn = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            return (EncodeTiledFn) nullptr;
        return reinterpret_cast<EncodeTiledFn>(f);
    }();
    return fn;
}

template <typename T, int HD>
cudaError_t rows_set() {
    return cudaFuncSetAttribute(attn_rows_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)RowsCfg<HD>::SMEM);
}

template <typename T, int HD>
cudaError_t rows_run(const AttnOp &a, const CUtensorMap &k, const CUtensorMap &v, int box, int nsm, cudaStream_t st) {
    return launch_k(attn_rows_kernel<T, HD>, dim3(nsm), dim3(RW_THREADS), RowsCfg<HD>::SMEM, st, a, k, v, box);
}

}  // namespace

// K or V as a tensor map: rows of head_dim elements, boxes of 64 columns x
// `box` positions of one head, 128-byte swizzle, zeros outside.  False if its
// strides cannot be described (a stride of zero).
bool kv_tensor_map(const AttnOp &a, bool v, int dtype, int box, CUtensorMap &m) {
    EncodeTiledFn fn = rows_encode_fn();
    if (!fn) return false;
    const int64_t *s = v ? a.vs : a.ks;
    const cuuint64_t rows = a.table ? a.page_size : a.T;
    // a dimension of one element has any stride
    const cuuint64_t unit = (cuuint64_t)((a.D * 2 + 15) / 16 * 16);
    auto stride = [&](int64_t x, cuuint64_t n) { return n == 1 ? unit : (cuuint64_t)x * 2; };
    const cuuint64_t dims[4] = {(cuuint64_t)a.D, rows, (cuuint64_t)a.KVH, (cuuint64_t)a.n_pages};
    const cuuint64_t strides[3] = {stride(s[1], rows), stride(s[2], a.KVH), stride(s[0], a.n_pages)};
    const cuuint32_t boxes[4] = {64u, (cuuint32_t)box, 1u, 1u}, es[4] = {1u, 1u, 1u, 1u};
    return fn(&m, dtype == PC_DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
              a.table ? 4 : 3, const_cast<void *>(v ? a.v : a.k), dims, strides, boxes, es,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

size_t attn_rows_part_floats(int nsm) { return (size_t)nsm * 2 * RowsCfg<128>::PART; }

cudaError_t attn_rows_configure() {
    cudaError_t e = rows_set<__half, 64>();
    if (e == cudaSuccess) e = rows_set<__half, 128>();
    if (e == cudaSuccess) e = rows_set<__nv_bfloat16, 64>();
    if (e == cudaSuccess) e = rows_set<__nv_bfloat16, 128>();
    return e;
}

bool launch_attn_rows(const AttnOp &a, int dtype, int nsm, cudaStream_t st, cudaError_t &e) {
    // positions per TMA box: the largest power of two that divides a page
    const int box = a.table ? min(a.page_size & -a.page_size, RW_KT) : RW_KT;
    CUtensorMap k, v;
    if (!kv_tensor_map(a, false, dtype, box, k) || !kv_tensor_map(a, true, dtype, box, v)) return false;
    if (dtype == PC_DT_F16)
        e = a.D <= 64 ? rows_run<__half, 64>(a, k, v, box, nsm, st) : rows_run<__half, 128>(a, k, v, box, nsm, st);
    else
        e = a.D <= 64 ? rows_run<__nv_bfloat16, 64>(a, k, v, box, nsm, st)
                      : rows_run<__nv_bfloat16, 128>(a, k, v, box, nsm, st);
    return true;
}

}  // namespace pc
