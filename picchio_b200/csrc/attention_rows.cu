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
//   warp 9          tcgen05.mma: S = Q K^T, both from shared memory
//   warp 11         tcgen05.mma: O += P V, P from TMEM, V from shared memory as
//                   it lies (keys are the strided, head columns the
//                   contiguous dimension)
//   warp 10         Q rows of the next item; V rows of masked tiles put in
//                   order (below)
//
// P takes the place of its S in TMEM.  Beside O (2 x head size columns) there
// is room for three such buffers at head sizes to 64 and for two at 128; they
// go round the row tiles in turn, so while one row tile is in the softmax, the
// other's products run, and with three the next S is ready before its row
// tile has finished.
// P is rounded to the type once.  With the remainder as a second product (it has
// room beside P in its S) the error of bf16 outputs would be that of their own
// rounding (16 prompts 2.11e-3 -> 1.66e-3 from the exact result, f16 2.7e-4 ->
// 2.1e-4), but the row warps' work and the product's would cost more than that
// gives: 16 prompts 311 -> 380 us, one 8k prompt 614 -> 883, window of 128 147 ->
// 162.
// The softmax goes through S 32 columns at a time in a short loop: with the
// row's 128 scores in registers the unrolled form had 900 instructions a tile
// and spent more time waiting for instructions than issuing them.
//
// Any reference within the exponent range gives the same quotient, so a row
// keeps its first one (at head sizes to 64 the maximum of its first 32 scores
// where all are seen, else that of its first tile), and later scores are not
// searched for their maximum first: the sum of 32 weights shows when one has
// grown past 2^14 (f16 weights, stored 2^7 up, end at 2^16), and then the tile
// is gone through the careful way from there on: maximum, reference moved to
// it or just above (a whole power of two from the old one), O and what is
// written of the tile rescaled.  (First references of whole powers of two, so
// that every move is one, round the largest weight, which is 1 otherwise: 16
// prompts 2.35e-3 from the exact result instead of 2.11e-3.  Each item's first
// tile searched whole: 16 prompts 341 us instead of 312.)
//
// A key that a row does not see has weight 0, but 0 x NaN is NaN: in tiles
// that some row does not see whole, V rows outside the item's keys (stale
// pages) are zeroed and non-finite V elements of the others taken out before
// the product; if there were any, the rows that see them get them added back
// from global memory at the end of the item.
//
// Bound by the row warps: a tile pair's products take 1024 tensor cycles, its
// 32,768 exponentials 2048 cycles of the special-function units, and the row
// warps need about 3000: two of them a scheduler use 41 % of its issue slots, and
// what lies between are the fixed latencies of dependent instructions (2.3 cycles
// an instruction) and waits for TMEM loads (2.0); instruction fetch is 0.2 in this
// form, and what made earlier ones slower (the weights' loop
// unrolled by two: 16 prompts 338 -> 393 us).  An item costs about 6000 cycles more,
// which the shares count as 256 keys (128, 384, 640: 16 prompts 340, 328, 360 us
// where it is 311; a window of 128 or 40 chunks of 100 alike).  At head size 128 the two S
// buffers leave each row tile waiting for its products (2000 of 4300 cycles a
// tile; S in halves of 64 keys or the row tiles in turn: no better).  Measured:
// 16 prompts of 100-2048 tokens, 64 query over 8 KV heads of 64, bf16: 311 us,
// 513 TFLOP/s; four of 1500-4000 with a window of 128: 146 us, 1.5 TB/s; one of
// 8191, 32 over 8 heads of 128, f16: 605 us, 910 TFLOP/s (cuBLAS bf16 1669).
#include <algorithm>
#include <climits>

#include "attention_half.cuh"
#include "launch.cuh"

namespace pc {

namespace {

constexpr int RW_R = 256, RW_KT = 128, RW_OV = 256, RW_MINK = 256, RW_THREADS = 384;
constexpr float RW_GROW = 8.0f;       // log2 of the growth that moves the reference in the careful way
constexpr float RW_LIMIT = 16384.0f;  // what 32 weights of a row may sum up to before it is taken
constexpr float RW_FAR = 8388608.0f;  // references from here on (2^23): see far_scores

template <int HD>
struct RowsCfg {
    static constexpr int PANELS = HD / 64;        // 64-column (128-byte) panels of a row
    static constexpr int TILE = PANELS * 16384;   // bytes of 128 rows
    static constexpr int STAGES = HD == 64 ? 3 : 2;
    static constexpr int QB = HD == 64 ? 2 : 1;   // Q buffers
    static constexpr int NB = HD == 64 ? 3 : 2;   // S / P buffers in TMEM, 128 columns each
    static constexpr int O0 = NB * 128;
    static constexpr size_t SMEM = 1024 + (size_t)TILE * (2 * QB + 2 * STAGES);
    static constexpr int PART = RW_R * (HD + 2);
};

struct KeySteps {
    int lo, hi;
};

// An item of the block's share as all roles read it: warp 8 walks the share
// (attention_plan.cuh) and leaves one after another, an item ahead of its
// tiles.  (With the walk in every role its 64-bit arithmetic stood in each
// one's way at every item, and five times in the instruction cache.)
struct ItemDesc {
    ItemGeo g;
    int b, kvh, q0, p0;  // request, KV head, its first row, that row's position
    int tl, th;          // this block's tiles; none: the share is done
    int k0, k1;          // blocks that share the item; k0 < 0: it is whole
};
constexpr int RW_ITEMS = 4;  // descriptors in the ring

struct RowsBars {
    uint64_t q_full[4], q_free[4], s_full[3], p_full[3], o_full[4];
    uint64_t k_full[3], k_free[3], v_full[3], v_free[3], v_fixed[3], d_full[RW_ITEMS], d_free[RW_ITEMS], both, drain[2];
};

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
// Waits for this thread's TMEM loads; the values pass through it, so that no
// use of them is scheduled before.
__device__ __forceinline__ void tmem_ld_wait16(uint32_t *v) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), 
                   "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_ld_wait32(uint32_t *v) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                   "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]),
                   "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]),
                   "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31])
                 :
                 : "memory");
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

// Whether a phase is complete, without waiting
__device__ __forceinline__ bool mbar_test(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}

// One lane of the warp
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
// The same value in all lanes, known as such to the compiler
template <typename V>
__device__ __forceinline__ V uniform(V v) { return __shfl_sync(0xffffffffu, v, 0); }

// Bits y of 32 with lo < y <= hi
__device__ __forceinline__ uint32_t seen_bits(int lo, int hi) {
    const uint32_t up = hi >= 31 ? ~0u : hi < 0 ? 0u : (2u << hi) - 1u;
    const uint32_t dn = lo >= 31 ? ~0u : lo < 0 ? 0u : (2u << lo) - 1u;
    return up & ~dn;
}

// -inf in the place of scores that are not seen
__device__ __forceinline__ void hide(uint32_t (&sv)[32], uint32_t seen) {
#pragma unroll
    for (int y = 0; y < 32; ++y)
        if (!(seen >> y & 1u)) sv[y] = 0xFF800000u;
}

__device__ __forceinline__ uint64_t f2_ex2(uint64_t v) { return f2_pack(ex2(f2_lo(v)), ex2(f2_hi(v))); }
// the largest of three, NaN if one of them is
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// A tile of keys (the block's tile t of an item) that some row of the item
// does not see whole
__device__ __forceinline__ bool rows_masked(const ItemGeo &g, int t, int window) {
    const int k0 = (g.t0 + t) * RW_KT;
    return k0 + RW_KT - 1 > g.pmin || (window > 0 && k0 < g.pmax - window + 1);
}

// What an item hardly ever or seldom needs is in functions of their own: the
// row warps' loops share the instruction cache with all that is inlined (16
// prompts to 2k took 7 % less with the waits' second half out alone).

// Adds what masked tiles hold of non-finite V to the O of a row that sees it.
template <typename T, int HD>
__device__ __noinline__ void add_odd(const AttnOp &a, const ItemDesc w, int pos, uint32_t ot) {
    const ItemGeo &g = w.g;
    const T *vb = reinterpret_cast<const T *>(a.v) + (int64_t)w.kvh * a.vs[2];
#pragma unroll 1
    for (int x = 0; x < HD; x += 16) {
        uint32_t o[16];
        tmem_ld16(ot + x, o);
        tmem_ld_wait16(o);
        for (int key = (g.t0 + w.tl) * RW_KT; key < (g.t0 + w.th) * RW_KT; ++key) {
            if (key < g.kb || key >= g.ke || key > pos || (a.window > 0 && key <= pos - a.window) ||
                !rows_masked(g, key / RW_KT - g.t0, a.window))
                continue;
            const T *vp = vb + (int64_t)(w.q0 + key) * a.vs[1];
            if (a.table) {
                const int page = a.table[(int64_t)w.b * a.max_pages + key / a.page_size];
                if (page < 0 || page >= a.n_pages) continue;
                vp = vb + page * a.vs[0] + (int64_t)(key % a.page_size) * a.vs[1];
            }
#pragma unroll
            for (int d = 0; d < 16; ++d) {
                const float v = x + d < a.D ? Half16<T>::up(reinterpret_cast<const unsigned short *>(vp)[x + d]) : 0.0f;
                if (!isfinite(v)) o[d] = __float_as_uint(__fadd_rn(__uint_as_float(o[d]), v));
            }
        }
        __syncwarp();
        tmem_st16(ot + x, o);
    }
    tmem_st_wait();
}

// A row's O, reference and sum to the workspace (`mine`: its place in the block's record).
template <int HD>
__device__ __noinline__ void leave_part(float *mine, uint32_t ot, float m, float l) {
#pragma unroll 1
    for (int x = 0; x < HD; x += 16) {
        uint32_t o[16];
        tmem_ld16(ot + x, o);
        tmem_ld_wait16(o);
#pragma unroll
        for (int d = 0; d < 16; ++d) __stcg(mine + (x + d) * RW_R, __uint_as_float(o[d]));
    }
    __stcg(mine + HD * RW_R, m);
    __stcg(mine + (HD + 1) * RW_R, l);
}

// The parts of blocks k0 .. k1 in block order: O into TMEM, (reference, sum).
template <int HD>
__device__ __noinline__ float2 join_parts(const float *part, int k0, int k1, uint32_t ot) {
    auto of = [&](int k) { return part + ((int64_t)k * 2 + (k == k0)) * RowsCfg<HD>::PART; };
    float mm = -INFINITY, l = 0.0f;
#pragma unroll 4
    for (int k = k0; k <= k1; ++k) mm = fmaxf(mm, __ldcg(of(k) + HD * RW_R));
    const float ms = mm == -INFINITY ? 0.0f : mm;
#pragma unroll 4
    for (int k = k0; k <= k1; ++k)
        l = __fmaf_rn(__ldcg(of(k) + (HD + 1) * RW_R), ex2(__fsub_rn(__ldcg(of(k) + HD * RW_R), ms)), l);
#pragma unroll 1
    for (int x = 0; x < HD; x += 16) {
        float o[16];
#pragma unroll
        for (int d = 0; d < 16; ++d) o[d] = 0.0f;
#pragma unroll 2
        for (int k = k0; k <= k1; ++k) {
            const float *p = of(k);
            const float e = ex2(__fsub_rn(__ldcg(p + HD * RW_R), ms));
#pragma unroll
            for (int d = 0; d < 16; ++d) o[d] = __fmaf_rn(__ldcg(p + (x + d) * RW_R), e, o[d]);
        }
        uint32_t ov[16];
#pragma unroll
        for (int d = 0; d < 16; ++d) ov[d] = __float_as_uint(o[d]);
        __syncwarp();
        tmem_st16(ot + x, ov);
    }
    tmem_st_wait();
    return make_float2(mm, l);
}

// A row's O (`cols` columns) times corr
static __device__ __noinline__ void scale_o(uint32_t ot, int cols, float corr) {
#pragma unroll 1
    for (int x = 0; x < cols; x += 16) {
        uint32_t ov[16];
        tmem_ld16(ot + x, ov);
        tmem_ld_wait16(ov);
#pragma unroll
        for (int y = 0; y < 16; ++y) ov[y] = __float_as_uint(__fmul_rn(__uint_as_float(ov[y]), corr));
        tmem_st16(ot + x, ov);
    }
    tmem_st_wait();
}
// A row's scores from column `from` on in the place of themselves, as powers of
// two beside its reference.  Far from 0 score x c - reference, rounded once, is
// off by as much as the reference is from the maximum's exact product (32
// powers of two at f16's lowest value, any number at bf16's): here the product
// is rounded first, as the reference was, and the maximum's own weight is 1.
static __device__ __noinline__ void far_scores(uint32_t st, int from, float c, float ref) {
#pragma unroll 1
    for (int x = from; x < RW_KT; x += 16) {
        uint32_t v[16];
        tmem_ld16(st + x, v);
        tmem_ld_wait16(v);
#pragma unroll
        for (int y = 0; y < 16; ++y) v[y] = __float_as_uint(__fsub_rn(__fmul_rn(__uint_as_float(v[y]), c), ref));
        tmem_st16(st + x, v);
    }
    tmem_st_wait();
}
// Written weights (`cols` columns of two) times corr: exact, it is a power of two
template <typename T>
__device__ __noinline__ void scale_p(uint32_t st, int cols, float corr) {
    using E = Half16<T>;
    tmem_st_wait();  // this thread's own stores of them: without the wait a load may come before them
#pragma unroll 1
    for (int x = 0; x < cols; x += 16) {
        uint32_t ov[16];
        tmem_ld16(st + x, ov);
        tmem_ld_wait16(ov);
#pragma unroll
        for (int y = 0; y < 16; ++y)
            ov[y] = E::pack(__fmul_rn(E::up(ov[y] & 0xFFFFu), corr), __fmul_rn(E::up(ov[y] >> 16), corr));
        tmem_st16(st + x, ov);
    }
    tmem_st_wait();
}

template <typename T, int HD>
__global__ void __launch_bounds__(RW_THREADS, 1)
    attn_rows_kernel(const __grid_constant__ AttnOp a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                     const __grid_constant__ CUtensorMap qmap, const int box, const bool qtma) {
    using C = RowsCfg<HD>;
    using E = Half16<T>;
    constexpr int NS = C::STAGES, QB = C::QB;
    extern __shared__ uint8_t rows_smem_raw[];
    uint8_t *smem = rows_smem_raw + (1024 - (smem_u32(rows_smem_raw) & 1023)) % 1024;
    uint8_t *qs = smem, *ks = qs + 2 * C::QB * C::TILE, *vs = ks + NS * C::TILE;
    __shared__ PlanScratch<RW_THREADS> sc;
    __shared__ RowsBars bar;
    __shared__ ItemDesc items[RW_ITEMS];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int dead;
    __shared__ int lastf;
    __shared__ volatile int odd[4];  // [i % 4] = i + 1: non-finite V in a masked tile of the block's item i
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (a.min_q > 1 && nothing_to_take(a.cu, a.B, a.T, a.G, a.min_q, a.max_q)) {
        pdl_trigger();
        pdl_wait();
        return;
    }
    if (tid == 0) {
        for (int t = 0; t < 4; ++t) {
            mbar_init(&bar.q_full[t], 1);
            mbar_init(&bar.q_free[t], 1);
        }
        for (int b = 0; b < C::NB; ++b) {
            mbar_init(&bar.s_full[b], 1);
            mbar_init(&bar.p_full[b], 128);
        }
        for (int i = 0; i < 4; ++i) mbar_init(&bar.o_full[i], 1);
        for (int s = 0; s < NS; ++s) {
            mbar_init(&bar.k_full[s], 1);
            mbar_init(&bar.k_free[s], 1);
            mbar_init(&bar.v_full[s], 1);
            mbar_init(&bar.v_free[s], 1);
            mbar_init(&bar.v_fixed[s], 32);
        }
        for (int i = 0; i < RW_ITEMS; ++i) {
            mbar_init(&bar.d_full[i], 1);
            mbar_init(&bar.d_free[i], 11);  // the warps that read it
        }
        mbar_init(&bar.both, 256);
        mbar_init(&bar.drain[0], 1);
        mbar_init(&bar.drain[1], 1);
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

    auto wait = [&](uint64_t *b, uint32_t parity) -> bool { return bounded_wait(b, parity, &dead, a.err); };
    auto wait_all = [&](uint64_t *b, uint32_t parity) -> bool { return __all_sync(0xffffffffu, wait(b, parity)); };
    // Item `i` of the share; false if the share is done (or a wait gave up: ok).
    auto take = [&](int i, ItemDesc &d, bool &ok) -> bool {
        if (!(ok = wait_all(&bar.d_full[i % RW_ITEMS], (i / RW_ITEMS) & 1))) return false;
        d = items[i % RW_ITEMS];
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.d_free[i % RW_ITEMS]);
        return d.th > d.tl;
    };
    // the steps of 16 keys of a tile that hold keys of the item (one at least)
    auto key_steps = [&](const ItemGeo &g, int t) -> KeySteps {
        const int k0 = (g.t0 + t) * RW_KT;
        KeySteps k;
        k.lo = max(g.kb - k0, 0) / 16;
        k.hi = min(max((g.ke - k0 + 15) / 16, k.lo + 1), RW_KT / 16);
        return k;
    };
    // after a failure: products in flight end before TMEM is freed
    auto drain = [&](bool ok, uint64_t *b) {
        if (!ok && elect_one()) {
            tc_commit(b);
            const long long t0 = clock64();
            while (!mbar_try_wait(b, 0))
                if (clock64() - t0 > ATTN_WAIT_CLOCKS) break;
        }
        __syncwarp();
    };
    if (sc.share.n == 0) {
        // no share
    } else if (warp == 8) {
        // ---- items; Q, K and V tiles ----
        PlanWalk<RW_R, RW_KT> walk(a, sc.share);
        ItemDesc w, next;
        int it = 0, item = 0, left = 0, fills[2] = {0, 0};
        bool ok = true, more = walk.load();
        auto leave = [&]() {  // the item of the walk, or the end, for the other warps
            next.th = next.tl = 0;
            if (more) {
                next.g = walk.g;
                next.b = walk.b;
                next.kvh = walk.kvh;
                next.q0 = walk.s.q0;
                next.p0 = walk.s.p0;
                next.tl = walk.tl;
                next.th = walk.th;
                next.k0 = -1;
                if (!walk.whole()) {
                    const CutItem c = cut_item(walk);
                    next.k0 = c.k0;
                    next.k1 = c.k1;
                }
            }
            if (left >= RW_ITEMS) ok = ok && wait_all(&bar.d_free[left % RW_ITEMS], (left / RW_ITEMS - 1) & 1);
            if (lane == 0) {
                items[left % RW_ITEMS] = next;
                mbar_arrive(&bar.d_full[left % RW_ITEMS]);
            }
            ++left;
            __syncwarp();
        };
        auto load_q = [&]() {
            for (int t = 0; t < 2; ++t) {
                const int b = item % QB * 2 + t;
                if (item >= QB && !(ok = wait_all(&bar.q_free[b], (item / QB - 1) & 1))) return;
                if (lane == 0) mbar_arrive_expect_tx(&bar.q_full[b], C::TILE);
                __syncwarp();
                if (lane < C::PANELS)
                    tma_load_3d(qs + b * C::TILE + lane * 16384, &qmap, &bar.q_full[b], lane * 64, w.kvh * a.G,
                                w.q0 + div_g(a, w.g.r0 + t * 128));
                __syncwarp();
            }
        };
        leave();
        for (; more && ok; ++item) {
            w = next;
            more = walk.next();
            leave();
            if (!ok) break;
            if (qtma && QB > 1) load_q();
            for (int t = w.tl; t < w.th && ok; ++t, ++it) {
                // one Q buffer: the item's first K and V need not wait for it
                if (qtma && QB == 1 && t == w.tl + 1) load_q();
                const int s = it % NS;
                const uint32_t ph = (it / NS) & 1;
                const int k0 = (w.g.t0 + t) * RW_KT;
                // boxes that hold keys of the item
                const int lo = max(w.g.kb - k0, 0) / box, hi = (min(w.g.ke - k0, RW_KT) + box - 1) / box;
                const int nb = max(hi - lo, 0);
                for (int kv = 0; kv < 2 && ok; ++kv) {
                    uint64_t *full = kv ? &bar.v_full[s] : &bar.k_full[s];
                    ok = wait_all(kv ? &bar.v_free[s] : &bar.k_free[s], ph ^ 1);
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
                            const int page = a.table[(int64_t)w.b * a.max_pages + key / a.page_size];
                            tma_load_4d(d, map, full, p * 64, key % a.page_size, w.kvh, page);
                        } else {
                            tma_load_3d(d, map, full, p * 64, w.q0 + key, w.kvh);
                        }
                    }
                    __syncwarp();
                }
            }
            if (qtma && QB == 1 && w.th == w.tl + 1 && ok) load_q();
        }
        if (!ok && lane == 0)  // copies in flight land before the block ends
            for (int s = 0; s < NS; ++s)
                for (int kv = 0; kv < 2; ++kv) {
                    const int n = (fills[kv] - s + NS - 1) / NS;  // fills of this stage
                    const long long t0 = clock64();
                    if (n > 0)
                        while (!mbar_try_wait(kv ? &bar.v_full[s] : &bar.k_full[s], (n - 1) & 1))
                            if (clock64() - t0 > ATTN_WAIT_CLOCKS) break;
                }
    } else if (warp == 9) {
        // ---- S = Q K^T ----
        // The whole warp walks, one elected lane issues: what the instructions
        // take stays in uniform registers.  A product's issue holds the warp
        // for as long as the tensor core takes it, so the other products have
        // their own warp, and each prepares its next while the other's run.
        constexpr uint32_t ID = (1u << 4) | (E::FMT << 7) | (E::FMT << 10) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
        const uint32_t tmu = uniform(tm);
        const uint64_t qd0 = sw128_desc(qs), kd0 = sw128_desc(ks);
        ItemDesc w;
        int n = 0, sbuf = 0, qbuf = 0, kst = 0;
        uint32_t qph = 0, kph = 0;
        bool ok = true;
        for (int item = 0; ok && take(item, w, ok); ++item) {
            const int left = uniform(w.th - w.tl);
            for (int j = 0; j < left && ok; ++j) {
#pragma unroll
                for (int t = 0; t < 2; ++t, ++n) {
                    if (j == 0 && !(ok = wait_all(&bar.q_full[qbuf * 2 + t], qph))) break;
                    if (t == 0 && !(ok = wait_all(&bar.k_full[kst], kph))) break;
                    // the buffer's last P has met its V
                    if (n >= C::NB && !(ok = wait_all(&bar.o_full[(n - C::NB) & 3], (n - C::NB) >> 2 & 1))) break;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint64_t qd = qd0 + (qbuf * 2 + t) * (C::TILE >> 4), kd = kd0 + kst * (C::TILE >> 4);
#pragma unroll
                        for (int k = 0; k < HD / 16; ++k) {
                            const int off = (k / 4) * (16384 >> 4) + (k % 4) * 2;
                            tc_mma_f16(tmu + sbuf * 128, qd + off, kd + off, ID, k > 0);
                        }
                        tc_commit(&bar.s_full[sbuf]);
                        if (j + 1 == left) tc_commit(&bar.q_free[qbuf * 2 + t]);
                        if (t == 1) tc_commit(&bar.k_free[kst]);
                    }
                    __syncwarp();
                    if (++sbuf == C::NB) sbuf = 0;
                }
                if (++kst == NS) {
                    kst = 0;
                    kph ^= 1;
                }
            }
            if (++qbuf == QB) {
                qbuf = 0;
                qph ^= 1;
            }
        }
        drain(ok, &bar.drain[0]);
    } else if (warp == 11) {
        // ---- O += P V ----
        constexpr uint32_t ID = (1u << 4) | (E::FMT << 7) | (E::FMT << 10) | (1u << 16) | (((uint32_t)HD >> 3) << 17) |
                                ((128u >> 4) << 24);
        const uint32_t tmu = uniform(tm);
        const uint64_t vd0 = sw128_desc_n(smem_u32(vs), 16384);
        ItemDesc w;
        int n = 0, pbuf = 0, vst = 0;
        uint32_t pph = 0, vph = 0;
        bool ok = true;
        for (int item = 0; ok && take(item, w, ok); ++item) {
            const int left = uniform(w.th - w.tl);
            for (int j = 0; j < left && ok; ++j) {
                const KeySteps ks_ = key_steps(w.g, w.tl + j);
                const int k0 = uniform(ks_.lo), k1 = uniform(ks_.hi);
                // V in order implies V there
                if (!(ok = wait_all(&bar.v_fixed[vst], vph))) break;
#pragma unroll
                for (int t = 0; t < 2; ++t, ++n) {
                    if (!(ok = wait_all(&bar.p_full[pbuf], pph))) break;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint64_t vd = vd0 + vst * (C::TILE >> 4);
#pragma unroll
                        for (int k = 0; k < RW_KT / 16; ++k)
                            if (k >= k0 && k < k1)
                                tc_mma_ts(tmu + C::O0 + t * HD, tmu + pbuf * 128 + k * 8, vd + k * (2048 >> 4), ID,
                                          j > 0 || k > k0);
                        tc_commit(&bar.o_full[n & 3]);
                        if (t == 1) tc_commit(&bar.v_free[vst]);
                    }
                    __syncwarp();
                    if (++pbuf == C::NB) {
                        pbuf = 0;
                        pph ^= 1;
                    }
                }
                if (++vst == NS) {
                    vst = 0;
                    vph ^= 1;
                }
            }
        }
        drain(ok, &bar.drain[1]);
    } else if (warp == 10) {
        // ---- Q rows; V rows of masked tiles ----
        ItemDesc w, wn = {};                               // the item at hand, the next one
        constexpr int CH = C::PANELS * 8, STEP = 32 / CH;  // 16-byte pieces of a row, rows at a time
        const int c = lane % CH;
        const bool col = c * 8 < a.D;
        auto load_q = [&](int item) {
            const T *q = reinterpret_cast<const T *>(a.q) + (int64_t)wn.q0 * a.qs[0] + (int64_t)wn.kvh * a.G * a.qs[1] + c * 8;
            for (int t = 0; t < 2; ++t) {
                const uint32_t dst = smem_u32(qs + (item % QB * 2 + t) * C::TILE) + (c / 8) * 16384;
#pragma unroll 4
                for (int r = lane / CH; r < 128; r += STEP) {
                    const int f = wn.g.r0 + t * 128 + r;
                    const bool in = f < wn.g.r1 && col;
                    const int tok = div_g(a, f);
                    const T *src = in ? q + (int64_t)tok * a.qs[0] + (int64_t)(f - tok * a.G) * a.qs[1]
                                      : reinterpret_cast<const T *>(a.q);
                    cp_async16_fill(dst + r * 128 + (((c % 8) ^ (r & 7)) << 4), src, in ? 16 : 0);
                }
                cp_async_commit();
            }
            cp_async_wait<0>();
            fence_async_smem();
            __syncwarp();
            if (lane < 2) mbar_arrive(&bar.q_full[item % QB * 2 + lane]);
        };
        int it = 0, item = 0, loaded = 0;  // key tiles and items done, items whose Q is loaded
        bool ok = true, qmore = take(0, wn, ok);
        auto q_turn = [&](bool block) -> bool {  // the next item's Q, once its buffer is free
            if (qtma || !qmore || loaded > item) return true;
            for (int t = 0; t < 2 && loaded >= QB; ++t) {
                uint64_t *b = &bar.q_free[loaded % QB * 2 + t];
                const uint32_t ph = (loaded / QB - 1) & 1;
                if (block) {
                    if (!wait_all(b, ph)) return false;
                } else if (!__all_sync(0xffffffffu, mbar_test(b, ph))) {
                    return true;
                }
            }
            load_q(loaded++);
            return true;
        };
        // `item`: the one whose Q comes next, wn
        ok = ok && q_turn(true);
        while (qmore && ok) {
            w = wn;
            const int at = item++;
            qmore = take(item, wn, ok);
            for (int t = w.tl; t < w.th && ok; ++t, ++it) {
                const int s = it % NS;
                if (!(ok = q_turn(false)) || !(ok = wait_all(&bar.v_full[s], (it / NS) & 1))) break;
                if (rows_masked(w.g, t, a.window)) {
                    const int k0 = (w.g.t0 + t) * RW_KT;
                    const KeySteps st = key_steps(w.g, t);
                    uint8_t *v = vs + s * C::TILE;
                    const int lo = st.lo * 16, hi = st.hi * 16;  // rows that the products read
                    const int kb = min(max(w.g.kb - k0, lo), hi), ke = min(max(w.g.ke - k0, kb), hi);  // those of the item's keys
                    // of those, the ones that every row sees
                    const int a0 = min(max(a.window > 0 ? w.g.pmax - a.window + 1 - k0 : kb, kb), ke);
                    const int b0 = min(max(w.g.pmin + 1 - k0, a0), ke);
                    auto clear = [&](int from, int to) {
                        for (int r = from + lane / 8; r < to; r += 4)
#pragma unroll
                            for (int p = 0; p < C::PANELS; ++p)
                                *(reinterpret_cast<uint4 *>(v + p * 16384 + r * 128) + lane % 8) = make_uint4(0, 0, 0, 0);
                    };
                    clear(lo, kb);
                    clear(ke, hi);
                    // is an exponent all ones: adding its lowest bit carries into the sign's place
                    uint32_t acc = 0;
                    auto look = [&](int from, int to) {
#pragma unroll 1
                        for (int r = from + lane / 8; r < to; r += 4)
#pragma unroll
                            for (int p = 0; p < C::PANELS; ++p) {
                                const uint4 x = *(reinterpret_cast<const uint4 *>(v + p * 16384 + r * 128) + lane % 8);
                                constexpr uint32_t M = E::EXP * 0x10001u, ONE = (E::EXP & (0u - E::EXP)) * 0x10001u;
                                acc |= (x.x & M) + ONE | (x.y & M) + ONE | (x.z & M) + ONE | (x.w & M) + ONE;
                            }
                    };
                    look(kb, a0);
                    look(b0, ke);
                    const bool bad = __any_sync(0xffffffffu, (acc & 0x80008000u) != 0);
                    if (bad)
                        for (int r = kb + lane / 8; r < ke; r += 4) {
                            if (r >= a0 && r < b0) continue;
#pragma unroll 1
                            for (int p = 0; p < C::PANELS * 4; ++p) {
                                uint32_t *q = reinterpret_cast<uint32_t *>(v + p / 4 * 16384 + r * 128 + lane % 8 * 16) + p % 4;
                                uint32_t x = *q;
                                if ((x & E::EXP) == E::EXP) x &= 0xFFFF0000u;
                                if ((x >> 16 & E::EXP) == E::EXP) x &= 0x0000FFFFu;
                                *q = x;
                            }
                        }
                    if (bad && lane == 0) odd[at & 3] = at + 1;
                    fence_async_smem();
                }
                mbar_arrive(&bar.v_fixed[s]);
            }
            ok = ok && q_turn(true);
        }
    } else {
        // ---- softmax and output of row tile t ----
        const int t = warp >> 2, r = tid & 127;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21, ot = tm + lanes + C::O0 + t * HD;
        const float c = __fmul_rn(a.scale, 1.4426950408889634f);
        ItemDesc w;
        int it = 0, item = 0;  // key tiles and items done
        uint32_t both_n = 0;
        bool ok = true;
        auto both = [&]() -> bool {  // the two row tiles' threads meet
            mbar_arrive(&bar.both);
            return wait_all(&bar.both, both_n++ & 1);
        };
        // O has all products so far.  A row tile's products take two barriers
        // in turn: a warp can be two tiles ahead of the slowest of its row
        // tile, and the phases of one barrier would look alike to it.
        auto o_done = [&]() -> bool {
            const bool done = wait_all(&bar.o_full[((it - 1) & 1) * 2 + t], (it - 1) >> 1 & 1);
            tc_fence_after();
            return done;
        };
        for (; ok && take(item, w, ok); ++item) {
            const ItemGeo &g = w.g;
            const int f = g.r0 + t * 128 + r, tok = div_g(a, f);
            const int pos = f < g.r1 ? w.p0 + tok : -1;
            const float sink = a.sinks && f < g.r1 ? a.sinks[w.kvh * a.G + f - tok * a.G] : 0.0f;
            // positions of the warp's rows, lowest and highest
            const int plo = __reduce_min_sync(0xffffffffu, pos < 0 && f >= g.r1 ? INT_MAX : pos),
                      phi = __reduce_max_sync(0xffffffffu, pos);
            float mr = f < g.r1 ? -INFINITY : 0.0f, l = 0.0f;  // reference in powers of two, sum
            for (int j = w.tl; j < w.th; ++j, ++it) {
                const int n = 2 * it + t, b = n % C::NB;
                const uint32_t st = tm + lanes + b * 128;
                ok = wait_all(&bar.s_full[b], (n / C::NB) & 1);
                if (!ok) break;
                tc_fence_after();
                const int k0 = (g.t0 + j) * RW_KT, hi = pos - k0, lo = a.window > 0 ? hi - a.window : -1;  // sees lo < x <= hi
                // of the four groups of 32 keys, those that some row of the warp sees, and those that all see
                const int x0 = a.window > 0 ? max((min(plo, phi) - a.window - k0 + 1) >> 5, 0) : 0;
                const int x1 = phi < k0 ? -1 : min((phi - k0) >> 5, 3);
                auto all_see = [&](int x) { return 32 * x + 31 <= plo - k0 && (a.window == 0 || 32 * x > phi - a.window - k0); };
                uint32_t sv[32];
                uint64_t sum[2] = {0, 0};
                const uint64_t c2 = f2_pack(c, c);
                int xs = 0;  // the group from which on the careful way goes
                bool grown = false;
                if (all_see(0) && all_see(3) && (HD == 64 || __all_sync(0xffffffffu, fabsf(mr) < RW_FAR))) {
                    // No look at the maximum first: the weights are taken against the reference as it is, and the
                    // sum of a group tells whether one has grown too large for it (or is no number).
                    tmem_ld32(st, sv);
                    if (HD == 64 && __any_sync(0xffffffffu, mr == -INFINITY)) {  // none yet: the first group's maximum
                        float mx = -INFINITY;
                        tmem_ld_wait32(sv);
#pragma unroll
                        for (int y = 0; y < 16; ++y) mx = max3(mx, __uint_as_float(sv[2 * y]), __uint_as_float(sv[2 * y + 1]));
                        if (mr == -INFINITY) mr = mx < INFINITY ? __fmul_rn(mx, c) : NAN;
                    }
                    const float nmc = __fsub_rn(E::BIAS, mr);
                    const uint64_t nmc2 = f2_pack(nmc, nmc);
                    if (HD == 128 || __all_sync(0xffffffffu, fabsf(mr) < RW_FAR))  // else none but -inf so far, or far off
#pragma unroll(HD == 128 ? 2 : 1)
                    for (; xs < 4; ++xs) {
                        uint64_t v[16], part[2] = {0, 0};
                        uint32_t pk[16];
                        tmem_ld_wait32(sv);
#pragma unroll
                        for (int y = 0; y < 16; ++y) v[y] = f2_fma(f2_pack_bits(sv[2 * y], sv[2 * y + 1]), c2, nmc2);
                        if (xs < 3) tmem_ld32(st + 32 * xs + 32, sv);
#pragma unroll
                        for (int y = 0; y < 16; ++y) {
                            const uint64_t p = f2_ex2(v[y]);
                            part[y & 1] = f2_add(part[y & 1], p);
                            pk[y] = E::pack(f2_lo(p), f2_hi(p));
                        }
                        part[0] = f2_add(part[0], part[1]);
                        if (__any_sync(0xffffffffu, !(__fadd_rn(f2_lo(part[0]), f2_hi(part[0])) <= RW_LIMIT))) {
                            grown = true;
                            break;
                        }
                        sum[xs & 1] = f2_add(sum[xs & 1], part[0]);
                        tmem_st16(st + 16 * xs, pk);  // over columns read by now
                    }
                    tmem_ld_wait32(sv);
                }
                if (xs < 4) {
                    // the careful way, from group xs on: tiles that some row does not see whole; the maximum is searched
                    // for where a row has no reference yet, or its own has been outgrown
                    bool search = grown || !__all_sync(0xffffffffu, fabsf(mr) < RW_FAR);
                    do {
                        if (search) {
                            float mx = -INFINITY;
#pragma unroll 1
                            for (int x = max(x0, xs); x <= x1; ++x) {
                                tmem_ld32(st + 32 * x, sv);
                                tmem_ld_wait32(sv);
                                if (!all_see(x)) hide(sv, seen_bits(lo - 32 * x, hi - 32 * x));
#pragma unroll
                                for (int y = 0; y < 16; ++y) mx = max3(mx, __uint_as_float(sv[2 * y]), __uint_as_float(sv[2 * y + 1]));
                            }
                            // move the reference of rows that have none, or whose maximum has grown: by a power of two, or
                            // where nothing is left of what was before, to the maximum itself (the old reference plus a
                            // large growth is rounded to the old one's spacing: 64 after scores of f16's lowest value)
                            const float top = __fmul_rn(mx, c), grow = ceilf(__fsub_rn(top, mr));
                            float corr = 1.0f;
                            if (mr == -INFINITY) {
                                mr = top;
                            } else if (grow > (grown ? 0.0f : RW_GROW)) {
                                mr = grow < 126.0f ? __fadd_rn(mr, grow) : top;
                                corr = grow < 126.0f ? __int_as_float((127 - (int)grow) << 23) : 0.0f;
                            }
                            if (!(mx < INFINITY)) mr = NAN;  // an infinite or NaN score: so are the row's weights
                            if (__any_sync(0xffffffffu, corr != 1.0f)) {
                                l = __fmul_rn(l, corr);
                                sum[0] = f2_mul(sum[0], f2_pack(corr, corr));
                                sum[1] = f2_mul(sum[1], f2_pack(corr, corr));
                                if (j > w.tl) {  // O of the tiles before
                                    ok = o_done();
                                    if (!ok) break;
                                    scale_o(ot, HD, corr);
                                }
                                if (xs) scale_p<T>(st, 16 * xs, corr);
                            }
                        }
                        const float ref = mr == -INFINITY ? 0.0f : mr;
                        const bool far = __any_sync(0xffffffffu, fabsf(ref) >= RW_FAR);  // then searched: all that is left follows
                        if (far) far_scores(st, 32 * xs, c, ref);
                        const float nmc = far ? E::BIAS : __fsub_rn(E::BIAS, ref), cc = far ? 1.0f : c;
                        const uint64_t nmc2 = f2_pack(nmc, nmc), cc2 = f2_pack(cc, cc);
#pragma unroll 1
                        for (; xs < 4; ++xs) {
                            uint32_t pk[16];
                            if (xs >= x0 && xs <= x1) {
                                uint64_t part[2] = {0, 0};
                                tmem_ld32(st + 32 * xs, sv);
                                const uint32_t seen = seen_bits(lo - 32 * xs, hi - 32 * xs);
                                tmem_ld_wait32(sv);
                                hide(sv, seen);
#pragma unroll
                                for (int y = 0; y < 16; ++y) {
                                    const uint64_t p = f2_ex2(f2_fma(f2_pack_bits(sv[2 * y], sv[2 * y + 1]), cc2, nmc2));
                                    part[y & 1] = f2_add(part[y & 1], p);
                                    pk[y] = E::pack(f2_lo(p), f2_hi(p));
                                }
                                part[0] = f2_add(part[0], part[1]);
                                if (!search && __any_sync(0xffffffffu, !(__fadd_rn(f2_lo(part[0]), f2_hi(part[0])) <= RW_LIMIT))) {
                                    search = grown = true;
                                    break;
                                }
                                sum[0] = f2_add(sum[0], part[0]);
                            } else {
#pragma unroll
                                for (int y = 0; y < 16; ++y) pk[y] = 0;
                            }
                            tmem_st16(st + 16 * xs, pk);
                        }
                    } while (xs < 4);
                    if (!ok) break;
                }
                tmem_st_wait();
                tc_fence_before();
                mbar_arrive(&bar.p_full[b]);
                const uint64_t both_sums = f2_add(sum[0], sum[1]);
                l = __fadd_rn(l, __fadd_rn(f2_lo(both_sums), f2_hi(both_sums)));
            }
            if (!ok || !(ok = o_done())) break;
            float mref = mr;
            if (odd[item & 3] == item + 1) add_odd<T, HD>(a, w, pos, ot);
            if (w.k0 >= 0) {
                leave_part<HD>(a.part + ((int64_t)blockIdx.x * 2 + (w.tl == 0)) * C::PART + tid, ot, mref, l);
                __threadfence();
                if (!(ok = both())) break;
                if (tid == 0) {
                    lastf = atomicAdd(a.ticket + w.k0, 1u) == (unsigned)(w.k1 - w.k0);
                    if (lastf) a.ticket[w.k0] = 0u;
                }
                if (!(ok = both())) break;
                if (!lastf) continue;
                __threadfence();
                const float2 ml = join_parts<HD>(a.part + tid, w.k0, w.k1, ot);
                mref = ml.x;
                l = ml.y;
            }
            const float inv = f < g.r1 ? row_factor<E>(mref, l, a.sinks != nullptr, __fmul_rn(sink, 1.4426950408889634f)) : 0.0f;
            T *out = reinterpret_cast<T *>(a.out) + (int64_t)(w.q0 + tok) * a.os[0] + (int64_t)(w.kvh * a.G + f - tok * a.G) * a.os[1];
#pragma unroll 1
            for (int x = 0; x < HD; x += 16) {
                uint32_t o[16];
                tmem_ld16(ot + x, o);
                tmem_ld_wait16(o);
                if (f < g.r1)
#pragma unroll
                    for (int ch = 0; ch < 2; ++ch)
                        if (x + ch * 8 < a.D) {
                            uint32_t e[4];
#pragma unroll
                            for (int y = 0; y < 4; ++y)  // a row without keys: 0 x 0
                                e[y] = E::pack(__fmul_rn(__uint_as_float(o[ch * 8 + 2 * y]), inv),
                                               __fmul_rn(__uint_as_float(o[ch * 8 + 2 * y + 1]), inv));
                            *reinterpret_cast<uint4 *>(out + x + ch * 8) = make_uint4(e[0], e[1], e[2], e[3]);
                        }
            }
            tc_fence_before();
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
cudaError_t rows_run(const AttnOp &a, const CUtensorMap &k, const CUtensorMap &v, const CUtensorMap &q, int box,
                     bool qtma, int nsm, cudaStream_t st) {
    return launch_k(attn_rows_kernel<T, HD>, dim3(nsm), dim3(RW_THREADS), RowsCfg<HD>::SMEM, st, a, k, v, q, box, qtma);
}

}  // namespace

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
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              // what lies behind a head's row is another head's
              a.D <= 64 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
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

// Q as a tensor map whose box is a row tile: 128 / G tokens x G heads x 64
// columns (G divides 128); false if there is none.
bool q_tensor_map(const AttnOp &a, int dtype, CUtensorMap &m) {
    EncodeTiledFn fn = rows_encode_fn();
    if (!fn || 128 % a.G) return false;
    const cuuint64_t unit = (cuuint64_t)((a.D * 2 + 15) / 16 * 16);
    const cuuint64_t dims[3] = {(cuuint64_t)a.D, (cuuint64_t)a.H, (cuuint64_t)a.T};
    const cuuint64_t strides[2] = {a.H == 1 ? unit : (cuuint64_t)a.qs[1] * 2, a.T == 1 ? unit : (cuuint64_t)a.qs[0] * 2};
    const cuuint32_t boxes[3] = {64u, (cuuint32_t)a.G, (cuuint32_t)(128 / a.G)}, es[3] = {1u, 1u, 1u};
    return fn(&m, dtype == PC_DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
              const_cast<void *>(a.q), dims, strides, boxes, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool launch_attn_rows(const AttnOp &a, int dtype, int nsm, cudaStream_t st, cudaError_t &e) {
    // positions per TMA box: the largest power of two that divides a page
    const int box = a.table ? std::min(a.page_size & -a.page_size, RW_KT) : RW_KT;
    CUtensorMap k, v, q;
    if (!kv_tensor_map(a, false, dtype, box, k) || !kv_tensor_map(a, true, dtype, box, v)) return false;
    const bool qtma = q_tensor_map(a, dtype, q);
    if (!qtma) q = k;  // not read
    if (dtype == PC_DT_F16)
        e = a.D <= 64 ? rows_run<__half, 64>(a, k, v, q, box, qtma, nsm, st)
                      : rows_run<__half, 128>(a, k, v, q, box, qtma, nsm, st);
    else
        e = a.D <= 64 ? rows_run<__nv_bfloat16, 64>(a, k, v, q, box, qtma, nsm, st)
                      : rows_run<__nv_bfloat16, 128>(a, k, v, q, box, qtma, nsm, st);
    return true;
}

}  // namespace pc
