// attention_few.cu - attention of few rows a request (single tokens, a few
// guessed ones) over pages, for f16 and bf16 tensors: bound by reading K and
// V once.
//
// A thread block (two per SM) takes the items of its share
// (attention_plan.cuh): up to 8 or 16 rows (tokens x query heads of one KV
// head) against all their keys, in tiles of 16 KB of K and V (64 keys at head
// sizes to 64, 32 at 128).  The warps take the tiles in turn, each with its
// own running maximum, sum and O in registers.  The products are mma.sync
// m16n8k16 with the few rows as the N side: S^T = K Q^T (16 keys x 8 rows) and
// O^T += V^T P^T (16 head columns x 8 rows), so eight rows leave nothing of a
// product unused; P^T turns from accumulator to operand by movmatrix.  P is
// rounded to the type, and what the rounding left has a product of its own: the
// tensor pipe has room, and the error of bf16 outputs is that of their own
// rounding (decode of 64 requests 1.97e-3 -> 1.66e-3 from the exact result; 109.5
// -> 110.0 us, head size 128 184.4 -> 186.0).  (With the rows as the M side, half
// of the products and of the exponentials were of rows that did not exist: head
// size 128 211 us where it was 184, one token 16 us where it was 14.)  The legacy
// products are far below their rate while the tiles arrive.
//
// A warp fetches its own tiles by TMA, the next one as soon as it is done with
// one and across the ends of items, so the memory system does not see where
// one ends, no two warps meet inside an item, and a tile's page lookups are
// spread over the warps (one warp fetching for all could not keep up: 2300
// cycles a tile).  At the end of an item the warps' parts are joined in shared
// memory, and those of several blocks (a row cut between shares) in the
// workspace.
//
// Measured: one token each of 64 requests of 500-8000 positions, 64 query over
// 8 KV heads of 64, bf16, pages of 16: 110 us, 5.4 TB/s (83 % of the measured
// copy; 114 with the launch of the many-row kernel behind it, which finds nothing
// to do); 32 over 8 heads of 128, f16, pages of 32: 186 us, 6.4 TB/s (98 %; 189).
// 64-wide heads read 128 bytes of each 1 KB row; with pages laid out heads
// first they are 6 % faster.  One token over 4096 positions takes 15 us: 2.5 us
// to find the shares, about 2 until the first tile is there, the rest its work,
// the joins and their trips to L2.  What an item costs beside its keys counts as
// 256 of them in the shares (128, 512: 64 requests 117, 111 us where it is 113, 300
// tokens to 600 of 128-wide heads 128, 95 where it is 90, one token 14.1, 15.2
// where it is 14.8).
#include <algorithm>

#include "attention_half.cuh"
#include "launch.cuh"

namespace pc {

namespace {

constexpr int FW_WARPS = 4, FW_THREADS = FW_WARPS * 32, FW_OV = 256, FW_MINK = 128;
constexpr int FW_PER_SM = 2, FW_AHEAD = 1;  // blocks an SM; stages a warp

template <int HD>
constexpr int FW_KT = 4096 / HD;

template <int HD, int NR>
struct FewCfg {
    static constexpr int R = 8 * NR;  // rows of an item
    static constexpr int KT = FW_KT<HD>, PANELS = HD / 64;
    static constexpr int STAGES = FW_WARPS * FW_AHEAD;
    static constexpr int PANEL = KT * 128, TILE = PANELS * PANEL;  // 8 KB of K, and of V
    static constexpr int LDR = HD + 4;                             // floats of a row of a warp's record
    static constexpr int REC = R * LDR;
    static constexpr size_t SMEM = 1024 + (size_t)STAGES * 2 * TILE + FW_WARPS * REC * 4;
    static constexpr int PART = R * (HD + 2);  // floats of a block's record: O, m, l
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
// An 8 x 8 matrix of 16-bit elements (lane 4 r + c: elements 2 c, 2 c + 1 of row r), transposed
__device__ __forceinline__ uint32_t turn8(uint32_t v) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
    return d;
}

template <typename T, int HD, int NR>
__global__ void __launch_bounds__(FW_THREADS, FW_PER_SM)
    attn_few_kernel(const AttnOp a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                    const int box) {
    using C = FewCfg<HD, NR>;
    using E = Half16<T>;
    constexpr int KT = C::KT, NS = C::STAGES, R = C::R;
    extern __shared__ uint8_t few_smem_raw[];
    uint8_t *ring = few_smem_raw + (1024 - (smem_u32(few_smem_raw) & 1023)) % 1024;
    float *recs = reinterpret_cast<float *>(ring + NS * 2 * C::TILE);
    __shared__ PlanScratch<FW_THREADS> sc;
    __shared__ uint64_t full[NS], meet_bar;
    __shared__ volatile int dead;
    __shared__ int lastf;
    __shared__ float wm[FW_WARPS][R], wl[FW_WARPS][R];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < NS; ++s) mbar_init(&full[s], 1);
        mbar_init(&meet_bar, FW_WARPS);
        fence_mbar_init();
        dead = 0;
        tma_prefetch_desc(&kmap);
        tma_prefetch_desc(&vmap);
    }
    pdl_wait();
    pdl_trigger();
    plan_share<R, KT, FW_OV, FW_MINK, FW_THREADS>(a, blockIdx.x, gridDim.x, sc);
    if (sc.share.n == 0) return;
    auto wait_all = [&](uint64_t *b, uint32_t parity) -> bool {
        return __all_sync(0xffffffffu, bounded_wait(b, parity, &dead, a.err));
    };

    // ---- fetching: this warp's tiles warp, warp + FW_WARPS, ... of the share, stage FW_AHEAD * warp + (its count) % FW_AHEAD
    uint64_t *wfull = full + warp * FW_AHEAD;
    uint8_t *wring = ring + warp * FW_AHEAD * 2 * C::TILE;
    PlanWalk<R, KT> wi(a, sc.share);
    bool imore = wi.load();
    int it_i = wi.tl, fetched = 0;  // tile of wi, tiles fetched
    auto settle = [&](int t) {      // tile t of wi's item, or of a later item
        while (imore && t >= wi.th) {
            t -= wi.th;
            imore = wi.next();
            t += wi.tl;
        }
        it_i = t;
    };
    // one box a lane: of K or V, a panel, `box` positions
    const int boxes = KT / box, brow = lane % boxes * box, bp = lane / boxes % C::PANELS, bv = lane / boxes / C::PANELS;
    const CUtensorMap *bmap = bv ? &vmap : &kmap;
    const int bdst = bv * C::TILE + bp * C::PANEL + brow * 128;
    int bpage = 0, boff = 0;  // this lane's page id and row in the page of tile it_i
    auto look_up = [&]() {
        if (!imore) return;
        const int key = (wi.g.t0 + it_i) * KT + brow, pg = key / a.page_size;
        boff = key - pg * a.page_size;
        bpage = pg < a.max_pages ? a.table[(int64_t)wi.b * a.max_pages + pg] : -1;
    };
    auto fetch = [&]() {
        if (!imore) return;
        const int s = fetched % FW_AHEAD, k0 = (wi.g.t0 + it_i) * KT, key = k0 + brow;
        const bool in = bv < 2 && key + box > wi.g.kb && key < wi.g.ke;  // boxes that hold keys of the item
        const int n = __popc(__ballot_sync(0xffffffffu, in));
        if (lane == 0) {
            if (n) mbar_arrive_expect_tx(&wfull[s], (uint32_t)n * box * 128);
            else mbar_arrive(&wfull[s]);
        }
        __syncwarp();
        if (in) {
            uint8_t *d = wring + s * 2 * C::TILE + bdst;
            tma_load_4d(d, bmap, &wfull[s], bp * 64, boff, wi.kvh, bpage);
        }
        ++fetched;
        settle(it_i + FW_WARPS);
        look_up();
    };
    // after a failure: copies in flight land before the block ends
    auto drain = [&]() {
        for (int s = 0; s < FW_AHEAD && lane == 0; ++s) {
            const int n = (fetched - s + FW_AHEAD - 1) / FW_AHEAD;
            const long long t0 = clock64();
            if (n > 0)
                while (!mbar_try_wait(&wfull[s], (n - 1) & 1))
                    if (clock64() - t0 > ATTN_WAIT_CLOCKS) break;
        }
    };
    settle(wi.tl + warp);
    look_up();
    for (int x = 0; x < FW_AHEAD; ++x) fetch();

    PlanWalk<R, KT> w(a, sc.share);
    const int g8 = lane >> 2, t4 = lane & 3;
    const float c = __fmul_rn(a.scale, 1.4426950408889634f);
    int it = 0, used = 0;  // tiles of the share before the item at hand, tiles of this warp done
    uint32_t meets = 0;
    auto meet = [&]() -> bool {  // all warps
        __syncwarp();
        if (lane == 0) mbar_arrive(&meet_bar);
        if (wait_all(&meet_bar, meets++ & 1)) return true;
        drain();
        return false;
    };
    for (bool more = w.load(); more; more = w.next()) {
        const ItemGeo g = w.g;
        // Q: rows g8 (and g8 + 8) of the item as the products' N side, zeros past it and past head_dim
        uint32_t qf[HD / 16][NR][2];
        int pos[NR][2];  // positions of rows 8 n + 2 t4, + 1: those of this lane's scores
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            const int f = g.r0 + g8 + 8 * n;
            const bool in = f < g.r1;
            const int tok = in ? div_g(a, f) : 0;
            const T *q = reinterpret_cast<const T *>(a.q) + (int64_t)(w.s.q0 + tok) * a.qs[0] +
                         (int64_t)(w.kvh * a.G + (in ? f - tok * a.G : 0)) * a.qs[1];
#pragma unroll
            for (int k = 0; k < HD / 16; ++k)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int d = k * 16 + x * 8 + 2 * t4;
                    qf[k][n][x] = in && d < a.D ? *reinterpret_cast<const uint32_t *>(q + d) : 0u;
                }
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int fr = g.r0 + 8 * n + 2 * t4 + x;
                pos[n][x] = fr < g.r1 ? w.s.p0 + div_g(a, fr) : -1;
            }
        }
        float m[NR][2], l[NR][2], o[HD / 16][NR][4];  // l: of this lane's keys
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.0f;
#pragma unroll
            for (int d = 0; d < HD / 16; ++d)
#pragma unroll
                for (int x = 0; x < 4; ++x) o[d][n][x] = 0.0f;
        }
        bool ok = true;
        const int mine = w.tl + (warp - it % FW_WARPS + FW_WARPS) % FW_WARPS;  // this warp's first
        for (int t = mine; t < w.th; t += FW_WARPS, ++used) {
            const int s = used % FW_AHEAD;
            if (!(ok = wait_all(&wfull[s], (used / FW_AHEAD) & 1))) break;
            const int k0 = (g.t0 + t) * KT;
            const uint32_t kt = smem_u32(wring + s * 2 * C::TILE), vt = kt + C::TILE;
            // S^T: element x of sc4[i][n] is key 16 i + g8 + 8 (x / 2), row 8 n + 2 t4 + x % 2
            float sc4[KT / 16][NR][4];
#pragma unroll
            for (int i = 0; i < KT / 16; ++i) {
#pragma unroll
                for (int n = 0; n < NR; ++n)
#pragma unroll
                    for (int x = 0; x < 4; ++x) sc4[i][n][x] = 0.0f;
#pragma unroll
                for (int k = 0; k < HD / 16; ++k) {
                    uint32_t f[4];
                    const int row = i * 16 + (lane & 15), ch = 2 * k + (lane >> 4);
                    ldsm4(f, kt + (ch >> 3) * C::PANEL + row * 128 + (((ch & 7) ^ (row & 7)) << 4));
#pragma unroll
                    for (int n = 0; n < NR; ++n) mma16<T>(sc4[i][n], f, qf[k][n][0], qf[k][n][1]);
                }
                // in powers of two, rounded here: maximum, weights and rescaling all go by the same numbers
#pragma unroll
                for (int n = 0; n < NR; ++n)
#pragma unroll
                    for (int x = 0; x < 4; ++x) sc4[i][n][x] = __fmul_rn(sc4[i][n][x], c);
            }
            const bool masked = k0 + KT - 1 > g.pmin || (a.window > 0 && k0 < g.pmax - a.window + 1);
            bool odd = false;  // non-finite V that only some rows see
            if (masked) {
#pragma unroll
                for (int i = 0; i < KT / 16; ++i)
#pragma unroll
                    for (int n = 0; n < NR; ++n)
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const int key = k0 + 16 * i + g8 + 8 * (x >> 1), p = pos[n][x & 1];
                            if (key > p || (a.window > 0 && key <= p - a.window)) sc4[i][n][x] = -INFINITY;
                        }
                // V rows outside the item's keys hold anything: zeros.  Non-finite V that only some rows see is
                // added to those and taken out.
                uint8_t *v = wring + (s * 2 + 1) * C::TILE;
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
                odd = __any_sync(0xffffffffu, bad);
            }
            uint32_t pf[KT / 16][NR][2], pr[KT / 16][NR][2];  // weights in the type, and what that rounding left
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                float corr[2], ms[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    float top = -INFINITY;
#pragma unroll
                    for (int i = 0; i < KT / 16; ++i) top = fmaxf(top, fmaxf(sc4[i][n][x], sc4[i][n][x + 2]));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                    const float mn = fmaxf(m[n][x], top);
                    ms[x] = mn == -INFINITY ? 0.0f : mn;
                    corr[x] = ex2(__fsub_rn(m[n][x], ms[x]));  // 1 while the maximum stands
                    m[n][x] = mn;
                    l[n][x] = __fmul_rn(l[n][x], corr[x]);
                }
#pragma unroll
                for (int i = 0; i < KT / 16; ++i)
#pragma unroll
                    for (int y = 0; y < 2; ++y) {  // keys g8, g8 + 8
                        const float p0 = ex2(__fadd_rn(__fsub_rn(sc4[i][n][2 * y], ms[0]), E::BIAS));
                        const float p1 = ex2(__fadd_rn(__fsub_rn(sc4[i][n][2 * y + 1], ms[1]), E::BIAS));
                        l[n][0] = __fadd_rn(l[n][0], p0);
                        l[n][1] = __fadd_rn(l[n][1], p1);
                        const uint32_t h = E::pack(p0, p1);
                        pf[i][n][y] = turn8(h);
                        pr[i][n][y] = turn8(E::pack(__fsub_rn(p0, E::up(h & 0xFFFFu)), __fsub_rn(p1, E::up(h >> 16))));
                    }
                if (__any_sync(0xffffffffu, corr[0] != 1.0f || corr[1] != 1.0f))
#pragma unroll
                    for (int d = 0; d < HD / 16; ++d)
#pragma unroll
                        for (int x = 0; x < 4; ++x) o[d][n][x] = __fmul_rn(o[d][n][x], corr[x & 1]);
            }
            if (odd) {  // after the rescaling, whose first factor is 0
                uint8_t *v = wring + (s * 2 + 1) * C::TILE;
#pragma unroll 1
                for (int r = 0; r < KT; ++r) {
                    const int key = k0 + r;
                    if (key < g.kb || key >= g.ke) continue;
#pragma unroll
                    for (int d = 0; d < HD / 16; ++d)
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const int c0 = d * 16 + g8 + 8 * (x >> 1), ch = c0 >> 3;
                            const float f = E::up(*reinterpret_cast<const unsigned short *>(
                                v + (ch >> 3) * C::PANEL + r * 128 + (((ch & 7) ^ (r & 7)) << 4) + (c0 & 7) * 2));
#pragma unroll
                            for (int n = 0; n < NR; ++n) {
                                const int p = pos[n][x & 1];
                                if (!isfinite(f) && key <= p && !(a.window > 0 && key <= p - a.window))
                                    o[d][n][x] = __fadd_rn(o[d][n][x], f);
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
            // O^T += V^T P^T; what the weights' rounding left apart, so that a V that is infinite does not meet it (0 or
            // below: inf would become NaN)
#pragma unroll
            for (int d = 0; d < HD / 16; ++d) {
                float rest[NR][4];
#pragma unroll
                for (int n = 0; n < NR; ++n)
#pragma unroll
                    for (int x = 0; x < 4; ++x) rest[n][x] = 0.0f;
#pragma unroll
                for (int i = 0; i < KT / 16; ++i) {
                    uint32_t f[4];
                    const int j = lane >> 3, row = 16 * i + (lane & 7) + 8 * (j >> 1), ch = 2 * d + (j & 1);
                    ldsm4_t(f, vt + (ch >> 3) * C::PANEL + row * 128 + (((ch & 7) ^ (row & 7)) << 4));
#pragma unroll
                    for (int n = 0; n < NR; ++n) {
                        mma16<T>(o[d][n], f, pf[i][n][0], pf[i][n][1]);
                        mma16<T>(rest[n], f, pr[i][n][0], pr[i][n][1]);
                    }
                }
#pragma unroll
                for (int n = 0; n < NR; ++n)
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        o[d][n][x] = isfinite(o[d][n][x]) ? __fadd_rn(o[d][n][x], rest[n][x]) : o[d][n][x];
            }
            if (masked) fence_async_smem();  // V rows written here, and by TMA next
            __syncwarp();
            fetch();
        }
        it += w.th - w.tl;
        if (!ok) {
            drain();
            return;
        }

        // the warps' parts in shared memory; thread: a row, CW columns
        float *rec = recs + warp * C::REC;
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int row = 8 * n + 2 * t4 + x;
#pragma unroll
                for (int d = 0; d < HD / 16; ++d) {
                    rec[row * C::LDR + d * 16 + g8] = o[d][n][x];
                    rec[row * C::LDR + d * 16 + g8 + 8] = o[d][n][x + 2];
                }
                float ll = l[n][x];
                ll = __fadd_rn(ll, __shfl_xor_sync(0xffffffffu, ll, 4));
                ll = __fadd_rn(ll, __shfl_xor_sync(0xffffffffu, ll, 8));
                ll = __fadd_rn(ll, __shfl_xor_sync(0xffffffffu, ll, 16));
                if (g8 == 0) {
                    wm[warp][row] = m[n][x];
                    wl[warp][row] = ll;
                }
            }
        if (!meet()) return;
        constexpr int TPR = FW_THREADS / R, CW = HD / TPR;
        const int row = tid / TPR, col = tid % TPR * CW;
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
            if (col == 0) {
                __stcg(p + R * HD + row, mm);
                __stcg(p + R * (HD + 1) + row, ll);
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
            constexpr int PK = 4;  // parts at a time: their loads go together
#pragma unroll 1
            for (int k = ci.k0; k <= ci.k1; k += PK) {
                float pm[PK], pl[PK];
                float4 po[PK][CW / 4];
#pragma unroll
                for (int x = 0; x < PK; ++x) {
                    const int kx = min(k + x, ci.k1);
                    const float *q = a.part + ((int64_t)kx * 2 + (kx == ci.k0)) * C::PART;
                    pm[x] = __ldcg(q + R * HD + row);
                    pl[x] = __ldcg(q + R * (HD + 1) + row);
#pragma unroll
                    for (int d = 0; d < CW / 4; ++d)
                        po[x][d] = __ldcg(reinterpret_cast<const float4 *>(q + row * HD + col) + d);
                }
                float mn = mm;
#pragma unroll
                for (int x = 0; x < PK; ++x) mn = fmaxf(mn, pm[x]);
                ms = mn == -INFINITY ? 0.0f : mn;
                const float old = ex2(__fsub_rn(mm, ms));
                mm = mn;
                ll = __fmul_rn(ll, old);
#pragma unroll
                for (int d = 0; d < CW; ++d) acc[d] = __fmul_rn(acc[d], old);
#pragma unroll
                for (int x = 0; x < PK; ++x) {
                    if (k + x > ci.k1) continue;
                    const float e = ex2(__fsub_rn(pm[x], ms));
                    ll = __fmaf_rn(pl[x], e, ll);
#pragma unroll
                    for (int d = 0; d < CW / 4; ++d) {
                        acc[4 * d] = __fmaf_rn(po[x][d].x, e, acc[4 * d]);
                        acc[4 * d + 1] = __fmaf_rn(po[x][d].y, e, acc[4 * d + 1]);
                        acc[4 * d + 2] = __fmaf_rn(po[x][d].z, e, acc[4 * d + 2]);
                        acc[4 * d + 3] = __fmaf_rn(po[x][d].w, e, acc[4 * d + 3]);
                    }
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
            for (int d = 0; d < CW; d += 4)  // head_dim is a multiple of 8, so of 4
                if (col + d < a.D)
                    *reinterpret_cast<uint2 *>(out + d) =
                        none ? make_uint2(0, 0)
                             : make_uint2(E::pack(__fmul_rn(acc[d], inv), __fmul_rn(acc[d + 1], inv)),
                                          E::pack(__fmul_rn(acc[d + 2], inv), __fmul_rn(acc[d + 3], inv)));
        }
        if (!meet()) return;  // the records may be written again
    }
}

template <typename T, int HD, int NR>
cudaError_t few_set() {
    return cudaFuncSetAttribute(attn_few_kernel<T, HD, NR>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)FewCfg<HD, NR>::SMEM);
}

template <typename T, int HD, int NR>
cudaError_t few_run(const AttnOp &a, const CUtensorMap &k, const CUtensorMap &v, int box, int nsm, cudaStream_t st) {
    return launch_k(attn_few_kernel<T, HD, NR>, dim3(nsm * FW_PER_SM), dim3(FW_THREADS), FewCfg<HD, NR>::SMEM, st, a, k,
                    v, box);
}

// Items of 8 rows where the batch has no more than that a request (what 16
// would add is products of rows that do not exist), else of 16 (a request of
// 9 to 16 rows reads its keys once).
template <typename T, int HD>
cudaError_t few_pick(const AttnOp &a, const CUtensorMap &k, const CUtensorMap &v, int box, int nsm, cudaStream_t st) {
    return (int64_t)a.T * a.G <= (int64_t)8 * a.B ? few_run<T, HD, 1>(a, k, v, box, nsm, st)
                                                  : few_run<T, HD, 2>(a, k, v, box, nsm, st);
}

template <typename T>
cudaError_t few_set_all() {
    cudaError_t e = few_set<T, 64, 1>();
    if (e == cudaSuccess) e = few_set<T, 64, 2>();
    if (e == cudaSuccess) e = few_set<T, 128, 1>();
    if (e == cudaSuccess) e = few_set<T, 128, 2>();
    return e;
}

}  // namespace

size_t attn_few_part_floats(int nsm) { return (size_t)nsm * FW_PER_SM * 2 * FewCfg<128, 2>::PART; }

cudaError_t attn_few_configure() {
    const cudaError_t e = few_set_all<__half>();
    return e == cudaSuccess ? few_set_all<__nv_bfloat16>() : e;
}

bool launch_attn_few(const AttnOp &a, int dtype, int nsm, cudaStream_t st, cudaError_t &e) {
    // positions per TMA box: the largest power of two that divides a page
    const int box = std::min(a.page_size & -a.page_size, a.D <= 64 ? FW_KT<64> : FW_KT<128>);
    CUtensorMap k, v;
    if (!kv_tensor_map(a, false, dtype, box, k) || !kv_tensor_map(a, true, dtype, box, v)) return false;
    if (dtype == PC_DT_F16)
        e = a.D <= 64 ? few_pick<__half, 64>(a, k, v, box, nsm, st) : few_pick<__half, 128>(a, k, v, box, nsm, st);
    else
        e = a.D <= 64 ? few_pick<__nv_bfloat16, 64>(a, k, v, box, nsm, st)
                      : few_pick<__nv_bfloat16, 128>(a, k, v, box, nsm, st);
    return true;
}

}  // namespace pc
