// attention_half.cuh - what the f16 / bf16 attention kernels over pages and
// packed prompts share: element types, bounded waits, TMA loads of 3 and 4
// dimensions, tensor maps of K and V.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "attention_plan.cuh"
#include "sm100.cuh"

namespace pc {

constexpr long long ATTN_WAIT_CLOCKS = 2000000000ll;  // about a second

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

// mbar_try_wait that may sleep up to 20 us: a waiting warp issues nothing
// that the other warps of its scheduler would have to wait for
__device__ __forceinline__ bool mbar_sleep_wait(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 20000;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}

// A bounded wait of one of a block's threads: false once it, or any other
// wait of the block, gave up (*dead, in shared memory); *err tells the host.
// What comes after the first try is a function of its own: inlined at every
// wait it filled the instruction cache.
static __device__ __noinline__ bool bounded_wait_on(uint64_t *bar, uint32_t parity, volatile int *dead, int *err) {
    const long long t0 = clock64();
    while (!mbar_sleep_wait(bar, parity)) {
        if (*dead) return false;
        if (clock64() - t0 > ATTN_WAIT_CLOCKS) {
            *dead = 1;
            atomicExch(err, 1);
            return false;
        }
    }
    return true;
}
__device__ __forceinline__ bool bounded_wait(uint64_t *bar, uint32_t parity, volatile int *dead, int *err) {
    return mbar_sleep_wait(bar, parity) || bounded_wait_on(bar, parity, dead, err);
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

// The factor of a finished row's O: m, l its reference (in powers of two) and
// sum, `sink` its sink's score in powers of two.  0 for a row without keys.
template <typename E>
__device__ __forceinline__ float row_factor(float m, float l, bool sinks, float sink) {
    if (m == -INFINITY && l == 0.0f) return 0.0f;
    if (!sinks) return __fdividef(1.0f, l);
    // both on the larger of the two references; E::BIAS is in l and O
    const float mm = fmaxf(m, sink), e = ex2(__fsub_rn(m, mm));
    return __fdividef(e, __fmaf_rn(l, e, ex2(__fadd_rn(__fsub_rn(sink, mm), E::BIAS))));
}

// K or V as a tensor map: rows of head_dim elements, boxes of 64 columns x
// `box` positions of one head, 128-byte swizzle, zeros outside.  False if its
// strides cannot be described (a stride of zero).
bool kv_tensor_map(const AttnOp &a, bool v, int dtype, int box, CUtensorMap &m);

}  // namespace pc
