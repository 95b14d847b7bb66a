// Fifth-generation tensor core (tcgen05) building blocks for sm_100a: tensor memory (TMEM)
// allocation, matrix instructions with bf16 operands and float32 accumulators, and the movement
// of accumulators between TMEM and registers.
//
// Conventions used throughout:
//   * a matrix instruction is issued by one thread; its completion is seen through
//     tcgen05.commit, which arrives on an mbarrier when every earlier instruction of that thread
//     is done.  Instructions of one thread execute in issue order, so a later one may overwrite
//     TMEM that an earlier one reads;
//   * the functions whose names end in _one are called by a whole converged warp with the same
//     arguments in every lane, and one elected lane (always the same) carries them out.  The warp
//     stays converged, so addresses and descriptors stay in uniform registers: eight matrix
//     instructions issue in 188 cycles, where the same ones inside a branch of one thread, which
//     moves every operand there first, took 650;
//   * TMEM is 128 lanes x 512 columns of 32 bits.  An accumulator with M = 128 rows has one row
//     per lane; warp w of a block reaches lanes 32 (w % 4) .. + 31, so a thread of a warpgroup
//     owns one row;
//   * shared-memory operand tiles are what a tiled TMA load with 64- or 128-byte swizzle writes:
//     rows of 64 or 128 bytes, split into column panels when a row is longer.
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

#include "tma.cuh"

namespace rfdetr {

// ---- TMEM allocation (whole warp) ----
__device__ __forceinline__ void tmem_alloc(uint32_t *slot, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)),
                 "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t base, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns) : "memory");
}

// ---- ordering ----
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Waits for this warp's loads from TMEM; the values are usable after pin() as well.
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// Keeps the compiler from using loaded registers before the wait above (the load is asynchronous,
// and nothing else ties its results to the wait).
template <int N> __device__ __forceinline__ void pin(float *v) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+f"(v[i]));
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Makes this thread's shared-memory writes visible to the tensor core and TMA (async proxy).
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Lets the stream's next kernel, launched to overlap this one, have the SMs that it leaves; that kernel waits
// for all of this one's results before it reads them.
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_primary() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ void mbar_arrive_one(uint64_t *bar) {
    asm volatile(
        "{\n.reg .pred q;\nelect.sync _|q, 0xffffffff;\n"
        "@q mbarrier.arrive.shared::cta.b64 _, [%0];\n}\n" ::"r"(smem_u32(bar))
        : "memory");
}
// Adds to the bytes that the current phase waits for, without arriving.
__device__ __forceinline__ void mbar_expect_one(uint64_t *bar, unsigned bytes) {
    asm volatile(
        "{\n.reg .pred q;\nelect.sync _|q, 0xffffffff;\n"
        "@q mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;\n}\n" ::"r"(smem_u32(bar)),
        "r"(bytes)
        : "memory");
}
__device__ __forceinline__ void mbar_arrive_expect_one(uint64_t *bar, unsigned bytes) {
    asm volatile(
        "{\n.reg .pred q;\nelect.sync _|q, 0xffffffff;\n"
        "@q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n}\n" ::"r"(smem_u32(bar)),
        "r"(bytes)
        : "memory");
}

// Arrives on `bar` once every matrix instruction issued so far by the elected lane has completed.
__device__ __forceinline__ void tc_commit_one(uint64_t *bar) {
    asm volatile(
        "{\n.reg .pred q;\nelect.sync _|q, 0xffffffff;\n"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_u32(bar))
        : "memory");
}

// ---- descriptors ----
// Swizzle modes of a shared-memory operand by its row length in bytes.
template <int ROWBYTES> struct SmemSwizzle;
template <> struct SmemSwizzle<128> { static constexpr uint64_t kMode = 2; };
template <> struct SmemSwizzle<64> { static constexpr uint64_t kMode = 4; };

// Operand descriptor of a swizzled tile at shared address `addr`; that of a part of it `bytes` further on is
// the descriptor + bytes / 16.  `sbo`: bytes from one group of
// eight rows to the next.  `lbo`: for a tile whose rows run along the contraction (the operand is
// "MN-major"), bytes from one column panel to the next; ignored when a row holds the contraction
// ("K-major").
template <int ROWBYTES>
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((addr >> 4) & 0x3fff) | ((uint64_t)((lbo >> 4) & 0x3fff) << 16) |
           ((uint64_t)((sbo >> 4) & 0x3fff) << 32) | (1ull << 46) | (SmemSwizzle<ROWBYTES>::kMode << 61);
}

// Instruction descriptor: bf16 x bf16 -> f32, M x N, B either K-major or MN-major (A K-major).
__host__ __device__ constexpr uint32_t mma_idesc(int m, int n, bool b_mn_major) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(m >> 4) << 24);
}

// N steps of 16 along the contraction, D[tmem] (+)= A B, the first adding to D where `accumulate` is set:
// A from shared memory (ss, descriptors AS and BS apart from step to step) or from TMEM (ts, two bf16 to a
// column, 8 columns a step), B from shared memory.  One block of code, so that a step is little more than the
// instruction itself: this warp shares its SM quarter, and the instruction cache of that, with warps whose
// unrolled code is larger than it.
template <int N, int AS, int BS>
__device__ __forceinline__ void mma_ss_one(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    static_assert(N == 2 || N == 4, "steps");
    if constexpr (N == 2) {
        asm volatile(
            "{\n.reg .pred p, q, t;\n.reg .b64 a, b;\nelect.sync _|q, 0xffffffff;\nsetp.ne.b32 p, %4, 0;\n"
            "setp.eq.b32 t, 0, 0;\n"
            "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\nadd.s64 a, %1, %5;\nadd.s64 b, %2, %6;\n"
            "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n}\n" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate), "n"(AS), "n"(BS)
            : "memory");
    } else {
        asm volatile(
            "{\n.reg .pred p, q, t;\n.reg .b64 a, b;\nelect.sync _|q, 0xffffffff;\nsetp.ne.b32 p, %4, 0;\n"
            "setp.eq.b32 t, 0, 0;\n"
            "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\nadd.s64 a, %1, %5;\nadd.s64 b, %2, %6;\n"
            "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\nadd.s64 a, a, %5;\nadd.s64 b, b, %6;\n"
            "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\nadd.s64 a, a, %5;\nadd.s64 b, b, %6;\n"
            "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n}\n" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate), "n"(AS), "n"(BS)
            : "memory");
    }
}
template <int N, int BS>
__device__ __forceinline__ void mma_ts_one(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    static_assert(N == 1 || N == 2 || N == 4, "steps");
    if constexpr (N == 1) {
        asm volatile(
            "{\n.reg .pred p, q;\nelect.sync _|q, 0xffffffff;\nsetp.ne.b32 p, %4, 0;\n"
            "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
            "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
            : "memory");
    } else if constexpr (N == 2) {
        asm volatile(
            "{\n.reg .pred p, q, t;\n.reg .b64 b;\n.reg .b32 a;\nelect.sync _|q, 0xffffffff;\nsetp.ne.b32 p, %4, 0;\n"
            "setp.eq.b32 t, 0, 0;\n"
            "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\nadd.s32 a, %1, 8;\nadd.s64 b, %2, %5;\n"
            "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n}\n" ::"r"(d),
            "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate), "n"(BS)
            : "memory");
    } else {
        asm volatile(
            "{\n.reg .pred p, q, t;\n.reg .b64 b;\n.reg .b32 a;\nelect.sync _|q, 0xffffffff;\nsetp.ne.b32 p, %4, 0;\n"
            "setp.eq.b32 t, 0, 0;\n"
            "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\nadd.s32 a, %1, 8;\nadd.s64 b, %2, %5;\n"
            "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\nadd.s32 a, a, 8;\nadd.s64 b, b, %5;\n"
            "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\nadd.s32 a, a, 8;\nadd.s64 b, b, %5;\n"
            "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n}\n" ::"r"(d),
            "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate), "n"(BS)
            : "memory");
    }
}

// ---- TMEM <-> registers: 32 consecutive columns of this thread's lane (whole warp) ----
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float *v) {
    uint32_t *r = reinterpret_cast<uint32_t *>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, float *v) {
    uint32_t *r = reinterpret_cast<uint32_t *>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// ---- registers of a warpgroup (all of its warps; the shares must add up to the launch's) ----
template <int N> __device__ __forceinline__ void regs_more() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N> __device__ __forceinline__ void regs_less() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// ---- clusters ----
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address in block `rank` of the cluster of what is at `addr` in this block's shared memory.
__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float cluster_ld(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

// ---- packed float32 pairs ----
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<uint64_t &>(d))
        : "l"(reinterpret_cast<uint64_t &>(a)), "l"(reinterpret_cast<uint64_t &>(b)),
          "l"(reinterpret_cast<uint64_t &>(c)));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t &>(d))
        : "l"(reinterpret_cast<uint64_t &>(a)), "l"(reinterpret_cast<uint64_t &>(b)));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("mul.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t &>(d))
        : "l"(reinterpret_cast<uint64_t &>(a)), "l"(reinterpret_cast<uint64_t &>(b)));
    return d;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 2^x of a pair on the FMA pipe, for sharing exponentials between it and the special-function unit
// (which takes 8 cycles of an SM quarter for a warp's exponentials, the other pipes idle).  x is
// split into its nearest integer n and a rest f in [-1/2, 1/2]; 2^f is a polynomial of degree 5 fitted
// by Lawson's reweighted least squares to the least relative error (2.4e-7 in float32 with the
// rounding of its steps, as ex2.approx).  2^n is made from n + 127 as its exponent field and multiplied:
// x is held at -127 and more, where that field is 0 and 2^n with it, so that -inf gives 0, and NaN, which
// the polynomial carries, stays NaN (adding n to the polynomial's own exponent field would turn it into a number).
__device__ __forceinline__ float2 exp2_poly(float2 x) {
    asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(x.x));  // -127
    asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(x.y));
    const float kMagic = 12582912.0f;  // 1.5 * 2^23: adding it rounds to an integer in the low bits
    const float2 t = add2(x, make_float2(kMagic, kMagic));
    const float2 n = add2(t, make_float2(-kMagic, -kMagic));
    const float2 f = fma2(n, make_float2(-1.0f, -1.0f), x);
    float2 p = make_float2(0.0013276472454890609f, 0.0013276472454890609f);
    p = fma2(p, f, make_float2(0.009675541892647743f, 0.009675541892647743f));
    p = fma2(p, f, make_float2(0.05550713092088699f, 0.05550713092088699f));
    p = fma2(p, f, make_float2(0.24022120237350464f, 0.24022120237350464f));
    p = fma2(p, f, make_float2(0.6931469440460205f, 0.6931469440460205f));
    p = fma2(p, f, make_float2(1.0000001192092896f, 1.0000001192092896f));
    return mul2(p, make_float2(__uint_as_float((__float_as_uint(t.x) << 23) + 0x3f800000u),
                               __uint_as_float((__float_as_uint(t.y) << 23) + 0x3f800000u)));
}
// Two bf16 (round to nearest even) in one register, `lo` in the low half.
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// 3-D tiled load of one box into shared memory, completing on `bar`.
__device__ __forceinline__ void tma_load_3d_one(uint32_t dst, const CUtensorMap *map, uint64_t *bar, int c0, int c1,
                                                int c2) {
    asm volatile(
        "{\n.reg .pred q;\nelect.sync _|q, 0xffffffff;\n"
        "@q cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, "
        "%4}], [%5];\n}\n" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
        : "memory");
}

}  // namespace rfdetr
