// tensor_core.cuh -- the fifth-generation tensor core in inline PTX: tensor
// memory, shared-memory operands, matrix instructions, barriers with bounded
// waits.  16-bit operands, 32-bit sums in tensor memory.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

namespace racb {
namespace tc {

__device__ __forceinline__ uint32_t smem(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

// ── barriers ──────────────────────────────────────────────────────────────
__device__ __forceinline__ void bar_init(uint64_t* bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(smem(bar)), "r"(count));
}
__device__ __forceinline__ void bar_init_done() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void bar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(smem(bar)) : "memory");
}
__device__ __forceinline__ void bar_expect(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(smem(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(smem(bar)), "r"(parity) : "memory");
    return ok != 0;
}

// Every wait ends: after kWaitNs, or when another thread of the block gave up,
// `gone` is set and the wait returns false.  The kernel then skips the rest of
// its work, settles, frees its tensor memory and returns.
constexpr uint64_t kWaitNs = 4000000000ull;
__device__ __forceinline__ uint64_t now_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity, volatile int* gone) {
    if (bar_try(bar, parity)) return true;
    const uint64_t t0 = now_ns();
#pragma unroll 1
    for (uint32_t i = 0; i < (1u << 30); ++i) {
        if (bar_try(bar, parity)) return true;
        if ((i & 63) == 63 && (*gone || now_ns() - t0 > kWaitNs)) break;
    }
    *gone = 1;
    return false;
}
constexpr unsigned int kErrTcWait = 16u;      // bit 4 of the device error word
// Before such a block leaves: its copies and products under way, which end by
// themselves within microseconds, must not land in memory that another block has
// got by then.  No barrier tells (one that would have is what the block gave up
// on), so it waits a millisecond; by every thread, after the block has met.
__device__ __forceinline__ void settle(volatile int* gone) {
    if (!*gone) return;
    const uint64_t t0 = now_ns();
#pragma unroll 1
    for (int i = 0; i < 4096 && now_ns() - t0 < 1000000ull; ++i) __nanosleep(1000);
}

// ── TMA ───────────────────────────────────────────────────────────────────
__device__ __forceinline__ void load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
                 " [%0], [%1, {%2, %3, %4}], [%5];"
                 :: "r"(smem(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem(bar))
                 : "memory");
}
// Shared memory written by this thread becomes visible to TMA and to matrix
// instructions.
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ── tensor memory ─────────────────────────────────────────────────────────
// One warp allocates (and later frees) a power of two of columns.
__device__ __forceinline__ void tmem_alloc(uint32_t* base, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem(base)), "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(base), "r"(columns));
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 columns of the thread's lane (address: lane of the warp's quarter << 16 | column).
__device__ __forceinline__ void ld32(uint32_t (&r)[32], uint32_t addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr) : "memory");
}
__device__ __forceinline__ void ld16(uint32_t (&r)[16], uint32_t addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
        "[%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr) : "memory");
}
__device__ __forceinline__ void st32(uint32_t addr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        :: "r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
           "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
           "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
           "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16};"
        :: "r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
           "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// ── matrix instructions ───────────────────────────────────────────────────
// A shared-memory operand: tiles of rows of SW bytes (64 or 128, the swizzle),
// eight rows an atom.  K-major (the summed axis runs along a row): `stride`
// leads from one group of eight rows to the next, `lead` is not used.
// MN-major (the summed axis runs across rows): `stride` leads from eight
// summed rows to the next eight, `lead` from SW bytes of the other axis to
// the next SW bytes.
template <int SW>
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t lead, uint32_t stride) {
    constexpr uint64_t swz = SW == 128 ? 2 : 4;
    return (uint64_t)((addr & 0x3ffff) >> 4) | (uint64_t)(lead >> 4) << 16 | (uint64_t)(stride >> 4) << 32 |
           (uint64_t)1 << 46 | swz << 61;
}

// D is 32-bit, A and B are both T.  b_rows: B is MN-major.
template <typename T>
__device__ constexpr uint32_t instruction(int m, int n, bool b_rows) {
    const uint32_t fmt = sizeof(T) == 2 && !std::is_same<T, __half>::value ? 1 : 0;      // 0 f16, 1 bf16
    return 1u << 4 | fmt << 7 | fmt << 10 | (b_rows ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 |
           (uint32_t)(m >> 4) << 24;
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t instr, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 :: "r"(d), "l"(a), "l"(b), "r"(instr), "r"((uint32_t)add) : "memory");
}
// A in tensor memory: a row a lane, two 16-bit values a column.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t instr, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 :: "r"(d), "r"(a), "l"(b), "r"(instr), "r"((uint32_t)add) : "memory");
}
// The barrier completes a phase when all matrix instructions that this thread
// has issued so far are done.
__device__ __forceinline__ void commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(smem(bar))
                 : "memory");
}

// Registers a thread of this warpgroup may use from here on.  The shares of a
// block's warpgroups add up to what it was launched with.
template <int N> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(N)); }
template <int N> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(N)); }

// Sums over a contiguous axis: D (+)= A B^T over 16 * STEPS summed values, both
// operands K-major in boxes of rows of SW bytes (box: bytes of one).  The
// addresses of the steps are constants apart, so that one thread issues a step
// in a few cycles.
template <int STEPS, int SW>
__device__ __forceinline__ void product_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t box, uint32_t instr) {
    const uint64_t da = operand<SW>(a, 16, 8 * SW), db = operand<SW>(b, 16, 8 * SW);
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
        const uint32_t off = ((k * 32 / SW) * box + (k * 32) % SW) >> 4;
        mma_ss(d, da + off, db + off, instr, k > 0);
    }
}

// ── values ────────────────────────────────────────────────────────────────
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <typename T> __device__ __forceinline__ float low_of(uint32_t p) {
    return std::is_same<T, __half>::value ? __low2float(*reinterpret_cast<const __half2*>(&p)) : __uint_as_float(p << 16);
}
template <typename T> __device__ __forceinline__ float high_of(uint32_t p) {
    return std::is_same<T, __half>::value ? __high2float(*reinterpret_cast<const __half2*>(&p)) : __uint_as_float(p & 0xffff0000u);
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The largest (smallest) of 32 values: two a step.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
    float r;
    asm("min.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float largest32(const uint32_t (&v)[32]) {
    float z[2] = {__uint_as_float(v[0]), __uint_as_float(v[1])};
#pragma unroll
    for (int i = 2; i < 30; i += 4) {
        z[0] = max3(z[0], __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
        z[1] = max3(z[1], __uint_as_float(v[i + 2]), __uint_as_float(v[i + 3]));
    }
    return fmaxf(max3(z[0], __uint_as_float(v[30]), __uint_as_float(v[31])), z[1]);
}
__device__ __forceinline__ float smallest32(const uint32_t (&v)[32]) {
    float z[2] = {__uint_as_float(v[0]), __uint_as_float(v[1])};
#pragma unroll
    for (int i = 2; i < 30; i += 4) {
        z[0] = min3(z[0], __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
        z[1] = min3(z[1], __uint_as_float(v[i + 2]), __uint_as_float(v[i + 3]));
    }
    return fminf(min3(z[0], __uint_as_float(v[30]), __uint_as_float(v[31])), z[1]);
}
// Two values at a time: one instruction where scalar code takes two, and it is
// instructions, not the exponential unit, that bound the softmax warps (taking
// part of the exponentials by polynomial on the FMA pipe made them slower).
__device__ __forceinline__ float2 pair(uint32_t a, uint32_t b) { return make_float2(__uint_as_float(a), __uint_as_float(b)); }
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 exp2_both(float2 x) { return make_float2(exp2_fast(x.x), exp2_fast(x.y)); }

}  // namespace tc
}  // namespace racb
