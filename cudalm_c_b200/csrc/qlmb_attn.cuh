// Shared by the attention kernels and the adapters' (qlmb_attn.cu, qlmb_prefix.cu, qlmb_lora.cu): bounded waits, 2^x, two-wide fp32.
#pragma once
#include "qlmb_tc.cuh"

namespace qlmb {

// Bounded wait of the attention kernels: a tile step takes microseconds, so a wait that has polled
// for about a second is broken; it raises the CTA's abort flag and records its site.  CTAs that
// start after an error was recorded leave at once (at_error_seen), so a broken pipeline ends the
// launch quickly instead of timing out CTA by CTA.
constexpr uint32_t AT_WAIT_LIMIT = 1u << 21;               // polls of the drain loops on the abort path
constexpr unsigned long long AT_WAIT_NS = 1000000000ull;    // one second of wall clock per wait
__device__ __forceinline__ unsigned long long at_now()
{
    unsigned long long t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
__device__ __forceinline__ uint32_t at_test(uint32_t bar, uint32_t parity)     // non-blocking probe
{
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok;
}
__device__ __forceinline__ bool at_wait(uint32_t bar, uint32_t parity, volatile int *abort_flag, int *errword, int site)
{
    if (mbar_try(bar, parity)) return true;
    unsigned long long t0 = 0;                 // read on the slow path only
    for (uint32_t i = 0;; i++) {
        if (at_test(bar, parity)) return true;
        if ((i & 1023u) == 1023u) {
            if (*abort_flag) return false;
            const unsigned long long now = at_now();
            if (!t0) t0 = now;
            else if (now - t0 > AT_WAIT_NS) break;
        }
    }
    if (!*abort_flag) {
        *abort_flag = 1;
        if (errword && atomicCAS(errword, 0, 200) == 0) { errword[1] = site; errword[2] = (int)blockIdx.x; errword[3] = (int)parity; }
    }
    return false;
}
// A warp's wait: all of its lanes go on (0), or none (the site).  Bounded like at_wait, by a second of the clock's lower half.  try_wait lets
// the hardware hold the warp until the phase ends or a time of its own is over: a loop of test_wait instead keeps the queue busy that
// the exponentials go through, too.
__device__ __forceinline__ uint32_t at_now_lo() { uint32_t t; asm volatile("mov.u32 %0, %%globaltimer_lo;" : "=r"(t)); return t; }
__device__ __forceinline__ int at_all_wait(uint32_t bar, uint32_t parity, volatile int *abort_flag, int site)
{
    uint32_t t0 = 0;
#pragma unroll 1
    for (uint32_t i = 0; !__all_sync(~0u, mbar_try(bar, parity)); i++)
        if ((i & 63u) == 63u) {
            const uint32_t now = __shfl_sync(~0u, at_now_lo(), 0);
            if (i == 63u) t0 = now;
            if (__any_sync(~0u, *abort_flag) || now - t0 > (uint32_t)AT_WAIT_NS) return site;
        }
    return 0;
}
__device__ __forceinline__ void at_give_up(int site, volatile int *abort_flag, int *errword)
{
    if (!site || *abort_flag) return;
    *abort_flag = 1;
    if (errword && atomicCAS(errword, 0, 200) == 0) { errword[1] = site; errword[2] = (int)blockIdx.x; }
}
__device__ __forceinline__ bool at_error_seen(const int *errword) { return errword && *reinterpret_cast<const volatile int *>(errword) != 0; }

// 2^x on the special-function unit (ex2.approx: 2 ulp, flushes denormal results to zero, -inf -> 0)
__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// two floats in one 64-bit register: sm_100's two-wide multiply-add and add
__device__ __forceinline__ uint64_t f2_packu(uint32_t a, uint32_t b) { uint64_t r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(a), "r"(b)); return r; }
__device__ __forceinline__ uint64_t f2_pack(float a, float b) { return f2_packu(__float_as_uint(a), __float_as_uint(b)); }
__device__ __forceinline__ void f2_unpack(uint64_t v, float &a, float &b)
{
    uint32_t x, y;
    asm("mov.b64 {%0, %1}, %2;" : "=r"(x), "=r"(y) : "l"(v));
    a = __uint_as_float(x); b = __uint_as_float(y);
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) { uint64_t r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) { uint64_t r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }

}  // namespace qlmb
