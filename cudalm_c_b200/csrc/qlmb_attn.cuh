// Shared by the attention kernels (qlmb_attn.cu, qlmb_prefix.cu): their bounded wait and 2^x.
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
__device__ __forceinline__ bool at_error_seen(const int *errword) { return errword && *reinterpret_cast<const volatile int *>(errword) != 0; }

// 2^x on the special-function unit (ex2.approx: 2 ulp, flushes denormal results to zero, -inf -> 0)
__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

}  // namespace qlmb
