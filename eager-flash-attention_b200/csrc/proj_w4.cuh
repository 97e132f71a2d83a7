// Launch arguments of the projections with 4-bit weights, and their launchers.
#pragma once

#include "host_util.h"
#include "sm100_ptx.cuh"

namespace efa {

constexpr int W4_UNIT = 128;            // k that are copied at a time: 64 bytes of each channel's codes

struct W4Args {
    const uint8_t* codes;
    const __half* scales;
    const uint8_t* zeros;
    const __half* X;
    void* out;
    int rows, d_in, d_out;
    long long code_stride, scale_stride, zero_stride, x_stride, out_stride;
    bool out_f32;
    int* status;
};

// Scales are asked for a step ahead, which is less than memory takes: they are fetched into the L2 this many groups ahead of that.
constexpr int W4_AHEAD = 12;
__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" :: "l"(p)); }

// mbar_wait (sm100_ptx.cuh) with a hint that the hardware may hold the thread for that long: many warps wait here beside others that need their issue slots.
__device__ __forceinline__ bool mbar_wait_idle(uint64_t* bar, uint32_t parity, volatile int* abort_word, int site)
{
    unsigned long long t0 = 0;
    while (true) {
        uint32_t done;
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n"
            "selp.u32 %0, 1, 0, p;\n"
            "}\n" : "=r"(done) : "r"(smem_u32(bar)), "r"(parity), "r"(20000u) : "memory");
        if (done) return true;
        if (*abort_word != 0) return false;
        const unsigned long long now = globaltimer_ns();
        if (t0 == 0) t0 = now;
        else if (now - t0 > kWaitLimitNs) {
            *abort_word = site;
            return false;
        }
    }
}

// tcgen05 over tiles of up to 64 rows (proj_w4_tc_sm100.cu).
int w4_tc_launch(const W4Args& a, int group, cudaStream_t stream);

}  // namespace efa
