// Launch arguments of the projections with 4-bit weights, and their launchers.
#pragma once

#include "host_util.h"
#include "sm100_ptx.cuh"
#include "w4_plan.h"

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
    bool out_f32, out_by_4;              // four channels of a row at once: base and rows are aligned for it
    int* status;
};

// tcgen05: scales are asked for a step ahead, which is less than memory takes: they are fetched into the L2 this many groups ahead of that (8192 x 32768: 74 us without, 60 with).
constexpr int W4_AHEAD = 12;
__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" :: "l"(p)); }

__device__ __forceinline__ void store_sum(const W4Args& a, float v, int m, int n)
{
    if (n >= a.d_out) return;
    if (a.out_f32) static_cast<float*>(a.out)[m * a.out_stride + n] = v;
    else static_cast<__half*>(a.out)[m * a.out_stride + n] = __float2half_rn(v);
}

// Of four neighbouring channels, the first a multiple of four.
__device__ __forceinline__ void store_sum4(const W4Args& a, const float4& v, int m, int n)
{
    const long long at = m * a.out_stride + n;
    if (n + 3 < a.d_out && a.out_by_4) {
        if (a.out_f32) *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = v;
        else *reinterpret_cast<uint2*>(static_cast<__half*>(a.out) + at) = make_uint2(pack_f16x2(v.x, v.y), pack_f16x2(v.z, v.w));
    } else {
        store_sum(a, v.x, m, n);
        store_sum(a, v.y, m, n + 1);
        store_sum(a, v.z, m, n + 2);
        store_sum(a, v.w, m, n + 3);
    }
}

// Sums [rows][block] in the shared memory of a cluster's blocks, added in their order and stored: every block has an equal share. All that is to be added is asked for
// before the first addition: a word from another SM's shared memory takes 400 cycles (64 rows x 256 channels of 6 blocks one after another: 3.7 us).
__device__ __forceinline__ void store_sums(const W4Args& a, const float* sum, int rows, int block, int parts, int part, int m0, int n0)
{
    for (int e = part * (int)blockDim.x + (int)threadIdx.x; e < rows * block; e += parts * (int)blockDim.x) {
        float y[8];
        #pragma unroll
        for (int q = 0; q < 8; q++) {
            y[q] = 0.f;
            if (q < parts) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(y[q]) : "r"(cluster_addr(sum + e, (uint32_t)q)));
        }
        float v = y[0];
        #pragma unroll
        for (int q = 1; q < 8; q++) v += y[q];
        store_sum(a, v, m0 + e / block, n0 + e % block);
    }
}

// tcgen05 over tiles of up to 64 rows (proj_w4_tc_sm100.cu).
int w4_tc_plan(const W4Args& a, int group, W4Division& to);
int w4_tc_launch(const W4Args& a, int group, const W4Division& to, cudaStream_t stream);

}  // namespace efa
