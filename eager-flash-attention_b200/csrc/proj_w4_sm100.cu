// Projections of few rows with weights of 4 bits and group scales: reading the weights is the time. out[m][n] = sum over groups g of s[g][n] * sum over
// the group's k of x[m][k] * (code[n][k] - zero[g][n]).
//
// mma.sync m16n8k16 with the weights as the side of 16 (output channels) and the rows of X as the side of 8: one token uses an eighth of it, which costs
// nothing while memory is the time. The order of k within a group is free as long as both sides agree on it, so codes go from memory to a fragment as they
// lie: a lane's four bytes are eight neighbouring k of one channel, `(word >> 4 i) & 0x000f000f` is the pair (k + i, k + i + 4) of two products' fragments, and x is
// paired alike. A code c becomes the fp16 number 1024 + c (or 1024 + 16 c, times 1/16) by one logical operation, and c - zero exactly by one more. All
// four lanes that share a channel must be in one group: 16, 8 or 4 bytes to a lane and load for groups of 128, 64 or 32.
#include "host_util.h"
#include "serving.h"
#include "sm100_ptx.cuh"

#include <algorithm>
#include <climits>

namespace efa {

namespace {

constexpr int W4_UNIT = 128;            // k that a warp takes at a time
constexpr int W4_ROWS = 64;             // rows of a tile

struct W4Args {
    const uint8_t* codes;
    const __half* scales;
    const uint8_t* zeros;
    const __half* X;
    void* out;
    int rows, d_in, d_out;
    long long code_stride, scale_stride, zero_stride, x_stride, out_stride;
    bool out_f32;
};

__device__ __forceinline__ uint32_t lop_and_or(uint32_t a, uint32_t mask, uint32_t with)
{
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(a), "r"(mask), "r"(with));     // (a & mask) | with
    return r;
}
__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b)
{
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c)
{
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}

// Eight codes to four pairs (i, i + 4) of numbers code - zero. low: 1024 + zero twice; high: -(64 + zero) twice.
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t low, uint32_t high, uint32_t (&f)[4])
{
    constexpr uint32_t MAGIC = 0x64006400u, SIXTEENTH = 0x2c002c00u;
    const uint32_t v = w >> 8;
    f[0] = sub2(lop_and_or(w, 0x000f000fu, MAGIC), low);
    f[1] = fma2(lop_and_or(w, 0x00f000f0u, MAGIC), SIXTEENTH, high);
    f[2] = sub2(lop_and_or(v, 0x000f000fu, MAGIC), low);
    f[3] = fma2(lop_and_or(v, 0x00f000f0u, MAGIC), SIXTEENTH, high);
}

__device__ __forceinline__ void mma_w4(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// A block: 16 MT channels, 8 NT rows, all k, its warps (and the blocks of its cluster, along z) taking units of 128 k in turn, added at the end in shared memory in the
// order of the warps and blocks.
template <int G, int MT, int NT>
__global__ void __launch_bounds__(256)
proj_w4_kernel(const W4Args a)
{
    constexpr int SUBS = W4_UNIT / G, WORDS = G / 32;          // groups of a unit, words of codes of a lane and group
    extern __shared__ float sum[];                             // [warp][8 NT][16 MT]
    pdl_wait();
    pdl_trigger();
    const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * 16 * MT, m0 = blockIdx.y * W4_ROWS;
    const int parts = gridDim.z, part = parts > 1 ? (int)cluster_rank() : 0;
    const int units = (a.d_in + W4_UNIT - 1) / W4_UNIT;
    const long long shares = (long long)warps * parts, share = (long long)part * warps + warp;
    const int u0 = (int)(units * share / shares), u1 = (int)(units * (share + 1) / shares);

    const uint8_t* row[MT][2];
    int channel[MT][2];
    #pragma unroll
    for (int m = 0; m < MT; m++)
        #pragma unroll
        for (int h = 0; h < 2; h++) {
            channel[m][h] = min(n0 + 16 * m + 8 * h + g, a.d_out - 1);
            row[m][h] = a.codes + channel[m][h] * a.code_stride + t * (G / 8);
        }
    const __half* x[NT];
    #pragma unroll
    for (int n = 0; n < NT; n++) x[n] = m0 + 8 * n + g < a.rows ? a.X + (long long)(m0 + 8 * n + g) * a.x_stride + t * (G / 4) : nullptr;

    float acc[MT][NT][4] = {};
    for (int u = u0; u < u1; u++) {
        #pragma unroll
        for (int s = 0; s < SUBS; s++) {
            const int k = u * W4_UNIT + s * G;
            if (k >= a.d_in) break;
            const long long group = k / G;
            uint32_t w[MT][2][WORDS];
            float scale[MT][2];
            uint32_t low[MT][2], high[MT][2];
            #pragma unroll
            for (int m = 0; m < MT; m++)
                #pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint8_t* p = row[m][h] + (k >> 1);
                    if constexpr (WORDS == 4) {
                        const uint4 q = *reinterpret_cast<const uint4*>(p);
                        w[m][h][0] = q.x; w[m][h][1] = q.y; w[m][h][2] = q.z; w[m][h][3] = q.w;
                    } else if constexpr (WORDS == 2) {
                        const uint2 q = *reinterpret_cast<const uint2*>(p);
                        w[m][h][0] = q.x; w[m][h][1] = q.y;
                    } else w[m][h][0] = *reinterpret_cast<const uint32_t*>(p);
                    scale[m][h] = __half2float(a.scales[group * a.scale_stride + channel[m][h]]);
                    const uint32_t z = a.zeros ? a.zeros[group * a.zero_stride + channel[m][h]] : 8u;
                    const uint32_t hl = __half_as_ushort(__uint2half_rn(1024u + z)), hh = __half_as_ushort(__int2half_rn(-(int)(64u + z)));
                    low[m][h] = hl | hl << 16;
                    high[m][h] = hh | hh << 16;
                }
            float part_sum[MT][NT][4] = {};
            #pragma unroll
            for (int i = 0; i < WORDS; i++) {
                uint32_t f[MT][2][4];
                #pragma unroll
                for (int m = 0; m < MT; m++) {
                    codes_to_f16(w[m][0][i], low[m][0], high[m][0], f[m][0]);
                    codes_to_f16(w[m][1][i], low[m][1], high[m][1], f[m][1]);
                }
                #pragma unroll
                for (int n = 0; n < NT; n++) {
                    uint4 q = make_uint4(0u, 0u, 0u, 0u);
                    if (x[n]) q = *reinterpret_cast<const uint4*>(x[n] + k + 8 * i);
                    const uint32_t b0 = __byte_perm(q.x, q.z, 0x5410), b1 = __byte_perm(q.x, q.z, 0x7632);
                    const uint32_t b2 = __byte_perm(q.y, q.w, 0x5410), b3 = __byte_perm(q.y, q.w, 0x7632);
                    #pragma unroll
                    for (int m = 0; m < MT; m++) {
                        mma_w4(part_sum[m][n], f[m][0][0], f[m][1][0], f[m][0][1], f[m][1][1], b0, b1);
                        mma_w4(part_sum[m][n], f[m][0][2], f[m][1][2], f[m][0][3], f[m][1][3], b2, b3);
                    }
                }
            }
            #pragma unroll
            for (int m = 0; m < MT; m++)
                #pragma unroll
                for (int n = 0; n < NT; n++)
                    #pragma unroll
                    for (int i = 0; i < 4; i++) acc[m][n][i] = fmaf(scale[m][i >> 1], part_sum[m][n][i], acc[m][n][i]);
        }
    }
    constexpr int TILE = 16 * MT * 8 * NT;
    float* const mine = sum + warp * TILE;
    #pragma unroll
    for (int m = 0; m < MT; m++)
        #pragma unroll
        for (int n = 0; n < NT; n++)
            #pragma unroll
            for (int i = 0; i < 4; i++) mine[(8 * n + 2 * t + (i & 1)) * (16 * MT) + 16 * m + 8 * (i >> 1) + g] = acc[m][n][i];
    __syncthreads();
    for (int e = threadIdx.x; e < TILE; e += blockDim.x) {
        float v = sum[e];
        for (int w = 1; w < warps; w++) v += sum[w * TILE + e];
        sum[e] = v;
    }
    if (parts > 1) cluster_sync(); else __syncthreads();
    for (int e = part * (int)blockDim.x + threadIdx.x; e < TILE; e += parts * blockDim.x) {
        float v = 0.f;
        if (parts > 1) {
            for (int q = 0; q < parts; q++) {
                float y;
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(y) : "r"(cluster_addr(sum + e, q)));
                v += y;
            }
        } else v = sum[e];
        const int m = m0 + e / (16 * MT), n = n0 + e % (16 * MT);
        if (m < a.rows && n < a.d_out) {
            if (a.out_f32) static_cast<float*>(a.out)[m * a.out_stride + n] = v;
            else static_cast<__half*>(a.out)[m * a.out_stride + n] = __float2half_rn(v);
        }
    }
    if (parts > 1) cluster_sync();                             // the others may still read this block's sums
}

template <int G, int MT, int NT>
int launch_w4(const W4Args& a, cudaStream_t stream)
{
    const int tiles = (a.d_out + 16 * MT - 1) / (16 * MT), units = (a.d_in + W4_UNIT - 1) / W4_UNIT;
    const int warps = 8;
    int cluster = 1;
    while (cluster < 8 && cluster * 2 * warps <= units && (long long)tiles * cluster < 2 * device_sms()) cluster *= 2;
    const dim3 grid(tiles, (a.rows + W4_ROWS - 1) / W4_ROWS, cluster);
    const size_t smem = (size_t)warps * 16 * MT * 8 * NT * sizeof(float);
    static bool set = false;
    if (smem > 48 * 1024 && !set) { EFA_CUDA(cudaFuncSetAttribute(proj_w4_kernel<G, MT, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem)); set = true; }
    EFA_CUDA(launch_value(proj_w4_kernel<G, MT, NT>, grid, warps * 32, smem, stream, a));
    return 0;
}

template <int G>
int launch_group(const W4Args& a, cudaStream_t stream)
{
    const int rows = std::min(a.rows, W4_ROWS);
    if (rows <= 8) return launch_w4<G, 2, 1>(a, stream);
    if (rows <= 16) return launch_w4<G, 2, 2>(a, stream);
    if (rows <= 32) return launch_w4<G, 2, 4>(a, stream);
    return launch_w4<G, 2, 8>(a, stream);
}

}  // namespace

const char* w4_check(const efa_w4& w)
{
    if (w.group != 32 && w.group != 64 && w.group != 128) return "w4: group must be 32, 64 or 128";
    if (w.d_in < 1 || w.d_in % w.group) return "w4: d_in must be a positive multiple of group";
    if (w.d_out < 1) return "w4: d_out must be positive";
    if (w.d_in > 1 << 24 || w.d_out > 1 << 24) return "w4: sizes too large";
    if (!w.codes || !w.scales) return "w4: codes and scales must not be null";
    if (!aligned16(w.codes)) return "w4: codes must be 16-byte aligned";
    if ((reinterpret_cast<uintptr_t>(w.scales) & 1) != 0) return "w4: scales must be aligned to their elements";
    if (w.code_stride != 0 && (w.code_stride < w.d_in / 2 || w.code_stride % 16)) return "w4: code_stride must be 0 or a multiple of 16 that holds a row";
    if (w.scale_stride != 0 && w.scale_stride < w.d_out) return "w4: scale_stride must be 0 or at least d_out";
    if (w.zero_stride != 0 && w.zero_stride < w.d_out) return "w4: zero_stride must be 0 or at least d_out";
    return nullptr;
}

int project_w4(const void* X, long long x_stride, const efa_w4& w, void* out, int out_dtype, long long out_stride, int rows, cudaStream_t stream)
{
    if (const char* why = w4_check(w)) { set_error("project_w4: %s", why); return 2; }
    if (rows < 0 || rows > 1 << 20) { set_error("project_w4: rows must be from 0 to 2^20 (got %d)", rows); return 2; }
    if (out_dtype != EFA_F16 && out_dtype != EFA_F32) { set_error("project_w4: out must be EFA_F16 or EFA_F32"); return 2; }
    if (x_stride != 0 && (x_stride < w.d_in || x_stride % 8)) { set_error("project_w4: x_stride must be 0 or a multiple of 8 that holds d_in"); return 2; }
    if (out_stride != 0 && out_stride < w.d_out) { set_error("project_w4: out_stride must be 0 or at least d_out"); return 2; }
    if (rows == 0) return 0;
    if (!X || !out) { set_error("project_w4: X or out is null"); return 2; }
    if (!aligned16(X) || (reinterpret_cast<uintptr_t>(out) & (out_dtype == EFA_F16 ? 1 : 3)) != 0) { set_error("project_w4: X must be 16-byte aligned, out to its elements"); return 2; }
    const void* const mem[] = {X, w.codes, w.scales, w.zeros, out};
    if (int rc = check_memory("project_w4", mem, 5)) return rc;
    const W4Args a{w.codes, static_cast<const __half*>(w.scales), w.zeros, static_cast<const __half*>(X), out, rows, w.d_in, w.d_out,
                   w.code_stride ? w.code_stride : w.d_in / 2, w.scale_stride ? w.scale_stride : w.d_out, w.zero_stride ? w.zero_stride : w.d_out,
                   x_stride ? x_stride : w.d_in, out_stride ? out_stride : w.d_out, out_dtype == EFA_F32};
    return w.group == 128 ? launch_group<128>(a, stream) : w.group == 64 ? launch_group<64>(a, stream) : launch_group<32>(a, stream);
}

}  // namespace efa
