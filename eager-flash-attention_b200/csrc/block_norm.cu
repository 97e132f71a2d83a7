// The norms after and before a block, its gate and its residual addition in one pass over the rows. A row is held in registers by the threads that share it,
// in fp32: its sums are taken over what is there already, and nothing is read twice. Layer norms sum the squares of what is left when the mean is
// taken off, not the squares less the mean's: a mean far above the spread costs no digits.
#include "host_util.h"
#include "serving.h"
#include "sm100_ptx.cuh"

#include <algorithm>
#include <climits>
#include <cmath>

namespace efa {

namespace {

constexpr int BN_MAX_D = 32768;

struct NormArgs {
    const void* x;
    const void* y;
    const __half* gate;
    const __half* post_w;
    const __half* post_b;
    const __half* pre_w;
    const __half* pre_b;
    void* x_out;
    __half* h;
    int rows, d;
    bool layer, post, pre, sigmoid, x_f32, y_f32;
    float eps, residual_scale, block_scale;
    long long x_stride, y_stride, out_stride, h_stride, gate_stride;
};

// Elements of a row that a thread has: VEC, chunks of eight next to one another; else every threads-th element.
template <bool VEC>
struct Place {
    int lane, threads;
    __device__ __forceinline__ int at(int chunk, int i) const { return VEC ? (chunk * threads + lane) * 8 + i : (chunk * 8 + i) * threads + lane; }
};

template <bool VEC>
__device__ __forceinline__ void load8(const void* base, bool f32, long long row0, const Place<VEC>& p, int chunk, int d, float (&v)[8])
{
    if constexpr (VEC) {
        const int at = p.at(chunk, 0);
        if (at >= d) {
            #pragma unroll
            for (int i = 0; i < 8; i++) v[i] = 0.f;
            return;
        }
        if (f32) {
            const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(base) + row0 + at);
            const float4 a = q[0], b = q[1];
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            const uint4 q = *reinterpret_cast<const uint4*>(static_cast<const __half*>(base) + row0 + at);
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
            #pragma unroll
            for (int i = 0; i < 4; i++) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                v[2 * i] = f.x; v[2 * i + 1] = f.y;
            }
        }
    } else {
        #pragma unroll
        for (int i = 0; i < 8; i++) {
            const int at = p.at(chunk, i);
            v[i] = at >= d ? 0.f : f32 ? static_cast<const float*>(base)[row0 + at] : __half2float(static_cast<const __half*>(base)[row0 + at]);
        }
    }
}

template <bool VEC>
__device__ __forceinline__ void store8(void* base, bool f32, long long row0, const Place<VEC>& p, int chunk, int d, const float (&v)[8])
{
    if constexpr (VEC) {
        const int at = p.at(chunk, 0);
        if (at >= d) return;
        if (f32) {
            float4* q = reinterpret_cast<float4*>(static_cast<float*>(base) + row0 + at);
            q[0] = make_float4(v[0], v[1], v[2], v[3]);
            q[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            *reinterpret_cast<uint4*>(static_cast<__half*>(base) + row0 + at) =
                make_uint4(pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3]), pack_f16x2(v[4], v[5]), pack_f16x2(v[6], v[7]));
        }
    } else {
        #pragma unroll
        for (int i = 0; i < 8; i++) {
            const int at = p.at(chunk, i);
            if (at >= d) continue;
            if (f32) static_cast<float*>(base)[row0 + at] = v[i];
            else static_cast<__half*>(base)[row0 + at] = __float2half_rn(v[i]);
        }
    }
}

// Sum over the threads of a row: a warp (WARP), or the block. `slot` is another one each time until all threads have passed the barrier after next.
template <bool WARP>
__device__ __forceinline__ float row_sum(float v, float (*part)[32], int& slot)
{
    #pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    if constexpr (WARP) return v;
    const int lane = threadIdx.x & 31;
    if (lane == 0) part[slot][threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < (int)(blockDim.x >> 5) ? part[slot][lane] : 0.f;
    #pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    slot ^= 1;
    return v;
}

template <int NC, bool VEC, bool WARP>
__device__ __forceinline__ void normalise(float (&v)[NC][8], const NormArgs& a, const Place<VEC>& p, const __half* w, const __half* b, float (*part)[32], int& slot)
{
    float s = 0.f;
    if (a.layer) {
        #pragma unroll
        for (int c = 0; c < NC; c++)
            #pragma unroll
            for (int i = 0; i < 8; i++) s += v[c][i];
        const float mean = row_sum<WARP>(s, part, slot) / (float)a.d;
        s = 0.f;
        #pragma unroll
        for (int c = 0; c < NC; c++)
            #pragma unroll
            for (int i = 0; i < 8; i++) {
                v[c][i] = p.at(c, i) < a.d ? v[c][i] - mean : 0.f;
                s += v[c][i] * v[c][i];
            }
    } else {
        #pragma unroll
        for (int c = 0; c < NC; c++)
            #pragma unroll
            for (int i = 0; i < 8; i++) s += v[c][i] * v[c][i];
    }
    const float scale = rsqrtf(row_sum<WARP>(s, part, slot) / (float)a.d + a.eps);
    #pragma unroll
    for (int c = 0; c < NC; c++) {
        float g[8];
        if (w) load8<VEC>(w, false, 0, p, c, a.d, g);
        #pragma unroll
        for (int i = 0; i < 8; i++) v[c][i] = w ? v[c][i] * scale * g[i] : v[c][i] * scale;
        if (b) {
            load8<VEC>(b, false, 0, p, c, a.d, g);
            #pragma unroll
            for (int i = 0; i < 8; i++) v[c][i] += g[i];
        }
    }
}

// A row to a block, or (WARP) to a warp, NC chunks of eight elements to a thread.
template <int NC, bool VEC, bool WARP>
__global__ void __launch_bounds__(WARP ? 128 : NC == 1 ? 512 : 1024)
block_norm_kernel(const NormArgs a)
{
    __shared__ float part[2][32];
    pdl_wait();
    pdl_trigger();
    const int per_block = WARP ? blockDim.x >> 5 : 1;
    const Place<VEC> p{WARP ? (int)(threadIdx.x & 31) : (int)threadIdx.x, WARP ? 32 : (int)blockDim.x};
    int slot = 0;
    for (int row = blockIdx.x * per_block + (WARP ? threadIdx.x >> 5 : 0); row < a.rows; row += gridDim.x * per_block) {
        // v: the block's output, then the sum. x is asked for together with y, so that it is there when the first norm is done; not where a thread
        // has 32 elements of each.
        float v[NC][8], x[NC == 4 ? 1 : NC][8];
        #pragma unroll
        for (int c = 0; c < NC; c++) {
            if (a.y) load8<VEC>(a.y, a.y_f32, row * a.y_stride, p, c, a.d, v[c]);
            if (NC < 4 && a.x) load8<VEC>(a.x, a.x_f32, row * a.x_stride, p, c, a.d, x[NC == 4 ? 0 : c]);
        }
        if (a.y && a.post) normalise<NC, VEC, WARP>(v, a, p, a.post_w, a.post_b, part, slot);
        #pragma unroll
        for (int c = 0; c < NC; c++) {
            float g[8], (&xc)[8] = x[NC == 4 ? 0 : c];
            if (NC == 4 && a.x) load8<VEC>(a.x, a.x_f32, row * a.x_stride, p, c, a.d, xc);
            if (a.gate) load8<VEC>(a.gate, false, row * a.gate_stride, p, c, a.d, g);
            #pragma unroll
            for (int i = 0; i < 8; i++) {
                float n = v[c][i] * a.block_scale;
                if (a.gate) n = a.sigmoid ? n / (1.f + __expf(-g[i])) : n * g[i];
                v[c][i] = !a.y ? a.residual_scale * xc[i] : a.x ? fmaf(a.residual_scale, xc[i], n) : n;
            }
            if (a.x_out) store8<VEC>(a.x_out, a.x_f32, row * a.out_stride, p, c, a.d, v[c]);
        }
        if (a.pre) {
            normalise<NC, VEC, WARP>(v, a, p, a.pre_w, a.pre_b, part, slot);
            #pragma unroll
            for (int c = 0; c < NC; c++) store8<VEC>(a.h, false, row * a.h_stride, p, c, a.d, v[c]);
        }
    }
}

template <int NC, bool VEC>
int launch_norm(const NormArgs& a, int threads, bool warp, cudaStream_t stream)
{
    const int per_block = warp ? threads / 32 : 1;
    const unsigned blocks = (unsigned)std::min<long long>((a.rows + per_block - 1) / per_block, (long long)device_sms() * 32);
    EFA_CUDA(warp ? launch_value(block_norm_kernel<NC, VEC, true>, dim3(blocks), threads, 0, stream, a)
                  : launch_value(block_norm_kernel<NC, VEC, false>, dim3(blocks), threads, 0, stream, a));
    return 0;
}

}  // namespace

const char* block_norm_check(const efa_block_norm_params& p, int rows)
{
    if (rows < 0) return "block_norm: negative number of rows";
    if (p.d < 1 || p.d > BN_MAX_D) return "block_norm: d must be from 1 to 32768";
    if (p.kind != EFA_NORM_RMS && p.kind != EFA_NORM_LAYER) return "block_norm: kind must be EFA_NORM_RMS or EFA_NORM_LAYER";
    if (p.gate != EFA_GATE_NONE && p.gate != EFA_GATE_PLAIN && p.gate != EFA_GATE_SIGMOID) return "block_norm: gate must be EFA_GATE_NONE, EFA_GATE_PLAIN or EFA_GATE_SIGMOID";
    if ((p.x_dtype != EFA_F16 && p.x_dtype != EFA_F32) || (p.y_dtype != EFA_F16 && p.y_dtype != EFA_F32)) return "block_norm: x and y must be EFA_F16 or EFA_F32";
    if (!std::isfinite(p.eps) || p.eps < 0.f) return "block_norm: eps must be finite and not negative";
    if (!std::isfinite(p.residual_scale) || !std::isfinite(p.block_scale)) return "block_norm: scales must be finite";
    for (const int64_t s : {p.x_stride, p.y_stride, p.out_stride, p.h_stride, p.gate_stride})
        if (s != 0 && s < p.d) return "block_norm: strides must be 0 or at least d";
    return nullptr;
}

int block_norm(const void* x, const void* y, const void* gate, const void* post_w, const void* post_b, const void* pre_w, const void* pre_b, void* x_out, void* h,
               int rows, const efa_block_norm_params& p, cudaStream_t stream)
{
    if (const char* why = block_norm_check(p, rows)) { set_error("%s", why); return 2; }
    if (rows == 0) return 0;
    if (!x && !y) { set_error("block_norm: x and y are null"); return 2; }
    if (!y && (p.post || p.gate != EFA_GATE_NONE)) { set_error("block_norm: a post norm or a gate needs y"); return 2; }
    if ((p.gate != EFA_GATE_NONE) != (gate != nullptr)) { set_error("block_norm: a gate's values come with its kind, and without one there are none"); return 2; }
    if (!x_out && !h) { set_error("block_norm: x_out and h are null"); return 2; }
    if (h && !p.pre) { set_error("block_norm: h is written by the pre norm only"); return 2; }
    const void* const mem[] = {x, y, gate, post_w, post_b, pre_w, pre_b, x_out, h};
    if (int rc = check_memory("block_norm", mem, 9)) return rc;
    const auto stride = [&](int64_t s) { return s ? (long long)s : (long long)p.d; };
    NormArgs a{x, y, static_cast<const __half*>(gate), static_cast<const __half*>(post_w), static_cast<const __half*>(post_b), static_cast<const __half*>(pre_w),
               static_cast<const __half*>(pre_b), x_out, static_cast<__half*>(h), rows, p.d, p.kind == EFA_NORM_LAYER, p.post != 0, h != nullptr, p.gate == EFA_GATE_SIGMOID,
               p.x_dtype == EFA_F32, p.y_dtype == EFA_F32, p.eps, p.residual_scale, p.block_scale,
               stride(p.x_stride), stride(p.y_stride), stride(p.out_stride), stride(p.h_stride), p.gate_rows ? stride(p.gate_stride) : 0};
    bool vec = p.d % 8 == 0;
    for (const void* q : mem) vec = vec && aligned16(q);
    for (const long long s : {a.x_stride, a.y_stride, a.out_stride, a.h_stride, a.gate_stride}) vec = vec && s % 8 == 0;
    const int chunks = (p.d + 7) / 8;
    const bool warp = chunks <= 128;
    const int nc = warp ? (chunks <= 32 ? 1 : chunks <= 64 ? 2 : 4) : chunks <= 512 ? 1 : chunks <= 2048 ? 2 : 4;
    const int threads = warp ? 128 : ((chunks + nc - 1) / nc + 31) / 32 * 32;
    if (vec) return nc == 1 ? launch_norm<1, true>(a, threads, warp, stream) : nc == 2 ? launch_norm<2, true>(a, threads, warp, stream) : launch_norm<4, true>(a, threads, warp, stream);
    return nc == 1 ? launch_norm<1, false>(a, threads, warp, stream) : nc == 2 ? launch_norm<2, false>(a, threads, warp, stream) : launch_norm<4, false>(a, threads, warp, stream);
}

}  // namespace efa
