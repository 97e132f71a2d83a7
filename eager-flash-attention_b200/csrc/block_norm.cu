// The norms after and before a block, its gate and its residual addition in one pass over the rows. A row is held in registers by the threads that share it,
// in fp32: its sums are taken over what is there already, and nothing is read twice. Layer norms sum the squares of what is left when the mean is
// taken off, not the squares less the mean's: a mean far above the spread costs no digits.
//
// Memory is the floor: x, y, the gate, x_out and h once. GPU time in graphs of 30 calls, some milliseconds: 8192 x 4096 with a gate of every row 54.8 us, 6.1 TB/s (94 % of a copy's rate; after a second of such
// calls, at the power cap, 62, 83 %); 16384 x 1024 two layer norms 27.0 (76 %: two passes over registers between barriers), 2000 x 12000 fp32 75.7 (78 %), 1237 x 2049 fp32 8.7 (62 %: little more than
// a round); one row 3.1, of which the launch is 2.
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
    float eps, residual_scale, block_scale, inv_d;
    long long x_stride, y_stride, out_stride, h_stride, gate_stride;
    int ahead;                           // rows to the one whose inputs a block fetches into the L2
};

// How a thread has its elements. ALIGNED: chunks of eight neighbours, each 16 bytes of fp16. SHIFTED: rows that begin anywhere, but at the same place within 16
// bytes in all tensors (dense ones of an odd width): chunks from the row's first 16-byte boundary on, and what is left at both ends, 15 elements at most, one
// to a thread. SINGLE: every T-th element.
enum { ALIGNED, SHIFTED, SINGLE };

// Eight elements as they lie in memory: fp16 in four words (SINGLE: one to a word), fp32 one to a word. They are turned into numbers where they are used, so that
// nothing waits for a load before all of them are under way.
template <int W> struct Raw { uint32_t w[W]; };

// The part of a row that a thread has.
template <int T, int MODE>
struct Share {
    static constexpr int ENDS = MODE != SHIFTED ? 0 : T >= 16 ? 1 : 2;          // elements of the ends
    int lane, d, head, body;             // elements before the first boundary, chunks behind it

    __device__ __forceinline__ Share(int lane_, int d_, unsigned past /* elements from a boundary to the row's first */) : lane(lane_), d(d_)
    {
        head = MODE == SHIFTED ? (int)(8u - past) & 7 : 0;
        // Where there is a head the weights of a chunk are in two of theirs, of which the second has to be there whole.
        body = MODE == SHIFTED && head ? max(0, (d - 8) / 8) : d / 8;
    }
    __device__ __forceinline__ bool has(int chunk) const { return MODE == SINGLE || chunk * T + lane < body; }
    __device__ __forceinline__ int at(int chunk) const { return head + (chunk * T + lane) * 8; }                  // first element of a chunk
    __device__ __forceinline__ int single(int chunk, int i) const { return (chunk * 8 + i) * T + lane; }
    // Element k of the ends, d or more: there is none.
    __device__ __forceinline__ int end(int k) const { const int j = k * T + lane; return j < head ? j : j + 8 * body; }
};

// Two fp32 at a time (the same roundings as one by one): half of the arithmetic, of which rows that are normalised twice have as much as memory has bytes.
__device__ __forceinline__ float2 two(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 from_bits(unsigned long long x) { return *reinterpret_cast<float2*>(&x); }
__device__ __forceinline__ unsigned long long bits(float2 x) { return *reinterpret_cast<unsigned long long*>(&x); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { unsigned long long r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b))); return from_bits(r); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { unsigned long long r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b))); return from_bits(r); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)), "l"(bits(c)));
    return from_bits(r);
}

// e = exp(-|g|) does not overflow, and e / (1 + e) or 1 / (1 + e) is the sigmoid: 1 / (1 + exp(-g)) is nothing below -87.3, where a large value is not yet small. All
// of it 2^24 times itself, so that an e down to 2^-150 is a normal number.
__device__ __forceinline__ float sigmoid(float g)
{
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fmaf(g < 0.f ? g : -g, 1.44269504f, 24.f)));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(e + 16777216.f));
    return (g < 0.f ? e : 16777216.f) * r;
}
// v times the sigmoid of g: in pairs where the threads have whole chunks (calls of 8192 x 4096 62.4 us one by one, 62.1 so); elsewhere pairs cost registers that there are not.
template <bool PAIRS> __device__ __forceinline__ float2 gated(float2 v, float2 g)
{
    if constexpr (!PAIRS) return make_float2(v.x * sigmoid(g.x), v.y * sigmoid(g.y));
    const float2 t = fma2(make_float2(fabsf(g.x), fabsf(g.y)), two(-1.44269504f), two(24.f));
    float2 e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(t.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(t.y));
    const float2 sum = add2(e, two(16777216.f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(sum.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(sum.y));
    return mul2(v, mul2(make_float2(g.x < 0.f ? e.x : 16777216.f, g.y < 0.f ? e.y : 16777216.f), r));
}

__device__ __forceinline__ float element(const void* row, bool f32, int e) { return f32 ? static_cast<const float*>(row)[e] : __half2float(static_cast<const __half*>(row)[e]); }

// Streamed rows do not stay in the L1: what all rows read (KEEP; fp16) does, and is read where it is used.
template <bool KEEP = false, int T, int MODE, int W>
__device__ __forceinline__ void load8(Raw<W>& r, const void* row, bool f32, const Share<T, MODE>& p, int chunk)
{
    if constexpr (MODE == SINGLE) {
        #pragma unroll
        for (int i = 0; i < 8; i++) {
            const int e = p.single(chunk, i);
            r.w[i] = e >= p.d ? 0u : f32 ? static_cast<const uint32_t*>(row)[e] : (uint32_t)static_cast<const unsigned short*>(row)[e];
        }
    } else if (!p.has(chunk)) {
        #pragma unroll
        for (int i = 0; i < W; i++) r.w[i] = 0u;
    } else if constexpr (KEEP) {
        const uint4* const q = reinterpret_cast<const uint4*>(static_cast<const __half*>(row) + p.at(chunk) - p.head);
        const uint4 lo = q[0];
        if (MODE == ALIGNED || p.head == 0) { r.w[0] = lo.x; r.w[1] = lo.y; r.w[2] = lo.z; r.w[3] = lo.w; return; }
        // The weights begin at a boundary: the two chunks that hold the eight elements, moved by the head's bits.
        const uint4 hi = q[1];
        const uint32_t s[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
        uint32_t t[6], u[5];
        #pragma unroll
        for (int i = 0; i < 6; i++) t[i] = p.head & 4 ? s[i + 2] : s[i];
        #pragma unroll
        for (int i = 0; i < 5; i++) u[i] = p.head & 2 ? t[i + 1] : t[i];
        #pragma unroll
        for (int i = 0; i < 4; i++) r.w[i] = __funnelshift_r(u[i], u[i + 1], (p.head & 1) * 16);
    } else {
        const char* q = static_cast<const char*>(row) + (long long)p.at(chunk) * (f32 ? 4 : 2);
        asm volatile("ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]) : "l"(q) : "memory");
        if constexpr (W == 8)
            if (f32) asm volatile("ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r.w[4]), "=r"(r.w[5]), "=r"(r.w[6]), "=r"(r.w[7]) : "l"(q + 16) : "memory");
    }
}

template <int MODE, int W>
__device__ __forceinline__ void numbers(const Raw<W>& r, bool f32, float2 (&v)[4])
{
    if (W == 8 && f32) {
        #pragma unroll
        for (int i = 0; i < 4; i++) v[i] = make_float2(__uint_as_float(r.w[2 * i % W]), __uint_as_float(r.w[(2 * i + 1) % W]));
    } else {
        #pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (MODE != SINGLE) v[i] = __half22float2(*reinterpret_cast<const __half2*>(&r.w[i]));
            else v[i] = make_float2(__half2float(__ushort_as_half((unsigned short)r.w[2 * i % W])), __half2float(__ushort_as_half((unsigned short)r.w[(2 * i + 1) % W])));
        }
    }
}

__device__ __forceinline__ void store1(void* row, bool f32, int e, float v)
{
    if (f32) static_cast<float*>(row)[e] = v;
    else static_cast<__half*>(row)[e] = __float2half_rn(v);
}
template <int T, int MODE>
__device__ __forceinline__ void store8(void* row, bool f32, const Share<T, MODE>& p, int chunk, const float2 (&v)[4])
{
    if constexpr (MODE == SINGLE) {
        #pragma unroll
        for (int i = 0; i < 8; i++)
            if (p.single(chunk, i) < p.d) store1(row, f32, p.single(chunk, i), i & 1 ? v[i / 2].y : v[i / 2].x);
    } else if (p.has(chunk)) {
        if (f32) {
            float4* q = reinterpret_cast<float4*>(static_cast<float*>(row) + p.at(chunk));
            q[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
            q[1] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
        } else {
            *reinterpret_cast<uint4*>(static_cast<__half*>(row) + p.at(chunk)) =
                make_uint4(pack_f16x2(v[0].x, v[0].y), pack_f16x2(v[1].x, v[1].y), pack_f16x2(v[2].x, v[2].y), pack_f16x2(v[3].x, v[3].y));
        }
    }
}

// A row (its 16-byte pieces) asked for into the L2.
__device__ __forceinline__ void prefetch_row(const char* row, unsigned bytes)
{
    const unsigned skip = (16u - (unsigned)reinterpret_cast<uintptr_t>(row)) & 15u;
    if (bytes >= skip + 16) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" :: "l"(row + skip), "r"((bytes - skip) & ~15u) : "memory");
}

// Sum over the T threads of a row. `slot` alternates: when it comes round again all threads have passed the barrier in between.
template <int T>
__device__ __forceinline__ float row_sum(float v, float (*part)[32], int& slot)
{
    #pragma unroll
    for (int d = (T < 32 ? T : 32) / 2; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    if constexpr (T > 32) {
        constexpr int WARPS = T / 32;
        if ((threadIdx.x & 31) == 0) part[slot][threadIdx.x >> 5] = v;
        __syncthreads();
        v = part[slot][threadIdx.x & (WARPS - 1)];
        #pragma unroll
        for (int d = WARPS / 2; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
        slot ^= 1;
    }
    return v;
}

template <int NC, int T, int MODE>
__device__ __forceinline__ void normalise(float2 (&v)[NC][4], float (&ends)[2], const NormArgs& a, const Share<T, MODE>& p, const __half* weights, const __half* biases, float (*part)[32], int& slot)
{
    constexpr int ENDS = Share<T, MODE>::ENDS;
    float2 s = two(0.f);
    if (a.layer) {
        #pragma unroll
        for (int c = 0; c < NC; c++)
            #pragma unroll
            for (int i = 0; i < 4; i++) s = add2(s, v[c][i]);
        #pragma unroll
        for (int k = 0; k < ENDS; k++) s.x += ends[k];
        const float mean = row_sum<T>(s.x + s.y, part, slot) * a.inv_d;
        s = two(0.f);
        #pragma unroll
        for (int c = 0; c < NC; c++) {
            const float2 off = two(MODE == SINGLE || p.has(c) ? -mean : 0.f);   // what is behind the row stays 0
            #pragma unroll
            for (int i = 0; i < 4; i++) {
                v[c][i] = add2(v[c][i], off);
                if constexpr (MODE == SINGLE) {
                    if (p.single(c, 2 * i) >= a.d) v[c][i].x = 0.f;
                    if (p.single(c, 2 * i + 1) >= a.d) v[c][i].y = 0.f;
                }
                s = fma2(v[c][i], v[c][i], s);
            }
        }
        #pragma unroll
        for (int k = 0; k < ENDS; k++) {
            ends[k] = p.end(k) < a.d ? ends[k] - mean : 0.f;
            s.x = fmaf(ends[k], ends[k], s.x);
        }
    } else {
        #pragma unroll
        for (int c = 0; c < NC; c++)
            #pragma unroll
            for (int i = 0; i < 4; i++) s = fma2(v[c][i], v[c][i], s);
        #pragma unroll
        for (int k = 0; k < ENDS; k++) s.x = fmaf(ends[k], ends[k], s.x);
    }
    const float scale = rsqrtf(row_sum<T>(s.x + s.y, part, slot) * a.inv_d + a.eps);
    #pragma unroll
    for (int c = 0; c < NC; c++) {
        float2 g[4];
        Raw<MODE == SINGLE ? 8 : 4> w;
        #pragma unroll
        for (int i = 0; i < 4; i++) v[c][i] = mul2(v[c][i], two(scale));
        if (weights) {
            load8<true>(w, weights, false, p, c);
            numbers<MODE>(w, false, g);
            #pragma unroll
            for (int i = 0; i < 4; i++) v[c][i] = mul2(v[c][i], g[i]);
        }
        if (biases) {
            load8<true>(w, biases, false, p, c);
            numbers<MODE>(w, false, g);
            #pragma unroll
            for (int i = 0; i < 4; i++) v[c][i] = add2(v[c][i], g[i]);
        }
    }
    #pragma unroll
    for (int k = 0; k < ENDS; k++) {
        const int e = p.end(k);
        if (e >= a.d) continue;
        ends[k] *= scale;
        if (weights) ends[k] *= __half2float(weights[e]);
        if (biases) ends[k] += __half2float(biases[e]);
    }
}

// Blocks that registers are kept free for: 64 to 128 of them to a thread. A kernel that takes fewer may have one block more. Rows above 16384 (1024 threads, four chunks, 64 registers) do not fit
// whole: five of the six kernels spill 36 to 172 bytes a thread.
constexpr int blocks_per_sm(int threads, int chunks, bool lean, bool lazy)
{
    const int registers = chunks == 1 ? 64 : lazy ? 64 : chunks == 2 ? (lean ? 64 : 96) : chunks == 3 ? (lean ? 80 : 112) : 128;
    return 65536 / (registers * threads) > 0 ? 65536 / (registers * threads) : 1;
}

// A row to T threads, NC chunks of eight elements to a thread; below 32 threads several rows to a warp. All that a row reads is asked for at once; LAZY: where a thread
// has too much for that, x and the gate in their turn.
template <int T, int NC, int MODE, bool WIDE, bool LAZY>
__global__ void __launch_bounds__(T <= 32 ? 128 : T, blocks_per_sm(T <= 32 ? 128 : T, NC, MODE != SINGLE && !WIDE, LAZY))
block_norm_kernel(const NormArgs a)
{
    __shared__ float part[2][32];
    constexpr int PER_BLOCK = T <= 32 ? 128 / T : 1;
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x % T, at = blockIdx.x * PER_BLOCK + (T <= 32 ? threadIdx.x / T : 0);
    constexpr int H = MODE == SINGLE ? 8 : 4, W = MODE == SINGLE || WIDE ? 8 : 4;   // words of eight fp16, and of what may be fp32
    const bool x_f32 = WIDE && a.x_f32, y_f32 = WIDE && a.y_f32;
    int slot = 0;
    // The lanes of a warp go together: rows behind the last are the last, without a store.
    const bool there = T > 32 || at < a.rows;
    const long long row = T > 32 ? at : min(at, a.rows - 1);
    const char* const xr = static_cast<const char*>(a.x) + row * a.x_stride * (x_f32 ? 4 : 2);
    const char* const yr = static_cast<const char*>(a.y) + row * a.y_stride * (y_f32 ? 4 : 2);
    const __half* const gr = a.gate + row * a.gate_stride;
    constexpr int ENDS = Share<T, MODE>::ENDS;
    const Share<T, MODE> p(lane, a.d, (unsigned)row * (unsigned)a.x_stride & 7u);
    float2 v[NC][4];
    float ends[2] = {0.f, 0.f}, x_ends[2], g_ends[2];
    Raw<W> x[LAZY ? 1 : NC];
    Raw<H> g[LAZY ? 1 : NC];
    {
        Raw<W> y[NC];
        #pragma unroll
        for (int c = 0; c < NC; c++) {
            if (a.y) load8(y[c], yr, y_f32, p, c);
            if constexpr (!LAZY) {
                if (a.x) load8(x[c], xr, x_f32, p, c);
                if (a.gate) a.gate_stride ? load8(g[c], gr, false, p, c) : load8<true>(g[c], gr, false, p, c);
            }
        }
        #pragma unroll
        for (int k = 0; k < ENDS; k++)
            if (p.end(k) < a.d) {
                if (a.y) ends[k] = element(yr, y_f32, p.end(k));
                if (a.x) x_ends[k] = element(xr, x_f32, p.end(k));
                if (a.gate) g_ends[k] = __half2float(gr[p.end(k)]);
            }
        #pragma unroll
        for (int c = 0; c < NC; c++) numbers<MODE>(y[c], y_f32, v[c]);
    }
    // While a block has its row, memory would wait: it fetches the row of the block that will have its place (or of one of those before it, where more blocks are resident than the launch's bound says: rows
    // that somebody is reading then), as soon as its own is there (not before, which delays it). us, without / with:
    // 8192 x 4096 60.2 / 54.8, 512 x 16384 fp32 34.6 / 31.7, 1000 x 5001 fp32 25.5 / 22.6; half as far again 2 to 4 % more; several rows to a warp nothing.
    auto prefetch = [&]() {
        if (T <= 32 || lane != 0 || a.rows - a.ahead <= at) return;
        if (a.y) prefetch_row(yr + a.ahead * a.y_stride * (y_f32 ? 4 : 2), a.d * (y_f32 ? 4 : 2));
        if (a.x) prefetch_row(xr + a.ahead * a.x_stride * (x_f32 ? 4 : 2), a.d * (x_f32 ? 4 : 2));
        if (a.gate && a.gate_stride) prefetch_row(reinterpret_cast<const char*>(gr + a.ahead * a.gate_stride), a.d * 2);
    };
    if (a.post) { normalise(v, ends, a, p, a.post_w, a.post_b, part, slot); prefetch(); }
    auto summed = [&](float n, float residual) { return a.y ? fmaf(a.residual_scale, residual, a.block_scale * n) : a.residual_scale * residual; };
    char* const out = static_cast<char*>(a.x_out) + row * a.out_stride * (x_f32 ? 4 : 2);
    #pragma unroll
    for (int c = 0; c < NC; c++) {
        float2 n[4];
        if constexpr (LAZY) {
            if (a.x) load8(x[0], xr, x_f32, p, c);
            if (a.gate) a.gate_stride ? load8(g[0], gr, false, p, c) : load8<true>(g[0], gr, false, p, c);
        }
        if (a.gate) {
            numbers<MODE>(g[LAZY ? 0 : c], false, n);
            #pragma unroll
            for (int i = 0; i < 4; i++) v[c][i] = a.sigmoid ? gated<MODE == ALIGNED>(v[c][i], n[i]) : mul2(v[c][i], n[i]);
        }
        if (a.x) {
            numbers<MODE>(x[LAZY ? 0 : c], x_f32, n);
            #pragma unroll
            for (int i = 0; i < 4; i++) v[c][i] = a.y ? fma2(two(a.residual_scale), n[i], mul2(two(a.block_scale), v[c][i])) : mul2(two(a.residual_scale), n[i]);
        } else {
            #pragma unroll
            for (int i = 0; i < 4; i++) v[c][i] = mul2(v[c][i], two(a.block_scale));
        }
        if (a.x_out && there) store8(out, x_f32, p, c, v[c]);
    }
    #pragma unroll
    for (int k = 0; k < ENDS; k++) {
        if (p.end(k) >= a.d) continue;
        if (a.gate) ends[k] *= a.sigmoid ? sigmoid(g_ends[k]) : g_ends[k];
        ends[k] = a.x ? summed(ends[k], x_ends[k]) : a.block_scale * ends[k];
        if (a.x_out && there) store1(out, x_f32, p.end(k), ends[k]);
    }
    if (!a.post) prefetch();
    if (a.pre) {
        normalise(v, ends, a, p, a.pre_w, a.pre_b, part, slot);
        #pragma unroll
        for (int c = 0; c < NC; c++)
            if (there) store8(a.h + row * a.h_stride, false, p, c, v[c]);
        #pragma unroll
        for (int k = 0; k < ENDS; k++)
            if (there && p.end(k) < a.d) store1(a.h + row * a.h_stride, false, p.end(k), ends[k]);
    }
}

template <int T, int NC, bool WIDE, bool LAZY = false>
int launch_norm(const NormArgs& a, int mode, cudaStream_t stream)
{
    constexpr int PER_BLOCK = T <= 32 ? 128 / T : 1;
    const dim3 grid((unsigned)(((long long)a.rows + PER_BLOCK - 1) / PER_BLOCK));
    const auto kernel = mode == ALIGNED ? block_norm_kernel<T, NC, ALIGNED, WIDE, LAZY> : mode == SHIFTED ? block_norm_kernel<T, NC, SHIFTED, WIDE, LAZY> : block_norm_kernel<T, NC, SINGLE, WIDE, LAZY>;
    NormArgs b = a;
    b.ahead = device_sms() * blocks_per_sm(T <= 32 ? 128 : T, NC, mode != SINGLE && !WIDE, LAZY);
    EFA_CUDA(launch_value(kernel, grid, T <= 32 ? 128 : T, 0, stream, b));
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
    if (!aligned(x, p.x_dtype == EFA_F32 ? 4 : 2) || !aligned(x_out, p.x_dtype == EFA_F32 ? 4 : 2) || !aligned(y, p.y_dtype == EFA_F32 ? 4 : 2) || !aligned(h, 2) || !aligned(gate, 2) ||
        !aligned(post_w, 2) || !aligned(post_b, 2) || !aligned(pre_w, 2) || !aligned(pre_b, 2)) {
        set_error("block_norm: tensors must be aligned to their elements");
        return 2;
    }
    const void* const mem[] = {x, y, gate, post_w, post_b, pre_w, pre_b, x_out, h};
    const auto stride = [&](int64_t s) { return s ? (long long)s : (long long)p.d; };
    NormArgs a{x, y, static_cast<const __half*>(gate), static_cast<const __half*>(post_w), static_cast<const __half*>(post_b), static_cast<const __half*>(pre_w),
               static_cast<const __half*>(pre_b), x_out, static_cast<__half*>(h), rows, p.d, p.kind == EFA_NORM_LAYER, p.post != 0, h != nullptr, p.gate == EFA_GATE_SIGMOID,
               p.x_dtype == EFA_F32, p.y_dtype == EFA_F32, p.eps, p.residual_scale, p.block_scale, (float)(1.0 / p.d),
               stride(p.x_stride), stride(p.y_stride), stride(p.out_stride), stride(p.h_stride), p.gate_rows ? stride(p.gate_stride) : 0};
    const int x_elem = a.x_f32 ? 4 : 2, y_elem = a.y_f32 ? 4 : 2;
    const auto span = [&](const void* at, long long n, long long s, int elem) { return RowSpan{at, n, (long long)p.d * elem, s * elem, elem}; };
    const RowSpan outs[] = {span(x_out, rows, a.out_stride, x_elem), span(h, rows, a.h_stride, 2)};
    const RowSpan ins[] = {span(x, rows, a.x_stride, x_elem), span(y, rows, a.y_stride, y_elem), a.gate_stride ? span(gate, rows, a.gate_stride, 2) : span(gate, 1, p.d, 2),
                           span(post_w, 1, p.d, 2), span(post_b, 1, p.d, 2), span(pre_w, 1, p.d, 2), span(pre_b, 1, p.d, 2)};
    for (int o = 0; o < 2; o++)
        for (int i = 0; i < 7; i++)
            if (rows_clash(outs[o], ins[i], i < 3)) {
                static const char* const names[] = {"x", "y", "gate", "post_w", "post_b", "pre_w", "pre_b"};
                set_error("block_norm: %s overlaps %s, and is not the same rows of the same type", o ? "h" : "x_out", names[i]);
                return 2;
            }
    if (rows_clash(outs[0], outs[1], true)) { set_error("block_norm: x_out and h overlap"); return 2; }
    if (int rc = check_memory("block_norm", mem, 9)) return rc;
    bool aligned = true, alike = true;
    for (const void* q : mem) aligned = aligned && aligned16(q);
    const long long strides[] = {x ? a.x_stride : a.y_stride, y ? a.y_stride : a.x_stride, x_out ? a.out_stride : a.x_stride, h ? a.h_stride : a.x_stride, gate && a.gate_stride ? a.gate_stride : a.x_stride};
    for (const long long t : strides) alike = alike && (t - strides[0]) % 8 == 0;
    a.x_stride = strides[0];
    const int mode = !aligned || !alike ? SINGLE : strides[0] % 8 == 0 && p.d % 8 == 0 ? ALIGNED : SHIFTED;
    // Threads to a row and chunks to a thread by d and the types alone, not by the number of rows: two chunks where all is fp16, one of fp32 (twice the registers), three where that many
    // threads would have half a chunk. us, one chunk / two / four: fp16 8192 x 4096 (one set of tensors) 59.4 / 52.7 / 55.9, 16384 x 1024 31.0 / 26.9 / 31.3; fp32 1237 x 4096 13.4 / 14.1 / 16.9, 2000 x 1024
    // 7.2 / 7.5 / 9.4; one / three: 1000 x 5001 28.9 / 22.7, 2000 x 2560 18.5 / 17.7; two of 1024 threads / three or four of 512: 2000 x 12000 78.2 / 75.7, 512 x 16384 32.4 / 33.6.
    const int d = mode == SINGLE ? p.d : p.d / 8 * 8;          // in chunks; the ends of a row are extra
    if (a.x_f32 || a.y_f32) {
        if (d <= 64) return launch_norm<8, 1, true>(a, mode, stream);
        if (d <= 128) return launch_norm<16, 1, true>(a, mode, stream);
        if (d <= 256) return launch_norm<32, 1, true>(a, mode, stream);
        if (d <= 512) return launch_norm<64, 1, true>(a, mode, stream);
        if (d <= 1024) return launch_norm<128, 1, true>(a, mode, stream);
        if (d <= 2048) return launch_norm<256, 1, true>(a, mode, stream);
        if (d <= 128 * 3 * 8) return launch_norm<128, 3, true>(a, mode, stream);
        if (d <= 4096) return launch_norm<512, 1, true>(a, mode, stream);
        if (d <= 256 * 3 * 8) return launch_norm<256, 3, true>(a, mode, stream);
        if (d <= 8192) return launch_norm<1024, 1, true>(a, mode, stream);
        if (d <= 512 * 3 * 8) return launch_norm<512, 3, true>(a, mode, stream);
        if (d <= 16384) return launch_norm<1024, 2, true>(a, mode, stream);
        return launch_norm<1024, 4, true, true>(a, mode, stream);
    }
    if (d <= 64) return launch_norm<8, 1, false>(a, mode, stream);
    if (d <= 128) return launch_norm<16, 1, false>(a, mode, stream);
    if (d <= 256) return launch_norm<32, 1, false>(a, mode, stream);
    if (d <= 512) return launch_norm<32, 2, false>(a, mode, stream);
    if (d <= 1024) return launch_norm<64, 2, false>(a, mode, stream);
    if (d <= 2048) return launch_norm<128, 2, false>(a, mode, stream);
    if (d <= 128 * 3 * 8) return launch_norm<128, 3, false>(a, mode, stream);
    if (d <= 4096) return launch_norm<256, 2, false>(a, mode, stream);
    if (d <= 256 * 3 * 8) return launch_norm<256, 3, false>(a, mode, stream);
    if (d <= 8192) return launch_norm<512, 2, false>(a, mode, stream);
    if (d <= 512 * 3 * 8) return launch_norm<512, 3, false>(a, mode, stream);
    if (d <= 16384) return launch_norm<512, 4, false>(a, mode, stream);
    return launch_norm<1024, 4, false, true>(a, mode, stream);
}

}  // namespace efa
