// Projections with 4-bit weights on tcgen05: D[128 channels][rows] = codes (tensor memory) x X^T (shared memory), one accumulator per group of weights.
//
// The weights are the operand in tensor memory, whose lanes are channels and so threads: a thread has the codes of its channel, 64 bytes per 128 k from shared memory
// (TMA), and writes them as fp16. A code c (byte 0 of a half, the other byte 0) is the fp16 number c 2^-24 as it stands: of a word of eight codes two logical
// operations make bytes of them (odd ones 16 times themselves), a byte permutation of each two puts neighbouring k into the halves of a register, one multiplication by (1, 1/16) with an
// addition takes the zero point off, exactly. X goes to shared memory as it lies (TMA). A group's sums come back in fp32 and are added up times scale * 2^24, by warps of their own.
//
// Why not the weights in shared memory: they would be written there and read again by the tensor core, 256 bytes for 64 of codes; in tensor memory the thread that has a channel's codes
// writes them where they are used. What bounds it (8192 x 32768 in graphs of 30 calls: 64 rows 44.7 us, 3.2 TB/s, 770 TFLOP/s; after a second of them, at the power cap, 52,
// 660 TFLOP/s; 16 rows 37.9): making the operand. A unit of 128 k x 256 channels takes some 3300 warp
// instructions, 768 of them the six logical ones to a word; of its 1290 cycles the logical pipe worked 57 % and the schedulers issued 71 % with seven (odd codes shifted: 45.8 and 39.4 us). More of the operand made before the wait
// for its place needs registers that the block does not have (49 us with spills); a tile of 256 channels to an SM leaves 20 of 148 SMs without one. 4096 x 4096, 64 rows: 11.2 us, of which start
// and sums of the cluster are 5.
#include "proj_w4.cuh"

#include <algorithm>
#include <atomic>

namespace efa {

namespace {

// Two tiles of 128 channels, and seven warpgroups: two to a tile that take steps in turn and make the operand of codes, one to a tile that adds up, and one whose
// first warp copies and whose next two issue. Making the operand of one step is some 1000 cycles of one wait after another, of which the arithmetic is a fifth: it
// takes four warps to a scheduler to hide them.
constexpr int TC_THREADS = 7 * 128, TC_COLLECT = 16, TC_COPY = 24;
constexpr int TC_REGS_MAKE = 56, TC_REGS_COLLECT = 120, TC_REGS_REST = 40;      // at launch 72 each: 64512
static_assert(4 * 128 * TC_REGS_MAKE + 2 * 128 * TC_REGS_COLLECT + 128 * TC_REGS_REST <= TC_THREADS * 72, "");

template <int G, int N>
struct TcCfg {
    static constexpr int STEP = G * 64 / N < W4_UNIT ? G * 64 / N : W4_UNIT;      // k between two hand-overs: no more than 64 columns of sums
    static constexpr int GROUPS = STEP / G, STEPS = W4_UNIT / STEP;                // groups of a step, steps of a unit
    // Copies of a unit's codes of both tiles, and of X for several units: a copy costs some 200 cycles however small it is.
    static constexpr int SLOT = 256 * 64, X_BLOCK = N * 128, X_BLOCKS = N == 64 ? 2 : 8, X_UNITS = X_BLOCKS / 2, X_SLOT = X_BLOCKS * X_BLOCK;
    static constexpr int STAGES = 8, X_STAGES = N == 64 ? 6 : 2;
    static constexpr int SMEM = 1024 + STAGES * SLOT + X_STAGES * X_SLOT;
    static_assert(GROUPS * N <= 64 && STAGES * SLOT >= 256 * N * 4 && SMEM > 114 * 1024 && SMEM <= 227 * 1024, "");     // one block to an SM: it has all of the tensor memory
};

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t s)
{
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(s));
    return r;
}
__device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c)
{
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)), "l"(*reinterpret_cast<unsigned long long*>(&c)));
    return *reinterpret_cast<float2*>(&r);
}

// Eight codes to four registers (k, k + 1) of (code - zero) 2^-24; minus: -zero 2^-24 twice. Odd codes come as 16 times themselves. A selector with its high bit set copies the sign of an even
// code's byte, which is 0.
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t minus, uint32_t* f)
{
    constexpr uint32_t ONE_SIXTEENTH = 0x2c003c00u;            // 1, 1/16
    const uint32_t even = w & 0x0f0f0f0fu, odd = w & 0xf0f0f0f0u;
    f[0] = fma2(prmt(even, odd, 0x8480u), ONE_SIXTEENTH, minus);
    f[1] = fma2(prmt(even, odd, 0x8581u), ONE_SIXTEENTH, minus);
    f[2] = fma2(prmt(even, odd, 0x8682u), ONE_SIXTEENTH, minus);
    f[3] = fma2(prmt(even, odd, 0x8783u), ONE_SIXTEENTH, minus);
}

template <int G, int N>
__global__ void __launch_bounds__(TC_THREADS, 1)
proj_w4_tc_kernel(const W4Args a, int tile_channels, bool x_blocks, const __grid_constant__ CUtensorMap codes_map, const __grid_constant__ CUtensorMap x_map)
{
    using C = TcCfg<G, N>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full[C::STAGES], empty[C::STAGES], x_full[C::X_STAGES], x_empty[C::X_STAGES], a_full[2][2], d_full[2][2], d_empty[2][2];
    __shared__ uint32_t tmem_at;
    __shared__ int abort_word;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int block = 2 * tile_channels, n0 = blockIdx.x * block, m0 = blockIdx.y * 64, rows = min(a.rows - m0, N);
    const int parts = gridDim.z, part = parts > 1 ? (int)cluster_rank() : 0;
    const int units = (a.d_in + W4_UNIT - 1) / W4_UNIT, u0 = (int)((long long)units * part / parts), u1 = (int)((long long)units * (part + 1) / parts);
    const int steps = (u1 - u0) * C::STEPS;
    uint8_t* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    // Copies of unit u0 + i's codes, and of the X of a unit that begins a copy of it.
    auto copy_codes = [&](unsigned i) {
        const unsigned slot = i % C::STAGES;
        mbar_expect_tx(&full[slot], 2 * tile_channels * 64);
        tma_load_2d(smem + slot * C::SLOT, &codes_map, &full[slot], (u0 + (int)i) * (W4_UNIT / 2), n0);
    };
    auto copy_x = [&](unsigned xi) {
        const unsigned slot = xi % C::X_STAGES;
        const int first = 2 * (u0 + (int)xi * C::X_UNITS);     // of the blocks of 64 k
        uint8_t* const to = smem + C::STAGES * C::SLOT + slot * C::X_SLOT;
        mbar_expect_tx(&x_full[slot], C::X_SLOT);
        if (x_blocks) tma_load_3d(to, &x_map, &x_full[slot], 0, m0, first);
        else
            for (int j = 0; j < C::X_BLOCKS; j++) tma_load_2d(to + j * C::X_BLOCK, &x_map, &x_full[slot], (first + j) * 64, m0);
    };
    const unsigned my_units = (unsigned)(u1 - u0);
    if (warp == TC_COPY && lane == 0) {
        for (int i = 0; i < C::STAGES; i++) { mbar_init(&full[i], 1); mbar_init(&empty[i], 8); }
        for (int i = 0; i < C::X_STAGES; i++) { mbar_init(&x_full[i], 1); mbar_init(&x_empty[i], 8); }
        for (int i = 0; i < 4; i++) { mbar_init(&a_full[i >> 1][i & 1], 4); mbar_init(&d_full[i >> 1][i & 1], 1); mbar_init(&d_empty[i >> 1][i & 1], 4); }
        mbar_fence_init();
        abort_word = 0;
        tma_prefetch_desc(&codes_map);
        tma_prefetch_desc(&x_map);
    }
    if (warp == TC_COPY + 1) tmem_alloc(&tmem_at, 512);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    pdl_wait();
    pdl_trigger();

    // Tensor memory of a tile (256 columns): two buffers of the operand, 64 columns each, then two of sums. A warp sees 32 lanes of it.
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    const int r = (warp & 3) * 32 + lane;                      // channel of the tile
    const int groups = a.d_in / G, group0 = u0 * (W4_UNIT / G);
    float* const sum = reinterpret_cast<float*>(smem);         // at the end: [N][channels of the block]

    if (warp >= TC_COPY) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(TC_REGS_REST));
        if (warp == TC_COPY) {
            if (lane == 0) {
                for (unsigned i = 0; i < my_units; i++) {
                    if (i % C::X_UNITS == 0) {
                        const unsigned xi = i / C::X_UNITS;
                        if (!mbar_wait(&x_empty[xi % C::X_STAGES], (xi / C::X_STAGES & 1) ^ 1u, &abort_word, 71)) break;
                        copy_x(xi);
                    }
                    if (!mbar_wait(&empty[i % C::STAGES], (i / C::STAGES & 1) ^ 1u, &abort_word, 72)) break;
                    copy_codes(i);
                }
            }
        } else if (warp <= TC_COPY + 2) {
            // Issue, a warp to a tile: all lanes wait, one issues.
            constexpr uint32_t IDESC = idesc_f16_f32(128, N, 0, 0);
            const int tile = warp - TC_COPY - 1;
            const uint32_t tmem = tmem_at + (uint32_t)tile * 256u;
            const uint64_t x_desc = smem_desc(smem_u32(smem) + C::STAGES * C::SLOT, 16, 1024, swizzle_code(128));
            const uint32_t x_lo = (uint32_t)x_desc, x_hi = (uint32_t)(x_desc >> 32);
            const bool leader = elect_one();
            for (unsigned s = 0; s < (unsigned)steps; s++) {
                const unsigned in_unit = s % C::STEPS, buf = s & 1, unit = s / C::STEPS, xi = unit / C::X_UNITS, slot = xi % C::X_STAGES;
                const bool going = mbar_wait(&x_full[slot], (uint32_t)(xi / C::X_STAGES) & 1u, &abort_word, 73)
                                && mbar_wait(&d_empty[tile][buf], (uint32_t)(s >> 1 & 1) ^ 1u, &abort_word, 74)
                                && mbar_wait(&a_full[tile][buf], (uint32_t)(s >> 1) & 1u, &abort_word, 75);
                if (!__all_sync(0xffffffffu, going)) break;
                tc_fence_after_sync();
                if (leader) {
                    const uint32_t x = x_lo + (uint32_t)(slot * (C::X_SLOT >> 4) + unit % C::X_UNITS * (2 * C::X_BLOCK >> 4)), d = tmem + 128u + buf * 64u, w = tmem + buf * 64u;
                    #pragma unroll
                    for (int j = 0; j < C::STEP / 16; j++) {
                        const int k = in_unit * C::STEP + 16 * j;
                        tc_mma_ts_lh(d + (uint32_t)(16 * j / G) * N, w + 8u * j, x + (uint32_t)(((k >> 6) * C::X_BLOCK + (k & 63) * 2) >> 4), x_hi, IDESC, 16 * j % G ? 1u : 0u);
                    }
                    tc_commit(&d_full[tile][buf]);
                }
                __syncwarp();
            }
        }
    } else if (warp >= TC_COLLECT) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(TC_REGS_COLLECT));
        const int tile = (warp - TC_COLLECT) >> 2;
        const uint32_t tmem = tmem_at + (uint32_t)tile * 256u + 128u + lanes;
        const __half* const scales = a.scales + min(n0 + tile * tile_channels + r, a.d_out - 1);
        float2 acc[N / 2];
        #pragma unroll
        for (int i = 0; i < N / 2; i++) acc[i] = make_float2(0.f, 0.f);
        __half next[C::GROUPS] = {};
        for (int i = 0; i < W4_AHEAD && group0 + i < groups; i++) prefetch_l2(scales + (group0 + i) * a.scale_stride);
        const __half* at = scales + group0 * a.scale_stride;
        int left = groups - group0;                            // groups from there on: a step may end behind the last
        auto ask = [&]() {
            #pragma unroll
            for (int i = 0; i < C::GROUPS; i++) {
                next[i] = G == W4_UNIT || i < left ? at[i * a.scale_stride] : __half(0.f);     // of no group: nothing, where the one before may have infinities
                if (i + W4_AHEAD < left) prefetch_l2(at + (i + W4_AHEAD) * a.scale_stride);
            }
            at += C::GROUPS * a.scale_stride;
            left -= C::GROUPS;
        };
        if (steps > 0) ask();
        for (unsigned s = 0; s < (unsigned)steps; s++) {
            const unsigned buf = s & 1;
            float2 v[C::GROUPS];
            #pragma unroll
            for (int i = 0; i < C::GROUPS; i++) { v[i].x = __half2float(next[i]) * 16777216.f; v[i].y = v[i].x; }
            if (s + 1 < (unsigned)steps) ask();
            if (!__all_sync(0xffffffffu, mbar_wait(&d_full[tile][buf], (uint32_t)(s >> 1) & 1u, &abort_word, 76))) break;
            tc_fence_after_sync();
            constexpr int COLS = N == 16 ? 16 : 32;
            #pragma unroll
            for (int c = 0; c < C::GROUPS * N / COLS; c++) {
                uint32_t d[COLS];
                if constexpr (COLS == 16) tmem_ld16(tmem + buf * 64u + 16u * c, d); else tmem_ld32(tmem + buf * 64u + 32u * c, d);
                tmem_wait_ld();
                const int i = COLS * c / N, at = (COLS * c % N) / 2;
                #pragma unroll
                for (int j = 0; j < COLS / 2; j++) acc[at + j] = fma2(v[i], make_float2(__uint_as_float(d[2 * j]), __uint_as_float(d[2 * j + 1])), acc[at + j]);
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&d_empty[tile][buf]);
                if (s % C::STEPS == C::STEPS - 1) {            // the products are done with X, and with the operand, which was made of the codes
                    const unsigned unit = s / C::STEPS;
                    mbar_arrive(&empty[unit % C::STAGES]);
                    if (unit % C::X_UNITS == C::X_UNITS - 1) mbar_arrive(&x_empty[unit / C::X_UNITS % C::X_STAGES]);
                }
            }
        }
        __syncthreads();                                       // [1]
        if (r < tile_channels) {
            #pragma unroll
            for (int i = 0; i < N; i++)
                if (i < rows) sum[i * block + tile * tile_channels + r] = i & 1 ? acc[i >> 1].y : acc[i >> 1].x;
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(TC_REGS_MAKE));
        const int tile = warp >> 2 & 1, buf = warp >> 3;
        const uint32_t to = tmem_at + (uint32_t)tile * 256u + buf * 64u + lanes;
        const int row = tile * tile_channels + r;             // of the copied box; rows behind a tile's last are the next one's, or what follows
        const uint32_t my_codes = smem_u32(smem) + row * 64, swizzle = (uint32_t)(row >> 1 & 3);
        const uint8_t* const zeros = a.zeros ? a.zeros + min(n0 + tile * tile_channels + r, a.d_out - 1) : nullptr;
        uint32_t next[C::GROUPS];
        #pragma unroll
        for (int i = 0; i < C::GROUPS; i++) next[i] = 8u;
        const uint8_t* at = zeros + (group0 + buf * C::GROUPS) * a.zero_stride;
        int left = groups - group0 - buf * C::GROUPS;
        auto ask = [&]() {
            if (!zeros) return;
            #pragma unroll
            for (int i = 0; i < C::GROUPS; i++) {
                if (G == W4_UNIT || i < left) next[i] = at[i * a.zero_stride];
                if (i + W4_AHEAD < left) prefetch_l2(at + (i + W4_AHEAD) * a.zero_stride);
            }
            at += 2 * C::GROUPS * a.zero_stride;
            left -= 2 * C::GROUPS;
        };
        if (zeros)
            for (int i = 0; i < W4_AHEAD && group0 + i < groups; i++) prefetch_l2(zeros + (group0 + i) * a.zero_stride);
        if (buf < steps) ask();
        for (unsigned s = buf; s < (unsigned)steps; s += 2) {
            const unsigned in_unit = s % C::STEPS, unit = s / C::STEPS, slot = unit % C::STAGES;
            uint32_t minus[C::GROUPS];
            #pragma unroll
            for (int i = 0; i < C::GROUPS; i++) minus[i] = (next[i] | next[i] << 16) | 0x80008000u;
            if (s + 2 < (unsigned)steps) ask();
            if (!__all_sync(0xffffffffu, mbar_wait(&full[slot], (uint32_t)(unit / C::STAGES) & 1u, &abort_word, 77))) break;
            constexpr int CHUNKS = C::STEP / 32;               // of 16 bytes
            bool going = true;
            #pragma unroll
            for (int c = 0; c < CHUNKS; c++) {
                uint32_t w[4], f[16];
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                             : "r"(my_codes + slot * C::SLOT + (((uint32_t)(in_unit * CHUNKS + c) ^ swizzle) << 4)) : "memory");
                #pragma unroll
                for (int i = 0; i < 4; i++) codes_to_f16(w[i], minus[32 * c / G], f + 4 * i);
                if (c == 0 && s >= 2) {                        // the operand that was here has been multiplied
                    going = __all_sync(0xffffffffu, mbar_wait(&d_full[tile][buf], (uint32_t)((s >> 1) - 1) & 1u, &abort_word, 78));
                    if (!going) break;
                    tc_fence_after_sync();
                }
                tmem_st16(to + 16u * c, f);
            }
            if (!going) break;
            tmem_wait_st();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&a_full[tile][buf]);
        }
    }
    if (warp < TC_COLLECT || warp >= TC_COPY) __syncthreads(); // [1]
    if (abort_word != 0) {                                     // copies and products in flight end first; what the block has is written
        for (int i = 0; i < 64; i++) __nanosleep(100000);
        if (threadIdx.x == 0 && a.status != nullptr && atomicCAS(a.status, 0, (int)KS_WAIT_TIMEOUT) == 0) {
            a.status[1] = blockIdx.x;
            a.status[2] = abort_word;
        }
    }
    __syncthreads();
    if (warp == TC_COPY + 1) { tc_fence_after_sync(); tmem_dealloc(tmem_at, 512); }
    if (parts > 1) {
        cluster_sync();
        store_sums(a, sum, rows, block, parts, part, m0, n0);
        cluster_sync();                                        // the others may still read this block's sums
    } else
        for (int e = 4 * threadIdx.x; e < rows * block; e += 4 * TC_THREADS) store_sum4(a, *reinterpret_cast<const float4*>(sum + e), m0 + e / block, n0 + e % block);
}

// Clusters of p blocks that the device holds at a time: blocks that have an SM each must find them in one part of the GPU. Asked once; a question that failed fails the
// call, as another division would be another order of the sums.
template <auto kernel>
int clusters_at_once(int p, int smem, int dev, int& n)
{
    static std::atomic<int> known[64][W4_MAX_PARTS + 1];       // one more than the number, 0: not asked yet
    if (dev < 64 && (n = known[dev][p].load(std::memory_order_relaxed)) != 0) { n--; return 0; }
    n = device_sms();
    if (p > 1) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(1, 1, p);
        cfg.blockDim = dim3(TC_THREADS);
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = attr.val.clusterDim.y = 1;
        attr.val.clusterDim.z = (unsigned)p;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        EFA_CUDA(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
    }
    if (dev < 64) known[dev][p].store(n + 1, std::memory_order_relaxed);
    return 0;
}

template <int G, int N>
int plan_tc(const W4Args& a, W4Division& to)
{
    using C = TcCfg<G, N>;
    constexpr auto kernel = proj_w4_tc_kernel<G, N>;
    const int units = (a.d_in + W4_UNIT - 1) / W4_UNIT;
    static std::atomic<bool> set[64];
    int dev = 0;
    EFA_CUDA(cudaGetDevice(&dev));
    if (dev >= 64 || !set[dev]) {
        EFA_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
        if (dev < 64) set[dev] = true;
    }
    int at_once[W4_MAX_PARTS + 1] = {};
    for (int p = 1; p <= std::min(W4_MAX_PARTS, units); p++)
        if (int rc = clusters_at_once<kernel>(p, C::SMEM, dev, at_once[p])) return rc;
    to = w4_division(a.d_out, (a.rows + 63) / 64, units, at_once);
    return 0;
}

template <int G, int N>
int launch_tc(const W4Args& a, const W4Division& to, cudaStream_t stream)
{
    using C = TcCfg<G, N>;
    constexpr auto kernel = proj_w4_tc_kernel<G, N>;
    const int channels = to.channels;
    CUtensorMap codes, x;
    const unsigned long long code_dims[2] = {(unsigned long long)a.d_in / 2, (unsigned long long)a.d_out}, code_stride[1] = {(unsigned long long)a.code_stride};
    const unsigned code_box[2] = {64, 2 * (unsigned)channels};
    if (make_tmap_u8(&codes, a.codes, 2, code_dims, code_stride, code_box)) return 1;
    // X as blocks of 64 k, several to a copy; or a copy each, where the last block of a row is half another row.
    const bool x_blocks = a.d_in % 64 == 0;
    if (x_blocks) {
        const unsigned long long dims[3] = {64, (unsigned long long)a.rows, (unsigned long long)a.d_in / 64}, strides[2] = {(unsigned long long)a.x_stride * 2, 128};
        const unsigned box[3] = {64, N, C::X_BLOCKS};
        if (make_tmap_f16(&x, a.X, 3, dims, strides, box)) return 1;
    } else {
        const unsigned long long dims[2] = {(unsigned long long)a.d_in, (unsigned long long)a.rows}, strides[1] = {(unsigned long long)a.x_stride * 2};
        const unsigned box[2] = {64, N};
        if (make_tmap_f16(&x, a.X, 2, dims, strides, box)) return 1;
    }
    const dim3 grid((a.d_out + 2 * channels - 1) / (2 * channels), (a.rows + 63) / 64, to.parts);
    EFA_CUDA(launch_value(kernel, grid, TC_THREADS, C::SMEM, stream, a, channels, x_blocks, codes, x));
    return 0;
}

template <int G>
int plan_rows(const W4Args& a, W4Division& to) { return a.rows <= 16 ? plan_tc<G, 16>(a, to) : a.rows <= 32 ? plan_tc<G, 32>(a, to) : plan_tc<G, 64>(a, to); }

template <int G>
int launch_rows(const W4Args& a, const W4Division& to, cudaStream_t stream)
{
    return a.rows <= 16 ? launch_tc<G, 16>(a, to, stream) : a.rows <= 32 ? launch_tc<G, 32>(a, to, stream) : launch_tc<G, 64>(a, to, stream);
}

}  // namespace

int w4_tc_plan(const W4Args& a, int group, W4Division& to)
{
    return group == 128 ? plan_rows<128>(a, to) : group == 64 ? plan_rows<64>(a, to) : plan_rows<32>(a, to);
}

int w4_tc_launch(const W4Args& a, int group, const W4Division& to, cudaStream_t stream)
{
    return group == 128 ? launch_rows<128>(a, to, stream) : group == 64 ? launch_rows<64>(a, to, stream) : launch_rows<32>(a, to, stream);
}

}  // namespace efa
