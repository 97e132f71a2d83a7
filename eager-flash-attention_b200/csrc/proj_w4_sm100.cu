// Projections of few rows with weights of 4 bits and group scales. out[m][n] = sum over groups g of s[g][n] * sum over the group's k of
// x[m][k] * (code[n][k] - zero[g][n]).
//
// mma.sync m16n8k16 with the weights as the side of 16 (output channels) and the rows of X as the side of 8: one token uses an eighth of it. The order of k
// within a group is free as long as both sides agree on it, so codes go from memory to a fragment as they lie: a lane's word is eight neighbouring k of one
// channel, `(word >> 4 i) & 0x000f000f` is the pair (k + i, k + i + 4) of two products' fragments, and x is paired alike. A code c becomes the fp16 number
// 1024 + c (or 1024 + 16 c, times 1/16) by one logical operation, and c - zero exactly by one more: nine instructions to eight weights. (Integers that are put into a float's mantissa below a power of
// two: the method of Kim et al., "Who Says Elephants Can't Run", 2022, for weights of 4 and 8 bits.) All four lanes that share a channel are in one group: 16, 8 or 4 bytes to a lane for
// groups of 128, 64 or 32.
//
// Reading the weights is the floor (a group of 128: 0.516 bytes each). What bounds it: up to some 10 us the way from the launch to the first codes, the sums and the end (one row,
// 4096 x 4096: 4.1 us of which the bytes are 1.3; 1056 x 4163: 3.0). From six rows on a warp waits for each of its units: there is no room for a second one in flight. Beyond, instructions: 624 to 656 to a warp's 32 channels x 256 k, of which 320 make fragments and multiply, issued
// at 0.6 to a cycle and scheduler (one row, 8192 x 32768: 33 us, 4.1 TB/s of the 6.5; 2048 x 65536: 21 us; without the scales' part, a tenth of the instructions, a tenth less).
#include "proj_w4.cuh"
#include "serving.h"

#include <algorithm>
#include <atomic>

namespace efa {

namespace {

// Sixteen warps to an SM, in one block or two: four to a scheduler hide one another's waits. Of up to three stages as many as have room: two up to five rows (four with groups of 32), one beyond.
// The kernels of 9 to 16 rows with groups of 64 and 128 spill 24 and 44 bytes a thread at 128 registers.
constexpr int W4_STAGES = 3;
constexpr int W4_MT = 2;                // tiles of 16 channels to a warp

// (a & mask) | with
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t mask, uint32_t with)
{
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(a), "r"(mask), "r"(with));
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

// Eight codes to four pairs (i, i + 4) of numbers code - zero, exactly. low: 1024 + zero twice; high: -(64 + zero) twice.
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t low, uint32_t high, uint32_t (&f)[4])
{
    constexpr uint32_t MAGIC = 0x64006400u, SIXTEENTH = 0x2c002c00u;            // 1024, 1/16
    const uint32_t v = w >> 8;
    f[0] = sub2(and_or(w, 0x000f000fu, MAGIC), low);
    f[1] = fma2(and_or(w, 0x00f000f0u, MAGIC), SIXTEENTH, high);
    f[2] = sub2(and_or(v, 0x000f000fu, MAGIC), low);
    f[3] = fma2(and_or(v, 0x00f000f0u, MAGIC), SIXTEENTH, high);
}

// c += A B, or (first) c = A B.
__device__ __forceinline__ void mma_w4(float (&c)[4], bool first, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    if (first)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int N> __device__ __forceinline__ void load_shared(uint32_t addr, uint32_t (&w)[N])
{
    if constexpr (N == 4) asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr) : "memory");
    else if constexpr (N == 2) asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr) : "memory");
    else asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(addr) : "memory");
}

// What a warp keeps in shared memory: stages of codes (128 bytes of each of 16 MT channels), of X (512 bytes of each row), and a unit's scales.
constexpr int W4_K = 256;               // k of a unit
template <int WARPS> struct W4Head { uint64_t bars[WARPS][W4_STAGES], full[2], empty[2]; int abort_word; };     // in the first 1024 bytes
template <int G, int MT, int NT, int WARPS>
struct W4Cfg {
    static constexpr int SMEM = WARPS == 16 ? 227 * 1024 : 113 * 1024;         // of the SM's 228 KB, less one to each block
    static_assert(sizeof(W4Head<WARPS>) <= 1024, "");
    static constexpr int CHANNELS = 16 * MT, SUBS = W4_K / G;
    static constexpr int CODE_BYTES = CHANNELS * 128, TABLE = SUBS * CHANNELS * (int)sizeof(float2);
    __host__ __device__ static constexpr int copies(int rows, int stages) { return WARPS * (stages * (CODE_BYTES + rows * 512) + TABLE); }
    // Sums of a block that goes on to another tile are not where its copies are.
    static int smem(int rows, int stages, bool again)
    {
        const int sums = WARPS * rows * CHANNELS * (int)sizeof(float);
        return 1024 + (again ? copies(rows, stages) + 2 * sums : std::max(copies(rows, stages), sums));
    }
    static bool ahead(int rows) { return smem(rows, 2, true) <= SMEM; }
    static_assert(CODE_BYTES % 1024 == 0, "");
};

// Which channel of eight a lane's fragments hold, so that the lanes that read codes together find different banks: 16-byte chunk c of a row's eight lies at
// c ^ (row % 8) (the 128-byte swizzle of the copy). Of X, chunk c of a row's sixteen to 128 k at x_place.
template <int G> __device__ __forceinline__ int channel_of(int g) { return G == 128 ? g >> 1 | (g & 1) << 2 : G == 64 ? (g & 3) * 2 + (g >> 2) : g; }
template <int G> __device__ __forceinline__ int x_place(int row, int c)
{
    return G == 128 ? c ^ (c >> 3 & 1) ^ (row & 1) << 1 : G == 64 ? c ^ (row & 1) : c ^ (row & 1) << 2;
}

// A block: 16 MT channels, 8 NT rows, all k, its warps (and the blocks of its cluster, along z) taking the units of 256 k in turn, added at the end in shared
// memory in the order of the warps and blocks. A warp copies its own units, ahead where there is more than one stage, codes by TMA, X by its lanes: nobody waits for anybody before the sums.
template <int G, int MT, int NT, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, 16 / WARPS)
proj_w4_kernel(const W4Args a, int stages, const __grid_constant__ CUtensorMap codes_map)
{
    using C = W4Cfg<G, MT, NT, WARPS>;
    constexpr int SUBS = C::SUBS, WORDS = G / 32;              // groups of a unit, words of codes of a lane and group
    constexpr int CHANNELS = C::CHANNELS, PER_LANE = (CHANNELS + 31) / 32;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint64_t (&bars)[WARPS][W4_STAGES] = reinterpret_cast<W4Head<WARPS>*>(smem_raw)->bars;
    uint64_t (&full)[2] = reinterpret_cast<W4Head<WARPS>*>(smem_raw)->full, (&empty)[2] = reinterpret_cast<W4Head<WARPS>*>(smem_raw)->empty;
    int& abort_word = reinterpret_cast<W4Head<WARPS>*>(smem_raw)->abort_word;
    constexpr int warps = WARPS;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int first = blockIdx.x * CHANNELS, next_tile = gridDim.x * CHANNELS, m0 = blockIdx.y * 8 * NT, rows = min(a.rows - m0, 8 * NT);
    const int parts = gridDim.z, part = parts > 1 ? (int)cluster_rank() : 0;
    const int units = (a.d_in + W4_K - 1) / W4_K;
    // Warps take the units of a block in turn, so that what they read at a time is neighbours in the rows of codes.
    const int step = warps, u0 = (int)((long long)units * part / parts) + warp, u1 = (int)((long long)units * (part + 1) / parts);

    uint8_t* const smem = smem_raw + 1024;
    // Codes of all warps first, then X, then the tables.
    uint8_t* const slots = smem + warp * (stages * C::CODE_BYTES);
    const uint32_t x_slots = smem_u32(smem) + warps * (stages * C::CODE_BYTES) + warp * (stages * rows * 512);
    uint2* const table = reinterpret_cast<uint2*>(smem + warps * stages * (C::CODE_BYTES + rows * 512) + warp * C::TABLE);
    uint64_t* const bar = bars[warp];
    if (lane == 0) {
        for (int i = 0; i < stages; i++) mbar_init(&bar[i], 33);               // the copy of codes, and what each lane copies of X
        mbar_fence_init();
        tma_prefetch_desc(&codes_map);
    }
    const int adders = min(warps, units);                      // warps that have units, where a block has them all
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; i++) { mbar_init(&full[i], adders); mbar_init(&empty[i], 1); }
        mbar_fence_init();
        abort_word = 0;
    }
    __syncthreads();
    pdl_wait();
    pdl_trigger();

    // The units of this warp: of a tile of channels, then of the block's next. Copies run `stages` of them ahead, over the ends of tiles.
    struct Unit { int u, n; } copied{u0, u0 < u1 ? first : a.d_out}, asked = copied;
    auto after = [&](Unit& at) {
        at.u += step;
        if (at.u >= u1) { at.u = u0; at.n += next_tile; return true; }
        return false;
    };
    auto fetch = [&](int slot) {
        if (copied.n >= a.d_out) return;
        if (lane == 0) {
            mbar_expect_tx(&bar[slot], C::CODE_BYTES);
            tma_load_2d(slots + slot * C::CODE_BYTES, &codes_map, &bar[slot], copied.u * (W4_K / 2), copied.n);
        }
        if (copied.u * W4_K + 8 * lane < a.d_in)
            for (int r = 0; r < rows; r++)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                             :: "r"(x_slots + (slot * rows + r) * 512 + ((lane & 16) | x_place<G>(r, lane & 15)) * 16), "l"(a.X + (m0 + r) * a.x_stride + copied.u * W4_K + 8 * lane) : "memory");
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" :: "r"(smem_u32(&bar[slot])) : "memory");
        after(copied);
    };
    for (int i = 0; i < stages; i++) fetch(i);
    // Scales and zeros of a unit's channels: to registers a unit ahead, and from there as scale and 1024 + zero (twice, fp16) to the table.
    const __half* s_at[PER_LANE];
    const uint8_t* z_at[PER_LANE];
    auto begin = [&]() {
        #pragma unroll
        for (int i = 0; i < PER_LANE; i++) {
            const int n = min(asked.n + lane + 32 * i, a.d_out - 1);
            s_at[i] = a.scales + (long long)u0 * SUBS * a.scale_stride + n;
            z_at[i] = a.zeros + (long long)u0 * SUBS * a.zero_stride + n;
        }
    };
    const int groups = a.d_in / G;
    __half s_next[SUBS][PER_LANE];
    uint8_t z_next[SUBS][PER_LANE];
    auto ask = [&]() {
        if (asked.n >= a.d_out) return;
        #pragma unroll
        for (int s = 0; s < SUBS; s++)
            if (asked.u * SUBS + s < groups) {
                #pragma unroll
                for (int i = 0; i < PER_LANE; i++) {
                    s_next[s][i] = s_at[i][s * a.scale_stride];
                    if (a.zeros) z_next[s][i] = z_at[i][s * a.zero_stride];
                }
            }
        #pragma unroll
        for (int i = 0; i < PER_LANE; i++) {
            s_at[i] += (long long)step * SUBS * a.scale_stride;
            z_at[i] += (long long)step * SUBS * a.zero_stride;
        }
        if (after(asked)) begin();
    };
    auto tabulate = [&]() {
        #pragma unroll
        for (int s = 0; s < SUBS; s++)
            #pragma unroll
            for (int i = 0; i < PER_LANE; i++)
                if (CHANNELS >= 32 || lane < CHANNELS)
                    table[s * CHANNELS + lane + 32 * i] = make_uint2(__float_as_uint(__half2float(s_next[s][i])), 0x64006400u + 0x00010001u * (a.zeros ? (uint32_t)z_next[s][i] : 8u));
    };
    begin();
    ask();
    const int row = channel_of<G>(g);
    const uint32_t code_base = smem_u32(slots) + row * 128;
    // Columns behind the last row are the last row's: nobody looks at their sums.
    int x_row[NT];
    uint32_t x[NT];
    #pragma unroll
    for (int n = 0; n < NT; n++) {
        x_row[n] = min(8 * n + g, rows - 1);
        x[n] = x_slots + x_row[n] * 512;
    }
    const int tile_sums = rows * CHANNELS;
    int slot = 0;
    uint32_t phase = 0;
    float acc[MT][NT][4];
    auto tile = [&]() {
        #pragma unroll
        for (int m = 0; m < MT; m++)
            #pragma unroll
            for (int n = 0; n < NT; n++)
                #pragma unroll
                for (int i = 0; i < 4; i++) acc[m][n][i] = 0.f;
        for (int u = u0; u < u1; u += step) {
            tabulate();
            ask();
            if (!__all_sync(0xffffffffu, mbar_wait(&bar[slot], phase, &abort_word, 70))) break;
            __syncwarp();                                      // the table is other lanes' writing: a vote orders no memory
            const uint32_t codes = code_base + slot * C::CODE_BYTES;
            #pragma unroll
            for (int s = 0; s < SUBS; s++) {
                if (u * W4_K + s * G >= a.d_in) break;
                uint32_t b[WORDS][NT][4];
                #pragma unroll
                for (int i = 0; i < WORDS; i++)
                    #pragma unroll
                    for (int n = 0; n < NT; n++) {
                        uint32_t q[4];
                        const int c = s * (G / 8) + t * WORDS + i;     // 16-byte chunk of the row's 512
                        load_shared(x[n] + slot * (rows * 512) + ((c & 16) | x_place<G>(x_row[n], c & 15)) * 16, q);
                        b[i][n][0] = __byte_perm(q[0], q[2], 0x5410); b[i][n][1] = __byte_perm(q[0], q[2], 0x7632);
                        b[i][n][2] = __byte_perm(q[1], q[3], 0x5410); b[i][n][3] = __byte_perm(q[1], q[3], 0x7632);
                    }
                const int at = s * (G / 2) + t * (G / 8);          // byte of the row's 128
                const uint32_t code_at = codes + ((at >> 4) ^ row) * 16 + (at & 15);
                #pragma unroll
                for (int m = 0; m < MT; m++) {
                    uint32_t w[2][WORDS], high[2];
                    uint2 scale[2];
                    #pragma unroll
                    for (int h = 0; h < 2; h++) {
                        load_shared(code_at + (16 * m + 8 * h) * 128, w[h]);
                        scale[h] = table[s * CHANNELS + 16 * m + 8 * h + row];
                        high[h] = sub2(0x63806380u, scale[h].y);       // 960 - (1024 + zero)
                    }
                    float sum[NT][4];
                    #pragma unroll
                    for (int i = 0; i < WORDS; i++) {
                        uint32_t p[4], q[4];
                        codes_to_f16(w[0][i], scale[0].y, high[0], p);
                        codes_to_f16(w[1][i], scale[1].y, high[1], q);
                        #pragma unroll
                        for (int n = 0; n < NT; n++) {
                            mma_w4(sum[n], i == 0, p[0], q[0], p[1], q[1], b[i][n][0], b[i][n][1]);
                            mma_w4(sum[n], false, p[2], q[2], p[3], q[3], b[i][n][2], b[i][n][3]);
                        }
                    }
                    #pragma unroll
                    for (int n = 0; n < NT; n++)
                        #pragma unroll
                        for (int j = 0; j < 4; j++) acc[m][n][j] = fmaf(__uint_as_float(scale[j >> 1].x), sum[n][j], acc[m][n][j]);
                }
            }
            __syncwarp();
            fetch(slot);
            if (++slot == stages) { slot = 0; phase ^= 1; }
        }
    };
    // Sums of the warps [warp][8 NT][16 MT].
    auto put = [&](float* to) {
        #pragma unroll
        for (int m = 0; m < MT; m++)
            #pragma unroll
            for (int n = 0; n < NT; n++)
                #pragma unroll
                for (int i = 0; i < 4; i++) if (8 * n + 2 * t + (i & 1) < rows) to[warp * tile_sums + (8 * n + 2 * t + (i & 1)) * CHANNELS + 16 * m + 8 * (i >> 1) + row] = acc[m][n][i];
    };
    auto added = [&](const float* from) {
        float v = from[0];
        #pragma unroll
        for (int w = 1; w < warps; w++)
            if (w < adders) v += from[w * tile_sums];
        return v;
    };
    auto settle = [&]() {                                      // copies in flight land first, then what the block has is written
        for (int i = 0; i < 64; i++) __nanosleep(100000);
        if (threadIdx.x == 0 && a.status != nullptr && atomicCAS(a.status, 0, (int)KS_WAIT_TIMEOUT) == 0) {
            a.status[1] = blockIdx.x;
            a.status[2] = abort_word;
        }
    };
    if (NT == 1 && next_tile < a.d_out) {
        // Several tiles to a block: nobody waits at the end of one. The warps add up in turn, from two buffers behind the copies.
        float* const sums = reinterpret_cast<float*>(smem + C::copies(rows, stages));
        for (int n0 = first, i = 0; n0 < a.d_out && u0 < u1; n0 += next_tile, i++) {
            float* const sum = sums + (i & 1) * (warps * tile_sums);
            tile();
            if (!__all_sync(0xffffffffu, mbar_wait(&empty[i & 1], (uint32_t)(i >> 1 & 1) ^ 1u, &abort_word, 69))) break;
            put(sum);
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[i & 1]);
            if (i % adders == warp) {
                if (!__all_sync(0xffffffffu, mbar_wait(&full[i & 1], (uint32_t)(i >> 1 & 1), &abort_word, 69))) break;
                for (int e = lane; e < rows * CHANNELS; e += 32) store_sum(a, added(sum + e), m0 + e / CHANNELS, n0 + e % CHANNELS);
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty[i & 1]);
            }
        }
        __syncthreads();
        if (abort_word != 0) settle();
        return;
    }
    // One tile: the sums are where the copies were.
    float* const sum = reinterpret_cast<float*>(smem);
    tile();
    __syncthreads();
    if (abort_word != 0) { settle(); __syncthreads(); }
    put(sum);
    __syncthreads();
    for (int e = threadIdx.x; e < rows * CHANNELS; e += blockDim.x) {
        const float v = added(sum + e);
        if (parts > 1) sum[e] = v;
        else store_sum(a, v, m0 + e / CHANNELS, first + e % CHANNELS);
    }
    if (parts > 1) {
        cluster_sync();
        store_sums(a, sum, rows, CHANNELS, parts, part, m0, first);
        cluster_sync();                                        // the others may still read this block's sums
    }
}

template <int G, int NT, int WARPS>
int launch_w4(const W4Args& a, int sms, cudaStream_t stream)
{
    using C = W4Cfg<G, W4_MT, NT, WARPS>;
    constexpr auto kernel = proj_w4_kernel<G, W4_MT, NT, WARPS>;
    const int tiles = (a.d_out + C::CHANNELS - 1) / C::CHANNELS, row_tiles = (a.rows + 8 * NT - 1) / (8 * NT), units = (a.d_in + W4_K - 1) / W4_K;
    const int parts = w4_parts((long long)tiles * row_tiles, units, WARPS, sms);
    CUtensorMap codes;
    const unsigned long long dims[2] = {(unsigned long long)a.d_in / 2, (unsigned long long)a.d_out}, strides[1] = {(unsigned long long)a.code_stride};
    const unsigned box[2] = {W4_K / 2, C::CHANNELS};
    if (make_tmap_u8(&codes, a.codes, 2, dims, strides, box)) return 1;
    const int rows = std::min(a.rows, 8 * NT);
    // More tiles than blocks at a time: a block goes on to another tile, whose copies are under way before the sums of this one, if there is room for a stage of them beside the one in
    // use. us, blocks of one tile / of several: one row, 2048 x 65536 27.0 / 21.0, 4096 x 28672 25.1 / 19.9; with one stage 8 rows, 8192 x 32768 39.4 / 42.
    const bool again = NT == 1 && tiles > 16 / WARPS * sms && C::ahead(rows);
    const int blocks = again ? 16 / WARPS * sms : tiles;
    int stages = W4_STAGES;
    while (stages > 1 && C::smem(rows, stages, again) > C::SMEM) stages--;
    static std::atomic<bool> set[64];
    int dev = 0;
    EFA_CUDA(cudaGetDevice(&dev));
    if (dev >= 64 || !set[dev]) {
        EFA_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, std::max(C::SMEM, C::smem(8 * NT, 1, false))));
        if (dev < 64) set[dev] = true;
    }
    EFA_CUDA(launch_value(kernel, dim3(blocks, row_tiles, parts), WARPS * 32, C::smem(rows, stages, again), stream, a, stages, codes));
    return 0;
}

template <int G>
int launch_group(const W4Args& a, int sms, cudaStream_t stream)
{
    if (a.rows > 8) return launch_w4<G, 2, 8>(a, sms, stream);
    // One block to an SM has all sixteen warps; and of tiles that go round, those of much k: seven rounds of 148 are less than four of 296. us, two blocks of eight / one of sixteen: 8 rows,
    // 4096 x 4096 5.4 / 4.7, 14336 x 4096 13.8 / 11.7; one row, 8192 x 32768 37.6 / 33.4. Against it: 4096 x 6144 (192 tiles) 7.3 / 10.2, 4096 x 28672 (16 units: one to a
    // warp) 20.0 / 21.6, 8192 x 1024 (a cluster to a tile) 4.2 / 4.8.
    const int tiles = (a.d_out + 16 * W4_MT - 1) / (16 * W4_MT), units = (a.d_in + W4_K - 1) / W4_K;
    const bool sixteen = tiles <= sms ? units >= 16 && 2 * tiles > sms : units >= 32 && tiles > 2 * sms && W4Cfg<G, W4_MT, 1, 16>::ahead(a.rows);
    return sixteen ? launch_w4<G, 1, 16>(a, sms, stream) : launch_w4<G, 1, 8>(a, sms, stream);
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
    if (!aligned(w.scales, 2)) return "w4: scales must be aligned to their elements";
    if (w.code_stride != 0 && (w.code_stride < w.d_in / 2 || w.code_stride % 16)) return "w4: code_stride must be 0 or a multiple of 16 that holds a row";
    if (w.scale_stride != 0 && w.scale_stride < w.d_out) return "w4: scale_stride must be 0 or at least d_out";
    if (w.zero_stride != 0 && w.zero_stride < w.d_out) return "w4: zero_stride must be 0 or at least d_out";
    return nullptr;
}

int project_w4(const void* X, long long x_stride, const efa_w4& w, void* out, int out_dtype, long long out_stride, int rows, cudaStream_t stream)
{
    if (const char* why = w4_check(w)) { set_error("project_w4: %s", why); return 2; }
    if (rows < 0 || rows > 1 << 19) { set_error("project_w4: rows must be from 0 to 2^19 (got %d)", rows); return 2; }
    if (out_dtype != EFA_F16 && out_dtype != EFA_F32) { set_error("project_w4: out must be EFA_F16 or EFA_F32"); return 2; }
    if (x_stride != 0 && (x_stride < w.d_in || x_stride % 8)) { set_error("project_w4: x_stride must be 0 or a multiple of 8 that holds d_in"); return 2; }
    if (out_stride != 0 && out_stride < w.d_out) { set_error("project_w4: out_stride must be 0 or at least d_out"); return 2; }
    if (rows == 0) return 0;
    if (!X || !out) { set_error("project_w4: X or out is null"); return 2; }
    if (!aligned16(X) || !aligned(out, out_dtype == EFA_F16 ? 2 : 4)) { set_error("project_w4: X must be 16-byte aligned, out to its elements"); return 2; }
    const W4Args a{w.codes, static_cast<const __half*>(w.scales), w.zeros, static_cast<const __half*>(X), out, rows, w.d_in, w.d_out,
                   w.code_stride ? w.code_stride : w.d_in / 2, w.scale_stride ? w.scale_stride : w.d_out, w.zero_stride ? w.zero_stride : w.d_out,
                   x_stride ? x_stride : w.d_in, out_stride ? out_stride : w.d_out, out_dtype == EFA_F32, aligned16(out) && (out_stride ? out_stride : w.d_out) % 4 == 0, kernel_status_word()};
    const int elem = a.out_f32 ? 4 : 2;
    if (rows_clash(RowSpan{out, rows, (long long)a.d_out * elem, a.out_stride * elem, elem}, RowSpan{X, rows, 2ll * a.d_in, 2 * a.x_stride, 2}, false)) {
        set_error("project_w4: out overlaps X");
        return 2;
    }
    const void* const mem[] = {X, w.codes, w.scales, w.zeros, out};
    if (int rc = check_memory("project_w4", mem, 5)) return rc;
    // Up to eight rows the products of mma.sync are not the time. Beyond, tiles of 16 rows that read the weights again, or tcgen05 with up to 64 rows to a tile, whose start and
    // end cost more, and every group of a row its sums: by what either takes (w4_plan.h).
    const int sms = device_sms();
    if (rows > 8) {
        const double mma = w4_mma_time(w.d_in, w.d_out, rows, w.group, sms);
        if (w4_tc_least(w.d_in, w.d_out, rows, w.group) < mma) {
            W4Division to;
            if (int rc = w4_tc_plan(a, w.group, to)) return rc;
            if (w4_tc_time(to, w.d_in, w.d_out, rows, w.group) < mma) return w4_tc_launch(a, w.group, to, stream);
        }
    }
    return w.group == 128 ? launch_group<128>(a, sms, stream) : w.group == 64 ? launch_group<64>(a, sms, stream) : launch_group<32>(a, sms, stream);
}

}  // namespace efa
