// Projections of few rows with weights of 4 bits and group scales: reading the weights is the time. out[m][n] = sum over groups g of s[g][n] * sum over
// the group's k of x[m][k] * (code[n][k] - zero[g][n]).
//
// mma.sync m16n8k16 with the weights as the side of 16 (output channels) and the rows of X as the side of 8: one token uses an eighth of it, which costs
// nothing while memory is the time. The order of k within a group is free as long as both sides agree on it, so codes go from memory to a fragment as they
// lie: a lane's four bytes are eight neighbouring k of one channel, `(word >> 4 i) & 0x000f000f` is the pair (k + i, k + i + 4) of two products' fragments, and x is
// paired alike. A code c becomes the fp16 number 1024 + c (or 1024 + 16 c, times 1/16) by one logical operation, and c - zero exactly by one more. All
// four lanes that share a channel must be in one group: 16, 8 or 4 bytes to a lane and load for groups of 128, 64 or 32.
#include "proj_w4.cuh"
#include "serving.h"

#include <algorithm>

namespace efa {

namespace {

// Eight warps, and two blocks to an SM: four warps to a scheduler hide one another's waits. Of up to three stages as many as leave room for the second block.
constexpr int W4_WARPS = 8, W4_BLOCKS = 2, W4_STAGES = 3, W4_SMEM = 113 * 1024;
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

// What a warp keeps in shared memory: stages of codes (128 bytes of each of 16 MT channels), of X (512 bytes of each row), and two units of scales.
constexpr int W4_K = 256;               // k of a unit
template <int G, int MT, int NT>
struct W4Cfg {
    static constexpr int CHANNELS = 16 * MT, SUBS = W4_K / G;
    static constexpr int CODE_BYTES = CHANNELS * 128, TABLE = SUBS * CHANNELS * (int)sizeof(float2), TILE = CHANNELS * 8 * NT;
    static int smem(int rows, int stages) { return 1024 + W4_WARPS * std::max(stages * (CODE_BYTES + rows * 512) + 2 * TABLE, TILE * (int)sizeof(float)); }
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
// memory in the order of the warps and blocks. A warp has its own units copied ahead, codes by TMA, X by its lanes: nobody waits for anybody before the sums.
template <int G, int MT, int NT>
__global__ void __launch_bounds__(32 * W4_WARPS, W4_BLOCKS)
proj_w4_kernel(const W4Args a, int stages, const __grid_constant__ CUtensorMap codes_map)
{
    using C = W4Cfg<G, MT, NT>;
    constexpr int SUBS = C::SUBS, WORDS = G / 32;              // groups of a unit, words of codes of a lane and group
    constexpr int CHANNELS = C::CHANNELS, PER_LANE = (CHANNELS + 31) / 32;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bars[W4_WARPS][W4_STAGES];
    __shared__ int abort_word;
    constexpr int warps = W4_WARPS;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * CHANNELS, m0 = blockIdx.y * 8 * NT, rows = min(a.rows - m0, 8 * NT);
    const int parts = gridDim.z, part = parts > 1 ? (int)cluster_rank() : 0;
    const int units = (a.d_in + W4_K - 1) / W4_K;
    // Warps take the units of a block in turn, so that what they read at a time is neighbours in the rows of codes.
    const int step = warps, u0 = (int)((long long)units * part / parts) + warp, u1 = (int)((long long)units * (part + 1) / parts);

    uint8_t* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    // Codes of all warps first, then X, then the tables.
    uint8_t* const slots = smem + warp * (stages * C::CODE_BYTES);
    const uint32_t x_slots = smem_u32(smem) + warps * (stages * C::CODE_BYTES) + warp * (stages * rows * 512);
    uint2* const table = reinterpret_cast<uint2*>(smem + warps * stages * (C::CODE_BYTES + rows * 512) + warp * 2 * C::TABLE);
    uint64_t* const bar = bars[warp];
    if (lane == 0) {
        for (int i = 0; i < stages; i++) mbar_init(&bar[i], 33);               // the copy of codes, and what each lane copies of X
        mbar_fence_init();
        tma_prefetch_desc(&codes_map);
    }
    if (threadIdx.x == 0) abort_word = 0;
    __syncthreads();
    pdl_wait();
    pdl_trigger();

    auto fetch = [&](int u, int slot) {
        if (lane == 0) {
            mbar_expect_tx(&bar[slot], C::CODE_BYTES);
            tma_load_2d(slots + slot * C::CODE_BYTES, &codes_map, &bar[slot], u * (W4_K / 2), n0);
        }
        if (u * W4_K + 8 * lane < a.d_in)
            for (int r = 0; r < rows; r++)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                             :: "r"(x_slots + (slot * rows + r) * 512 + ((lane & 16) | x_place<G>(r, lane & 15)) * 16), "l"(a.X + (m0 + r) * a.x_stride + u * W4_K + 8 * lane) : "memory");
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" :: "r"(smem_u32(&bar[slot])) : "memory");
    };
    for (int i = 0; i < stages && u0 + i * step < u1; i++) fetch(u0 + i * step, i);
    // Scales and zeros of a unit's channels: to registers a unit ahead, and from there as scale and 1024 + zero (twice, fp16) to the table.
    const __half* s_at[PER_LANE];
    const uint8_t* z_at[PER_LANE];
    #pragma unroll
    for (int i = 0; i < PER_LANE; i++) {
        const int n = min(n0 + lane + 32 * i, a.d_out - 1);
        s_at[i] = a.scales + (long long)u0 * SUBS * a.scale_stride + n;
        z_at[i] = a.zeros + (long long)u0 * SUBS * a.zero_stride + n;
    }
    const int groups = a.d_in / G;
    __half s_next[SUBS][PER_LANE];
    uint8_t z_next[SUBS][PER_LANE];
    auto ask = [&](int u) {
        #pragma unroll
        for (int s = 0; s < SUBS; s++)
            if (u * SUBS + s < groups) {
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
    };
    auto tabulate = [&](uint2* to) {
        #pragma unroll
        for (int s = 0; s < SUBS; s++)
            #pragma unroll
            for (int i = 0; i < PER_LANE; i++)
                if (CHANNELS >= 32 || lane < CHANNELS)
                    to[s * CHANNELS + lane + 32 * i] = make_uint2(__float_as_uint(__half2float(s_next[s][i])), 0x64006400u + 0x00010001u * (a.zeros ? (uint32_t)z_next[s][i] : 8u));
    };
    if (u0 < u1) ask(u0);
    const int row = channel_of<G>(g);
    const uint32_t code_base = smem_u32(slots) + row * 128, x_base = x_slots + g * 512;
    float acc[MT][NT][4] = {};
    int slot = 0;
    uint32_t phase = 0;
    for (int u = u0, odd = 0; u < u1; u += step, odd ^= 1) {
        uint2* const scales = table + odd * (SUBS * CHANNELS);
        tabulate(scales);
        if (u + step < u1) ask(u + step);
        if (!mbar_wait(&bar[slot], phase, &abort_word, 70)) break;
        __syncwarp();
        const uint32_t codes = code_base + slot * C::CODE_BYTES, x = x_base + slot * (rows * 512);
        #pragma unroll
        for (int s = 0; s < SUBS; s++) {
            if (u * W4_K + s * G >= a.d_in) break;
            uint32_t w[MT][2][WORDS];
            const int at = s * (G / 2) + t * (G / 8);          // byte of the row's 128
            const uint32_t code_at = ((at >> 4) ^ row) * 16 + (at & 15);
            #pragma unroll
            for (int m = 0; m < MT; m++)
                #pragma unroll
                for (int h = 0; h < 2; h++) load_shared(codes + code_at + (16 * m + 8 * h) * 128, w[m][h]);
            uint2 scale[MT][2];
            uint32_t high[MT][2];
            #pragma unroll
            for (int m = 0; m < MT; m++)
                #pragma unroll
                for (int h = 0; h < 2; h++) {
                    scale[m][h] = scales[s * CHANNELS + 16 * m + 8 * h + row];
                    high[m][h] = sub2(0x63806380u, scale[m][h].y);              // 960 - (1024 + zero)
                }
            float sum[MT][NT][4];
            #pragma unroll
            for (int i = 0; i < WORDS; i++) {
                uint32_t b[NT][4];
                #pragma unroll
                for (int n = 0; n < NT; n++) {
                    uint32_t q[4] = {0u, 0u, 0u, 0u};
                    const int c = s * (G / 8) + t * WORDS + i;     // 16-byte chunk of the row's 512
                    if (8 * n + g < rows) load_shared(x + n * 4096 + ((c & 16) | x_place<G>(g, c & 15)) * 16, q);
                    b[n][0] = __byte_perm(q[0], q[2], 0x5410); b[n][1] = __byte_perm(q[0], q[2], 0x7632);
                    b[n][2] = __byte_perm(q[1], q[3], 0x5410); b[n][3] = __byte_perm(q[1], q[3], 0x7632);
                }
                #pragma unroll
                for (int m = 0; m < MT; m++) {
                    uint32_t p[4], q[4];
                    codes_to_f16(w[m][0][i], scale[m][0].y, high[m][0], p);
                    codes_to_f16(w[m][1][i], scale[m][1].y, high[m][1], q);
                    #pragma unroll
                    for (int n = 0; n < NT; n++) {
                        mma_w4(sum[m][n], i == 0, p[0], q[0], p[1], q[1], b[n][0], b[n][1]);
                        mma_w4(sum[m][n], false, p[2], q[2], p[3], q[3], b[n][2], b[n][3]);
                    }
                }
            }
            #pragma unroll
            for (int m = 0; m < MT; m++)
                #pragma unroll
                for (int n = 0; n < NT; n++)
                    #pragma unroll
                    for (int j = 0; j < 4; j++) acc[m][n][j] = fmaf(__uint_as_float(scale[m][j >> 1].x), sum[m][n][j], acc[m][n][j]);
        }
        __syncwarp();
        if (u + stages * step < u1) fetch(u + stages * step, slot);
        if (++slot == stages) { slot = 0; phase ^= 1; }
    }
    // Sums of the warps, in the shared memory that they had for their copies: [warp][8 NT][16 MT].
    constexpr int TILE = C::TILE;
    float* const sum = reinterpret_cast<float*>(smem);
    __syncthreads();
    if (abort_word != 0) {                                     // copies in flight land first, then what the block has is written
        for (int i = 0; i < 64; i++) __nanosleep(100000);
        if (threadIdx.x == 0 && a.status != nullptr && atomicCAS(a.status, 0, (int)KS_WAIT_TIMEOUT) == 0) {
            a.status[1] = blockIdx.x;
            a.status[2] = abort_word;
        }
        __syncthreads();
    }
    #pragma unroll
    for (int m = 0; m < MT; m++)
        #pragma unroll
        for (int n = 0; n < NT; n++)
            #pragma unroll
            for (int i = 0; i < 4; i++) sum[warp * TILE + (8 * n + 2 * t + (i & 1)) * CHANNELS + 16 * m + 8 * (i >> 1) + row] = acc[m][n][i];
    __syncthreads();
    for (int e = threadIdx.x; e < rows * CHANNELS; e += blockDim.x) {
        float v = sum[e];
        #pragma unroll
        for (int w = 1; w < warps; w++) v += sum[w * TILE + e];
        if (parts > 1) sum[e] = v;
        else store_sum(a, v, m0 + e / CHANNELS, n0 + e % CHANNELS);
    }
    if (parts > 1) {
        cluster_sync();
        store_sums(a, sum, rows, CHANNELS, parts, part, m0, n0);
        cluster_sync();                                        // the others may still read this block's sums
    }
}

template <int G, int NT>
int launch_w4(const W4Args& a, cudaStream_t stream)
{
    using C = W4Cfg<G, W4_MT, NT>;
    constexpr auto kernel = proj_w4_kernel<G, W4_MT, NT>;
    const int tiles = (a.d_out + C::CHANNELS - 1) / C::CHANNELS, row_tiles = (a.rows + 8 * NT - 1) / (8 * NT), units = (a.d_in + W4_K - 1) / W4_K;
    // Few tiles: a cluster shares k, as long as every warp has a unit and every block an SM. us in 1 / 2 / 4 parts: 16 rows, 8192 x 1024 10.0 / 7.0 / 5.6,
    // 4096 x 4096 (one part) 6.8 / 7.2.
    int parts = 1;
    while (parts < 8 && 2 * parts * W4_WARPS <= units && (long long)tiles * row_tiles * 2 * parts <= device_sms()) parts *= 2;
    CUtensorMap codes;
    const unsigned long long dims[2] = {(unsigned long long)a.d_in / 2, (unsigned long long)a.d_out}, strides[1] = {(unsigned long long)a.code_stride};
    const unsigned box[2] = {W4_K / 2, C::CHANNELS};
    if (make_tmap_u8(&codes, a.codes, 2, dims, strides, box)) return 1;
    const int rows = std::min(a.rows, 8 * NT);
    int stages = W4_STAGES;
    while (stages > 1 && C::smem(rows, stages) > W4_SMEM) stages--;
    static bool set[64] = {};
    int dev = 0;
    EFA_CUDA(cudaGetDevice(&dev));
    if (dev >= 64 || !set[dev]) {
        EFA_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, std::max(W4_SMEM, C::smem(8 * NT, 1))));
        if (dev < 64) set[dev] = true;
    }
    EFA_CUDA(launch_value(kernel, dim3(tiles, row_tiles, parts), W4_WARPS * 32, C::smem(rows, stages), stream, a, stages, codes));
    return 0;
}

template <int G>
int launch_group(const W4Args& a, cudaStream_t stream)
{
    return a.rows <= 8 ? launch_w4<G, 1>(a, stream) : launch_w4<G, 2>(a, stream);
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
    const void* const mem[] = {X, w.codes, w.scales, w.zeros, out};
    if (int rc = check_memory("project_w4", mem, 5)) return rc;
    const W4Args a{w.codes, static_cast<const __half*>(w.scales), w.zeros, static_cast<const __half*>(X), out, rows, w.d_in, w.d_out,
                   w.code_stride ? w.code_stride : w.d_in / 2, w.scale_stride ? w.scale_stride : w.d_out, w.zero_stride ? w.zero_stride : w.d_out,
                   x_stride ? x_stride : w.d_in, out_stride ? out_stride : w.d_out, out_dtype == EFA_F32, aligned16(out) && (out_stride ? out_stride : w.d_out) % 4 == 0, kernel_status_word()};
    // Up to eight rows the products of mma.sync are not the time. Beyond, tiles of 16 rows that read the weights again, or tcgen05 with up to 64 rows to a tile, whose start and
    // end cost more: by the work, in weights times tiles of 16. us, tiles of 16 / tcgen05: 16 rows, 4096 x 4096 6.8 / 8.8, 4096 x 6144 13.2 / 10.7, 8192 x 32768 55 / 39;
    // 32 rows, 2048 x 4096 7.9 / 8.2, 8192 x 1024 6.9 / 9.8, 4096 x 4096 9.8 / 10.1; 64 rows, 1024 x 1024 3.4 / 7.3, 1056 x 4163 15 / 12.4, 4096 x 4096 18 / 12.
    if (rows > 8 && (double)((rows + 15) / 16) * w.d_in * w.d_out > (double)(1 << 24)) return w4_tc_launch(a, w.group, stream);
    return w.group == 128 ? launch_group<128>(a, stream) : w.group == 64 ? launch_group<64>(a, stream) : launch_group<32>(a, stream);
}

}  // namespace efa
