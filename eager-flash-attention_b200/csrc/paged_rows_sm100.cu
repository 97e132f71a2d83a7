// Attention of few rows over the paged cache: the next token of each sequence, or some tokens, of all query heads that share a kv head
// (up to 64 rows to a tile; longer chunks as several tiles). For row i over the keys j it sees, with s_ij = scale * log2(e) * q_i . k_j,
//     m_i = max_j s_ij,  l_i = sum_j 2^(s_ij - m_i),  O_i = sum_j 2^(s_ij - m_i) v_j / l_i
// in one pass: m, l and O of what has been seen are rescaled when m grows.
//
// Few rows do little with each key that they load, so it is the loading that takes the time: every key and value comes from memory once per
// group of heads, and the blocks' work is a contiguous share of all keys of all sequences (paged_part), whatever their lengths.
// A block is four warps in teams: WM warps of 16 rows each share a team's keys, 4 / WM teams take 16 * WM keys each of a unit of 64 (8 bits: twice as many). A team has a
// ring of stages in shared memory that its warps fill with asynchronous 16-byte copies and wait for by themselves, so no barrier of
// the block is in the loop. The products are mma.sync m16n8k16: a tile of 16 rows is what there is, and tcgen05's least 64 rows would need the
// softmax to cross tensor memory for nothing.
//
// Measured (64 sequences of 129 to 8192 keys, one token, 32 heads of 128 on 8, fp16): 1.11 GB in 170 us, 6.5 TB/s; call after call on inputs in turn 177 us (6.27 TB/s,
// 0.96 of a copy). ncu (32 x 4096 keys): 537 MB from DRAM for 537 MB of keys and values, three of four stalls are waits for them.
// Of 8 bits: 16 sequences of 2051 to 32768 keys, up to four tokens: 0.60 GB in 110 us, 118 to 125 in turn, by the box (5.1 to 4.8 TB/s): half the bytes for the same arithmetic and the conversion, issue
// slots half busy with twelve warps that wait for their own results. Tried and slower: all keys' heads in another order of shares (0), two to six times as many
// shares (+0 to +20 %), values that are not finite made 0 in shared memory instead of in registers (small calls +15 %).
//
// fp16 keys reach the registers by ldmatrix. Codes of e4m3 are read as 16 bytes of a key per thread and converted there (exactly): the order of
// the head's elements in Q K^T, and that of O's columns, is then each thread's own, and Q's fragments and the stores follow it. The exponents of keys
// multiply the scores; those of values the converted values, which stay exact. In the weights, which are rounded to fp16, they would leave the others' a few bits beside
// a value row 2^16 times as large, in columns where they are all there is; and be slower for the softmax's part in it (us, 64 sequences of 4096 keys, one token, exponents
// in the weights / here: 32 heads of 128 on 8 102.2 / 100.6, 16 of 64 128.4 / 121.2, 32 of 32 185.5 / 170.2, 64 of 16 322.6 / 277.6).
#include "paged_kernels.cuh"
#include "fa_args.cuh"

#include <climits>

namespace efa {

namespace {

constexpr int PR_THREADS = 128;

// Blocks of an SM and stages of each: where loading is the time (fp16 heads of 64 and 128) few blocks with deep rings, else more warps. us, 64 sequences of 4096
// keys, one token, as here / as two blocks of 96 KB: 16 heads of 64 fp16 168 / 168 (three blocks of 64 KB: 210), 8 bits 122 / 133; 32 heads of
// 32 181 / 207, 171 / 196; 64 heads of 16 256 / 352, 276 / 394; 16 sequences of 16000 keys, 8 heads of 128 165 / 166, 95 / 101.
constexpr int rows_blocks(int d, bool f8) { return d >= 64 ? (f8 ? 3 : 2) : d == 16 && f8 ? 6 : 4; }
template <int D, bool F8> constexpr int blocks_of = rows_blocks(D, F8);
constexpr int rows_stages(int d, bool f8) { return d == 128 ? (f8 ? 2 : 3) : d == 64 ? (f8 ? 4 : 6) : d == 16 && f8 ? 4 : 6; }

template <int D, bool F8, int WM>
struct RowsCfg {
    static constexpr int WK = F8 ? 32 : 16;                                   // keys that a warp copies of a unit
    static constexpr int TEAMS = 4 / WM, TILE = 16 * WM, KS = WK * WM, UNIT = KS * TEAMS;       // rows; a team's keys of a unit; keys of a unit
    static constexpr int STEP = KS >= 32 ? 2 : 1;                             // 16-key blocks to a step of the softmax
    static constexpr int RB = D * (F8 ? 1 : 2);                               // bytes of a key
    static constexpr int STAGE = 2 * KS * RB + (F8 ? 2 * KS : 0);             // of a team
    static constexpr int UNIT_BYTES = TEAMS * STAGE;
    static constexpr int STAGES = rows_stages(D, F8);
    static constexpr int RING = STAGES * UNIT_BYTES;
    static constexpr int OPITCH = D + 4;
    static constexpr int MERGE = 4 * 16 * OPITCH * 4 + 8 * 16 * 8;            // four warps' O, their (m, l), and that of the block
    static constexpr int SMEM = RING > MERGE ? RING : MERGE;
};

// Where 16-byte chunk c of key r of a stage lies. Rows of 128 bytes or more: chunk ^ f(r), f one to one on 0..7, so that eight rows' equal chunks (ldmatrix)
// lie in eight different bank groups; f(2p) and f(2p+1) differ in bit 2 (two keys x four chunks, a phase of the e4m3 key loads), and f(0), f(2), f(4),
// f(6) above bit 0 (two chunks x four keys, a phase of its value loads). Shorter rows: the same over lines of 128 bytes.
template <int RB>
__device__ __forceinline__ int rows_swizzled(int r, int c)
{
    if constexpr (RB >= 128) return r * RB + ((c ^ ((r & 7) ^ ((r & 1) << 2))) << 4);
    if constexpr (RB == 64) return (r >> 1) * 128 + ((((r & 1) * 4 + c) ^ ((0x6530 >> (4 * ((r >> 1) & 3))) & 7)) << 4);
    if constexpr (RB == 32) return (r >> 2) * 128 + ((((r & 3) * 2 + c) ^ ((r >> 2) & 1)) << 4);
    return r * RB + (c << 4);
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// BYTES (2 to 16) of shared memory as words.
template <int BYTES>
__device__ __forceinline__ void load_words(uint32_t addr, uint32_t (&w)[4])
{
    if constexpr (BYTES == 16) asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr) : "memory");
    if constexpr (BYTES == 8) asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr) : "memory");
    if constexpr (BYTES == 4) asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(addr) : "memory");
    if constexpr (BYTES == 2) asm volatile("{\n.reg .b16 x;\nld.shared.b16 x, [%1];\ncvt.u32.u16 %0, x;\n}\n" : "=r"(w[0]) : "r"(addr) : "memory");
}

__device__ __forceinline__ uint32_t load_half(uint32_t addr)
{
    uint32_t w[4];
    load_words<2>(addr, w);
    return w[0];
}

__device__ __forceinline__ float max3(float a, float b, float c)
{
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

template <int N>
__device__ __forceinline__ void load_cluster(uint32_t addr, float (&v)[N])
{
    if constexpr (N == 2) {
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v[0]), "=f"(v[1]) : "r"(addr) : "memory");
    } else {
        #pragma unroll
        for (int i = 0; i < N; i += 4)
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[i]), "=f"(v[i + 1]), "=f"(v[i + 2]), "=f"(v[i + 3]) : "r"(addr + i * 4) : "memory");
    }
}

// Eight columns of a row of O; none: the row sees nothing.
__device__ __forceinline__ void store_row8(__half* dst, const float (&acc)[8], float sum, bool none)
{
    const float inv = 1.f / sum;
    uint4 out;
    uint32_t* w = &out.x;
    #pragma unroll
    for (int x = 0; x < 4; x++) w[x] = none ? 0u : pack_f16x2(acc[2 * x] * inv, acc[2 * x + 1] * inv);
    *reinterpret_cast<uint4*>(dst) = out;
}

template <int D, bool F8, int WM>
__global__ void __launch_bounds__(PR_THREADS, blocks_of<D, F8>)
paged_rows_kernel(const PagedArgs c, const PagedAttnArgs a)
{
    using C = RowsCfg<D, F8, WM>;
    constexpr int RB = C::RB, KS = C::KS, NT = D / 8, KSTEPS = D / 16;
    constexpr int EB = D / 4 < 16 ? D / 4 : 16;            // e4m3: bytes of a key that a thread reads at a time
    constexpr int VB = D / 8;                              // e4m3: bytes of a value row that a thread reads, its columns of O

    extern __shared__ __align__(128) uint8_t smem_rows[];
    __shared__ PagedScratch scratch;

    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const int g = lane >> 2, t = lane & 3;                 // row pair and column pair of the fragments
    const int team = warp / WM, mrow = warp % WM;

    pdl_wait();
    pdl_trigger();

    PagedAt at, first;
    int left;
    const bool cut = a.parts.cut != nullptr;
    if (cut) {
        left = paged_part<PR_THREADS>(c, a.w, blockIdx.x, gridDim.x, scratch, at, 51);
        first = at;
        if (tid == 0) {
            PagedCut here{};
            if (left > 0) here = PagedCut{at.h, at.b, at.rt, max(0, at.off - a.w.extra), paged_units(a.w, paged_seq(c, at.b), at.rt), 0, 0, 0};
            a.parts.cut[blockIdx.x] = here;
        }
    } else {
        const int per = c.H_kv * a.w.max_tiles, b = blockIdx.x / per, rest = blockIdx.x - b * per;
        at = first = PagedAt{rest % c.H_kv, b, rest / c.H_kv, 0};
        if (tid == 0 && rest == 0 && blockIdx.z == 0) paged_seq<true>(c, b, 51);
        left = at.rt < paged_tiles(a.w, paged_seq(c, b)) ? INT_MAX : 0;
    }

    const uint32_t ring = smem_u32(smem_rows) + team * C::STAGE;       // stage s of this team: + s * UNIT_BYTES

    for (; left > 0; paged_next(c, a.w, at)) {
        const PagedPiece piece = paged_piece(c, a.w, at, left);
        const PagedSeq& q = piece.q;
        int u_lo = piece.u_lo, u_hi = piece.u_hi;
        const bool whole = u_lo == 0 && u_hi == piece.units;
        if (cut) {
            if (u_hi == u_lo) continue;
        } else {
            left = 0;
            if (gridDim.z > 1) {                           // a cluster's blocks share the item
                u_lo = (int)((unsigned)(piece.units * blockIdx.z) / gridDim.z);
                u_hi = (int)((unsigned)(piece.units * (blockIdx.z + 1)) / gridDim.z);
            }
        }
        const int rows = min(C::TILE, q.n * a.w.G - at.rt * C::TILE), r0 = at.rt * C::TILE;      // of the item

        // ---- the asynchronous copies of a unit: this warp's WK keys of the team's, 16 at a time (they are in one page)
        int page_of = 0, page_from = u_lo - 32;            // lane l: page of 16 keys, WK / 16 lanes to a unit from unit page_from on
        const int first_key = team * KS + mrow * C::WK;
        constexpr int PER = C::WK / 16, AHEAD = 32 / PER;
        uint32_t to[PER][(RB + 31) / 32];                  // where this lane's chunks go in a stage
        #pragma unroll
        for (int x = 0; x < PER; x++)
            #pragma unroll
            for (int i = 0; i < (RB + 31) / 32; i++) to[x][i] = ring + rows_swizzled<RB>(mrow * C::WK + x * 16 + (i * 32 + lane) / (RB / 16), (i * 32 + lane) % (RB / 16));
        auto load = [&](int u) {
            if (u < u_hi) {
                if (u - page_from >= AHEAD) {
                    page_from = u;
                    const int un = u + lane / PER, key = un * C::UNIT + first_key + lane % PER * 16;
                    page_of = key < q.kv && un < u_hi ? paged_page(c, at.b, key, 52) : -1;
                }
                const uint32_t stage = ((u - u_lo) % C::STAGES) * C::UNIT_BYTES;
                #pragma unroll
                for (int x = 0; x < PER; x++) {
                    const int page = __shfl_sync(0xffffffffu, page_of, (u - page_from) * PER + x);
                    const int key = u * C::UNIT + first_key + x * 16;
                    const int there = page >= 0 ? q.kv - key : 0;                 // keys that exist
                    const int row = (at.h << c.page_shift) + (key & ((1 << c.page_shift) - 1));
                    const long long src = (long long)max(page, 0) * c.page_stride + (long long)row * RB + lane * 16;
                    const uint8_t* ks = c.k + src;
                    const uint8_t* vs = c.v + src;
                    #pragma unroll
                    for (int i = 0; i < (RB + 31) / 32; i++) {
                        const bool is = (i * 32 + lane) / (RB / 16) < there;
                        if (RB < 32 && lane >= RB) break;
                        copy16(to[x][i] + stage, ks + i * 512, is);
                        copy16(to[x][i] + stage + KS * RB, vs + i * 512, is);
                    }
                    if (F8 && lane < 2) {
                        const long long e = ((long long)max(page, 0) * c.H_kv << c.page_shift) + row;
                        copy16(ring + stage + 2 * KS * RB + lane * KS + mrow * C::WK + x * 16, (lane ? c.v_exp : c.k_exp) + e, there > 0);
                    }
                }
            }
            copy_commit();
        };
        #pragma unroll
        for (int i = 0; i < C::STAGES - 1; i++) load(u_lo + i);

        // ---- Q fragments: rows g and g + 8 of this warp's 16
        uint32_t qf[KSTEPS][4];
        int sees[2];                                       // keys below this
        #pragma unroll
        for (int half = 0; half < 2; half++) {
            const int rr = mrow * 16 + g + half * 8, r = r0 + rr;
            const bool valid = rr < rows;
            sees[half] = valid ? paged_visible(a.w, q, r) : q.kv;
            const int token = valid ? r / a.w.G : 0;
            const __half* src = a.Q + (long long)(at.h * a.w.G + (valid ? r - token * a.w.G : 0)) * a.q_head + (long long)(q.row0 + token) * a.q_token;
            #pragma unroll
            for (int s = 0; s < KSTEPS; s++) {
                if constexpr (F8) {
                    const int col = (t + 4 * (s / (EB / 4))) * EB + (s % (EB / 4)) * 4;
                    const uint2 x = valid ? *reinterpret_cast<const uint2*>(src + col) : make_uint2(0u, 0u);
                    qf[s][half] = x.x;
                    qf[s][2 + half] = x.y;
                } else {
                    qf[s][half] = valid ? *reinterpret_cast<const uint32_t*>(src + s * 16 + t * 2) : 0u;
                    qf[s][2 + half] = valid ? *reinterpret_cast<const uint32_t*>(src + s * 16 + t * 2 + 8) : 0u;
                }
            }
        }
        // Keys that every row of this warp sees need no mask.
        const int all_see = __reduce_min_sync(0xffffffffu, min(min(sees[0], sees[1]), q.kv));

        float o[NT][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
        #pragma unroll
        for (int j = 0; j < NT; j++) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
        bool poison = false;                               // a value that some row does not see is not finite

        for (int u = u_lo; u < u_hi; u++) {
            copy_wait<C::STAGES - 2>();
            if constexpr (WM == 1) __syncwarp();
            else asm volatile("bar.sync %0, %1;" :: "r"(1 + team), "n"(32 * WM) : "memory");
            load(u + C::STAGES - 1);
            const uint32_t sk = ring + ((u - u_lo) % C::STAGES) * C::UNIT_BYTES, sv = sk + KS * RB, se = sv + KS * RB;
            constexpr int STEP = C::STEP, KT = 2 * STEP;   // key tiles of 8 in a step
            #pragma unroll 1
            for (int blk = 0; blk < KS / 16; blk += STEP) {
                const int key0 = u * C::UNIT + team * KS + blk * 16;
                if (key0 >= q.kv) break;
                // ---- S = Q K^T, 16 rows x KT * 8 keys
                float s[KT][4] = {};
                if constexpr (F8) {
                    #pragma unroll
                    for (int i = 0; i < D / (4 * EB); i++) {
                        uint32_t w[KT][4];
                        const int byte = (t + 4 * i) * EB;
                        #pragma unroll
                        for (int nt = 0; nt < KT; nt++) load_words<EB>(sk + rows_swizzled<RB>(blk * 16 + nt * 8 + g, byte >> 4) + (byte & 15), w[nt]);
                        #pragma unroll
                        for (int x = 0; x < EB / 4; x++)
                            #pragma unroll
                            for (int nt = 0; nt < KT; nt++) {
                                uint32_t b0, b1;
                                e4m3x4_to_f16x4(w[nt][x], b0, b1);
                                mma16816(s[nt], qf[i * (EB / 4) + x], b0, b1);
                            }
                    }
                } else {
                    #pragma unroll
                    for (int st = 0; st < KSTEPS; st++)
                        #pragma unroll
                        for (int y = 0; y < STEP; y++) {
                            uint32_t w[4];
                            ldsm4(sk + rows_swizzled<RB>((blk + y) * 16 + (lane & 7) + ((lane >> 4) << 3), st * 2 + ((lane >> 3) & 1)), w);
                            mma16816(s[2 * y], qf[st], w[0], w[1]);
                            mma16816(s[2 * y + 1], qf[st], w[2], w[3]);
                        }
                }
                // ---- softmax; this thread has keys key0 + nt * 8 + t * 2 + {0, 1} of rows g (s[.][0..1]) and g + 8
                uint32_t vexp[KT];                         // e4m3: 2^exponent of the two keys' values
                #pragma unroll
                for (int nt = 0; nt < KT; nt++) {
                    float f0 = a.scale_log2e, f1 = f0;
                    if constexpr (F8) {
                        const uint32_t ke = load_half(se + blk * 16 + nt * 8 + t * 2), ve = load_half(se + KS + blk * 16 + nt * 8 + t * 2);
                        f0 *= exp_byte_f32(ke & 0xffu);
                        f1 *= exp_byte_f32(ke >> 8);
                        vexp[nt] = exp_bytes_f16x2(ve);
                    }
                    s[nt][0] *= f0; s[nt][1] *= f1; s[nt][2] *= f0; s[nt][3] *= f1;
                }
                const bool masked = key0 + STEP * 16 > all_see;
                if (masked) {
                    #pragma unroll
                    for (int nt = 0; nt < KT; nt++)
                        #pragma unroll
                        for (int x = 0; x < 4; x++)
                            if (key0 + nt * 8 + t * 2 + (x & 1) >= min(sees[x >> 1], q.kv)) s[nt][x] = -INFINITY;
                }
                // The offset m is a row's largest weight so far, or up to rescale_above less: O is rescaled when it moves, and of 16 rows one would nearly always have a
                // new maximum.
                float off[2], mx[2];
                #pragma unroll
                for (int half = 0; half < 2; half++) {
                    mx[half] = -INFINITY;
                    #pragma unroll
                    for (int nt = 0; nt < KT; nt++) mx[half] = max3(mx[half], s[nt][half * 2], s[nt][half * 2 + 1]);
                    mx[half] = fmaxf(mx[half], __shfl_xor_sync(0xffffffffu, mx[half], 1));
                    mx[half] = fmaxf(mx[half], __shfl_xor_sync(0xffffffffu, mx[half], 2));
                }
                if (__any_sync(0xffffffffu, mx[0] > m[0] + a.rescale_above || mx[1] > m[1] + a.rescale_above)) {
                    float alpha[2];
                    #pragma unroll
                    for (int half = 0; half < 2; half++) {
                        const float top = fmaxf(m[half], mx[half]);
                        alpha[half] = m[half] == top ? 1.f : ex2(m[half] - (top == -INFINITY ? 0.f : top));
                        m[half] = top;
                        l[half] *= alpha[half];
                    }
                    #pragma unroll
                    for (int j = 0; j < NT; j++) { o[j][0] *= alpha[0]; o[j][1] *= alpha[0]; o[j][2] *= alpha[1]; o[j][3] *= alpha[1]; }
                }
                #pragma unroll
                for (int half = 0; half < 2; half++) off[half] = m[half] == -INFINITY ? 0.f : m[half];
                uint32_t p[STEP][4];
                #pragma unroll
                for (int nt = 0; nt < KT; nt++)
                    #pragma unroll
                    for (int half = 0; half < 2; half++) {
                        const float p0 = ex2(s[nt][half * 2] - off[half]), p1 = ex2(s[nt][half * 2 + 1] - off[half]);
                        l[half] += p0 + p1;
                        p[nt >> 1][(nt & 1) * 2 + half] = pack_f16x2(p0, p1);
                    }
                // ---- O += P V. A masked weight is 0, and 0 times what is not finite is not 0: such values are left out here and, for the rows that
                // do see them, put in at the end.
                auto clean = [&](uint32_t& w) {
                    const uint32_t bad = nonfinite_f16x2(w);
                    poison |= bad != 0;
                    w &= ~bad;
                };
                #pragma unroll
                for (int y = 0; y < STEP; y++) {
                    if constexpr (F8) {
                        uint32_t w[4][4];                  // keys t * 2, t * 2 + 1, t * 2 + 8, t * 2 + 9
                        #pragma unroll
                        for (int i = 0; i < 4; i++)
                            load_words<VB>(sv + rows_swizzled<RB>((blk + y) * 16 + (i >> 1) * 8 + t * 2 + (i & 1), (g * VB) >> 4) + ((g * VB) & 15), w[i]);
                        #pragma unroll
                        for (int j = 0; j < NT; j += 2) {  // columns j and j + 1: of each the codes of two keys side by side, then converted
                            const uint32_t sel = j & 2 ? 0x7362 : 0x5140;
                            uint32_t b0, b1, b2, b3;
                            e4m3x4_to_f16x4(__byte_perm(w[0][j >> 2], w[1][j >> 2], sel), b0, b2);
                            e4m3x4_to_f16x4(__byte_perm(w[2][j >> 2], w[3][j >> 2], sel), b1, b3);
                            b0 = mul_f16x2(b0, vexp[2 * y]); b1 = mul_f16x2(b1, vexp[2 * y + 1]);
                            b2 = mul_f16x2(b2, vexp[2 * y]); b3 = mul_f16x2(b3, vexp[2 * y + 1]);
                            if (masked) { clean(b0); clean(b1); clean(b2); clean(b3); }
                            mma16816(o[j], p[y], b0, b1);
                            mma16816(o[j + 1], p[y], b2, b3);
                        }
                    } else {
                        #pragma unroll
                        for (int j = 0; j < NT; j += 2) {
                            uint32_t w[4];
                            ldsm4_t(sv + rows_swizzled<RB>((blk + y) * 16 + (lane & 7) + (((lane >> 3) & 1) << 3), j + (lane >> 4)), w);
                            if (masked) { clean(w[0]); clean(w[1]); clean(w[2]); clean(w[3]); }
                            mma16816(o[j], p[y], w[0], w[1]);
                            mma16816(o[j + 1], p[y], w[2], w[3]);
                        }
                    }
                }
            }
        }
        copy_wait<0>();

        // Column of O that o[j][.] with column pair x (0, 1) is.
        auto column = [&](int j, int x) { return F8 ? (t * 2 + x) * VB + j : j * 8 + t * 2 + x; };
        if (__any_sync(0xffffffffu, poison)) {
            // Rare: the values that are not finite, of keys that some row of the warp does not see, for the rows that see them.
            for (int u = max(u_lo, max(all_see, 0) / C::UNIT); u < u_hi; u++)
                for (int x = 0; x < KS; x++) {
                    const int key = u * C::UNIT + team * KS + x;
                    if (key >= q.kv || (key | (16 * C::STEP - 1)) < all_see) continue;
                    const int page = paged_page(c, at.b, key, 52);
                    if (page < 0) continue;
                    const int row = (at.h << c.page_shift) + (key & ((1 << c.page_shift) - 1));
                    const uint8_t* src = c.v + (long long)page * c.page_stride + (long long)row * RB;
                    for (int half = 0; half < 2; half++) {
                        if (key >= sees[half]) continue;
                        #pragma unroll
                        for (int j = 0; j < NT; j++)
                            #pragma unroll
                            for (int y = 0; y < 2; y++) {
                                float v;
                                if constexpr (F8) v = (src[column(j, y)] & 0x7f) == 0x7f ? NAN : 0.f;
                                else v = __half2float(reinterpret_cast<const __half*>(src)[column(j, y)]);
                                if (!isfinite(v)) o[j][half * 2 + y] += v;
                            }
                    }
                }
        }

        // ---- the warps' results, merged through shared memory (the ring has been read by now)
        #pragma unroll
        for (int half = 0; half < 2; half++) {
            l[half] += __shfl_xor_sync(0xffffffffu, l[half], 1);
            l[half] += __shfl_xor_sync(0xffffffffu, l[half], 2);
        }
        __syncthreads();
        float* so = reinterpret_cast<float*>(smem_rows);                               // [4][16][OPITCH]
        float2* sml = reinterpret_cast<float2*>(so + 4 * 16 * C::OPITCH);              // [4][16]
        #pragma unroll
        for (int half = 0; half < 2; half++) {
            const int rr = warp * 16 + g + half * 8;
            if (t == 0) sml[rr] = make_float2(m[half], l[half]);
            float* dst = so + rr * C::OPITCH;
            #pragma unroll
            for (int j = 0; j < NT; j++) { dst[column(j, 0)] = o[j][half * 2]; dst[column(j, 1)] = o[j][half * 2 + 1]; }
        }
        __syncthreads();
        const int place = (int)blockIdx.x * 2 + (at.h == first.h && at.b == first.b && at.rt == first.rt ? 0 : 1);
        for (int e = tid; e < rows * (D / 8); e += PR_THREADS) {
            const int rr = whole ? e / (D / 8) : e % rows, col = (whole ? e % (D / 8) : e / rows) * 8;
            float top = -INFINITY, sum = 0.f, acc[8] = {};
            #pragma unroll
            for (int i = 0; i < C::TEAMS; i++) top = fmaxf(top, sml[i * C::TILE + rr].x);
            #pragma unroll
            for (int i = 0; i < C::TEAMS; i++) {
                const float2 ml = sml[i * C::TILE + rr];
                const float w = ml.x == top ? 1.f : ex2(ml.x - top);
                sum += w * ml.y;
                const float* src = so + (i * C::TILE + rr) * C::OPITCH + col;
                #pragma unroll
                for (int x = 0; x < 8; x++) acc[x] += w * src[x];
            }
            if (gridDim.z > 1) {
                float* dst = so + rr * C::OPITCH + col;                                // the first team's place, which only this thread reads
                #pragma unroll
                for (int x = 0; x < 8; x++) dst[x] = acc[x];
                if (col == 0) sml[4 * 16 + rr] = make_float2(top, sum);
            } else if (whole) {
                const int r = r0 + rr, token = r / a.w.G;
                store_row8(a.O + (long long)(q.row0 + token) * a.o_token + (long long)(at.h * a.w.G + r - token * a.w.G) * D + col, acc, sum, paged_visible(a.w, q, r) <= 0);
            } else {
                float4* dst = a.parts.o + ((long long)place * (D / 4) + col / 4) * C::TILE + rr;
                dst[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
                dst[C::TILE] = make_float4(acc[4], acc[5], acc[6], acc[7]);
                if (col == 0) a.parts.ml[(long long)place * C::TILE + rr] = make_float2(top, sum);
            }
        }
        if (gridDim.z > 1) {
            // The cluster's blocks, each for its part of the elements, out of one another's shared memory.
            cluster_sync();
            for (int e = blockIdx.z * PR_THREADS + tid; e < rows * (D / 8); e += gridDim.z * PR_THREADS) {
                const int rr = e / (D / 8), col = (e % (D / 8)) * 8, r = r0 + rr, token = r / a.w.G;
                float top = -INFINITY, sum = 0.f, acc[8] = {};
                #pragma unroll 4
                for (unsigned i = 0; i < gridDim.z; i++) {
                    float ml[2], v[8];
                    load_cluster(cluster_addr(&sml[4 * 16 + rr], i), ml);
                    load_cluster(cluster_addr(so + rr * C::OPITCH + col, i), v);
                    const float m = fmaxf(top, ml[0]), old = top == m ? 1.f : ex2(top - m), w = ml[0] == m ? 1.f : ex2(ml[0] - m);
                    top = m;
                    sum = sum * old + w * ml[1];
                    #pragma unroll
                    for (int x = 0; x < 8; x++) acc[x] = acc[x] * old + w * v[x];
                }
                store_row8(a.O + (long long)(q.row0 + token) * a.o_token + (long long)(at.h * a.w.G + r - token * a.w.G) * D + col, acc, sum, paged_visible(a.w, q, r) <= 0);
            }
            cluster_sync();
        }
        __syncthreads();
        if (left <= 0) break;          // not on to an item that is not there
    }
}

// Merge of what the blocks left of the items that a cut goes through (PagedCut), over the pieces i of an item:
//     O = sum_i 2^(m_i - max m) O_i / sum_i 2^(m_i - max m) l_i.
// Blocks (x, .) look at the beginning of share x + 1: where that is the first cut through its item they merge the item, a thread eight columns of
// a row at a time. Bound by the latency of the pieces' loads: BATCH pieces are asked for at once, and PG threads share a row's pieces where an item may
// be cut into many.
constexpr int PM_THREADS = 256;
template <int D, int PG>
__global__ void __launch_bounds__(PM_THREADS)
paged_merge_kernel(const PagedArgs c, const PagedAttnArgs a, int parts)
{
    constexpr int BATCH = PG > 1 ? 4 : 2;
    __shared__ float sm_acc[PG > 1 ? (PG - 1) * (PM_THREADS / PG) : 1][11];
    pdl_wait();
    pdl_trigger();
    const int part = blockIdx.x + 1;
    const PagedCut here = a.parts.cut[part], ahead = a.parts.cut[part - 1];
    auto same = [&](const PagedCut& x) { return x.units > 0 && x.h == here.h && x.b == here.b && x.rt == here.rt; };
    if (here.off == 0 || (same(ahead) && ahead.off > 0)) return;     // no cut, or not the item's first
    const PagedSeq q = paged_seq(c, here.b);
    const int tile = a.w.tile, rows = min(tile, q.n * a.w.G - here.rt * tile);
    // Piece 0 is the one of share part - 1, piece i that of share part - 1 + i, which begins inside the item.
    int pieces = 2, more;
    do {
        const int next = part - 1 + pieces + (int)threadIdx.x;
        more = __syncthreads_count(next < parts && same(a.parts.cut[next]));
        pieces += more;
    } while (more == PM_THREADS);
    const int place0 = (part - 1) * 2 + (same(ahead) ? 0 : 1);
    const int group = threadIdx.x / (PM_THREADS / PG), local = threadIdx.x % (PM_THREADS / PG);

    for (int x = blockIdx.y * (PM_THREADS / PG) + local; x - local < rows * (D / 8); x += gridDim.y * (PM_THREADS / PG)) {
        const bool mine = x < rows * (D / 8);
        const int rr = mine ? x % rows : 0, col = mine ? x / rows * 8 : 0;
        float top = -INFINITY, sum = 0.f, acc[8] = {};
        for (int i0 = group; i0 < pieces && mine; i0 += PG * BATCH) {
            float2 ml[BATCH];
            float4 o[BATCH][2];
            #pragma unroll
            for (int k = 0; k < BATCH; k++) {
                const int i = min(i0 + k * PG, pieces - 1);
                const long long place = i == 0 ? place0 : (part - 1 + i) * 2;
                ml[k] = __ldcg(a.parts.ml + place * tile + rr);
                const float4* src = a.parts.o + (place * (D / 4) + col / 4) * tile + rr;
                o[k][0] = __ldcg(src);
                o[k][1] = __ldcg(src + tile);
            }
            #pragma unroll
            for (int k = 0; k < BATCH; k++) {
                if (i0 + k * PG >= pieces) break;
                const float m = fmaxf(top, ml[k].x), old = top == m ? 1.f : ex2(top - m), w = ml[k].x == m ? 1.f : ex2(ml[k].x - m);
                const float* v = &o[k][0].x;
                top = m;
                sum = sum * old + w * ml[k].y;
                #pragma unroll
                for (int y = 0; y < 8; y++) acc[y] = acc[y] * old + w * v[y];
            }
        }
        if constexpr (PG > 1) {
            float* to = sm_acc[group > 0 ? (group - 1) * (PM_THREADS / PG) + local : 0];
            if (group > 0) {
                to[0] = top; to[1] = sum;
                #pragma unroll
                for (int y = 0; y < 8; y++) to[2 + y] = acc[y];
            }
            __syncthreads();
            if (group == 0) {
                #pragma unroll
                for (int k = 0; k < PG - 1; k++) {
                    if (k + 1 >= pieces) break;
                    const float* v = sm_acc[k * (PM_THREADS / PG) + local];
                    const float m = fmaxf(top, v[0]), old = top == m ? 1.f : ex2(top - m), w = v[0] == m ? 1.f : ex2(v[0] - m);
                    top = m;
                    sum = sum * old + w * v[1];
                    #pragma unroll
                    for (int y = 0; y < 8; y++) acc[y] = acc[y] * old + w * v[2 + y];
                }
            }
            __syncthreads();
        }
        if (!mine || group > 0) continue;
        const int r = here.rt * tile + rr, token = r / a.w.G;
        store_row8(a.O + (long long)(q.row0 + token) * a.o_token + (long long)(here.h * a.w.G + r - token * a.w.G) * D + col, acc, sum, paged_visible(a.w, q, r) <= 0);
    }
}

template <int D, bool F8, int WM>
int launch_rows(const PagedArgs& c, const PagedAttnArgs& a, int blocks, int cluster, cudaStream_t stream)
{
    using C = RowsCfg<D, F8, WM>;
    static bool configured[64] = {};
    int dev = 0;
    EFA_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        EFA_CUDA(cudaFuncSetAttribute(paged_rows_kernel<D, F8, WM>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    EFA_CUDA(paged_launch(paged_rows_kernel<D, F8, WM>, dim3(blocks, 1, cluster), PR_THREADS, C::SMEM, stream, c, a));
    return 0;
}

template <int D, bool F8>
int launch_rows(const PagedArgs& c, const PagedAttnArgs& a, int blocks, int cluster, cudaStream_t stream)
{
    switch (a.w.tile) {
        case 16: return launch_rows<D, F8, 1>(c, a, blocks, cluster, stream);
        case 32: return launch_rows<D, F8, 2>(c, a, blocks, cluster, stream);
        default: return launch_rows<D, F8, 4>(c, a, blocks, cluster, stream);
    }
}

}  // namespace

int paged_rows_tile(int rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }

int paged_rows_blocks_per_sm(int d_h, bool f8) { return rows_blocks(d_h, f8); }
int paged_rows_unit(bool f8) { return f8 ? 128 : 64; }

int paged_rows_launch(const PagedArgs& c, const PagedAttnArgs& a, int d_h, bool f8, int blocks, int cluster, cudaStream_t stream)
{
    switch (d_h) {
        case 16:  return f8 ? launch_rows<16, true>(c, a, blocks, cluster, stream) : launch_rows<16, false>(c, a, blocks, cluster, stream);
        case 32:  return f8 ? launch_rows<32, true>(c, a, blocks, cluster, stream) : launch_rows<32, false>(c, a, blocks, cluster, stream);
        case 64:  return f8 ? launch_rows<64, true>(c, a, blocks, cluster, stream) : launch_rows<64, false>(c, a, blocks, cluster, stream);
        default:  return f8 ? launch_rows<128, true>(c, a, blocks, cluster, stream) : launch_rows<128, false>(c, a, blocks, cluster, stream);
    }
}

template <int D>
static int launch_merge(const PagedArgs& c, const PagedAttnArgs& a, int blocks, int most_rows, cudaStream_t stream)
{
    // Tiles of few rows may be in hundreds of pieces, tiles of 256 rows mostly are in two or three.
    const int units = most_rows * (D / 8);
    if (a.w.tile <= 64) EFA_CUDA(paged_launch(paged_merge_kernel<D, 4>, dim3(blocks - 1, (units + 63) / 64), PM_THREADS, 0, stream, c, a, blocks));
    else EFA_CUDA(paged_launch(paged_merge_kernel<D, 1>, dim3(blocks - 1, (units + 511) / 512), PM_THREADS, 0, stream, c, a, blocks));
    return 0;
}

int paged_merge_launch(const PagedArgs& c, const PagedAttnArgs& a, int d_h, int blocks, int most_rows, cudaStream_t stream)
{
    switch (d_h) {
        case 16:  return launch_merge<16>(c, a, blocks, most_rows, stream);
        case 32:  return launch_merge<32>(c, a, blocks, most_rows, stream);
        case 64:  return launch_merge<64>(c, a, blocks, most_rows, stream);
        default:  return launch_merge<128>(c, a, blocks, most_rows, stream);
    }
}

}  // namespace efa
