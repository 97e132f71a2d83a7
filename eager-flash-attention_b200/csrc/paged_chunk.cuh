// Attention of long chunks over the paged cache (tensor-bound): tiles of 256 rows (token, query head of a group) of one sequence and kv head against its keys,
// 128 at a time; heads of 128, and smaller ones of 8 bits (of fp16 they have a kernel of their own, paged_chains.cuh). Included by fa_fwd_ws_sm100.cu, whose kernel's roles, chains and softmax it has: two 128-row tiles, each a chain
// S -> softmax -> P -> P*V -> Q*K^T -> S in tensor memory, half a period apart. What differs:
//   * Q's rows come from anywhere (a row's token and head are r / G and r % G): the softmax threads load a row each and swizzle it by hand.
//   * A stage's keys are pages: one TMA box per page and 64 columns, issued by the lanes of the producer warp side by side. A page that is
//     none, or keys that are not there, are boxes outside the tensor, which read as zeros.
//   * Where some row of the item does not see some key of a stage (the last stages), values there that are not finite must not meet the weight 0
//     of such a row: warps 10 and 11 put zeros in their place before the MMA may have the stage, and the rows that do see them add them at the end. What a page holds
//     behind the last key is left out of that: it may be anything, and the search for it cost prompts four to six times their time.
//   * e4m3: the codes (and exponent bytes) arrive in a small ring of their own, and four more warps convert every stage to fp16, exactly.
//   * Work is an item, or an equal share of all 128-key units of all items (paged_part), an item at a time; the barriers are rebuilt for each. What a share
//     has of an item that is cut goes to the workspace, as fp32 O relative to the row's maximum, and is merged afterwards.
//
// Measured: 2048 tokens x 32 heads of 128 on 8, 32768 keys: 1020 us (1.04 PFLOP/s, 0.63 of the burst peak, 0.77 of the sustained one; at the power limit), as shares 1080. A
// unit (256 rows x 128 keys) is 2.0 to 2.3 us, of 8 bits 2.6; what an item costs besides is 4 us to its first scores (lengths, Q, first keys), 1.5 behind the last (its
// softmax and P*V) and 2 to store. ncu (512 tokens, 8192 keys): tensor pipe 51 % of active cycles, 38 MB from DRAM. The conversion of 8 bits is in a loop
// that is not unrolled: with the softmax's code it is then about what the instruction caches hold (512 tokens, 8192 keys: 84 us, unrolled 115, fp16 75). Slower
// still: codes from memory straight into the converting warps' registers (167, they spill), two warps on keys and two on values (164). O through shared memory
// for stores of whole lines: +3 %. An item of one tile by both warpgroups, every second stage each: fp16, 64 rows x 16000 keys, 198 -> 188, but items of two tiles +3 %
// and 8 bits +30 %, where the conversion is then the chain; the softmax's registers go to it.
#pragma once

template <bool F8> constexpr int chunk_threads = F8 ? 512 : 384;

template <int D, bool F8>
struct ChunkCfg {
    // Threads: the softmax's 256, a warpgroup of producer, issuer and warps 10 and 11, and for e4m3 another that converts. Registers of each:
    // together no more than the block is launched with.
    static constexpr int THREADS    = chunk_threads<F8>;
    static constexpr int REG_SOFTMAX = F8 ? 208 : 224, REG_ISSUE = F8 ? 40 : 56, REG_CONVERT = 56;
    static constexpr int REGS       = 256 * REG_SOFTMAX + 128 * REG_ISSUE + (F8 ? 128 * REG_CONVERT : 0);
    static constexpr int SWB        = D >= 64 ? 128 : D * 2;
    static constexpr int BOXC       = SWB / 2;
    static constexpr int NBOX       = D / BOXC;
    static constexpr int BOX_BYTES  = 128 * SWB;
    static constexpr int TILE_BYTES = 128 * D * 2;
    static constexpr int NSTAGE_K   = D == 128 ? 2 : 4;
    static constexpr int NSTAGE_V   = D == 128 ? (F8 ? 2 : 3) : 4;
    static constexpr int NRAW       = F8 ? (D == 128 ? 2 : 4) : 0;         // codes of a K or V stage, in turn
    static constexpr int RAW_BYTES  = 128 * D + 128;
    static constexpr int SMEM_BYTES = TILE_BYTES * (2 + NSTAGE_K + NSTAGE_V) + NRAW * RAW_BYTES + 1024;
    static_assert(SMEM_BYTES <= 232448, "more than an SM has");
};

// Byte `at` of a tile of rows of SWB bytes, as the TMA unit and the tensor cores have it under the swizzle of that width.
template <int SWB>
__device__ __forceinline__ uint32_t swizzled(uint32_t at) { return at ^ ((at >> 3) & (SWB == 128 ? 0x70u : SWB == 64 ? 0x30u : 0x10u)); }

// Weights are 2^(scale * s - offset) in one instruction, the offset a rounded scale * max: off by half its last bit, for all keys of a row alike, which cancels as long as fp16
// holds the weights: up to offsets of 2^27 (a factor of 2^4, beside 2^8 by which a maximum may outgrow the offset). Rows of Q that might go beyond that, with keys of
// 65504, have their scores scaled first; a difference to the maximum is exact then.
__device__ __forceinline__ uint32_t max_abs_f16x2(uint32_t a, uint32_t b)
{
    uint32_t r;
    asm("max.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <int D>
__device__ __forceinline__ bool scores_far(uint32_t top /* largest |q|, of either half */, float scale_log2e)
{
    const float2 q = __half22float2(*reinterpret_cast<const __half2*>(&top));
    return fmaxf(fabsf(q.x), fabsf(q.y)) * (65504.f * D) * scale_log2e > 134217728.f;
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 :: "r"(dst), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
template <int N> __device__ __forceinline__ void setmaxnreg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(N)); }
template <int N> __device__ __forceinline__ void setmaxnreg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(N)); }
__device__ __forceinline__ uint4 lds128(uint32_t at)
{
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void sts128(uint32_t at, const uint4& v)
{
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" :: "r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

template <int D, bool F8>
__global__ void __launch_bounds__(chunk_threads<F8>, 1)
paged_chunk_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const PagedArgs c, const PagedAttnArgs a)
{
    using C = ChunkCfg<D, F8>;
    constexpr uint32_t SWZ = swizzle_code(C::SWB);
    constexpr uint32_t IDESC_QK = idesc_f16_f32(WS_BM, WS_BN, 0, 0);
    constexpr uint32_t IDESC_PV = idesc_f16_f32(WS_BM, D, 0, 1);
    constexpr int NSK = C::NSTAGE_K, NSV = C::NSTAGE_V, NRAW = F8 ? C::NRAW : 1;
    constexpr bool POLY = D == 128;

    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* sQ = smem;
    uint8_t* sK = sQ + 2 * C::TILE_BYTES;
    uint8_t* sV = sK + NSK * C::TILE_BYTES;
    uint8_t* sRaw = sV + NSV * C::TILE_BYTES;

    __shared__ __align__(8) uint64_t q_full[2];
    __shared__ __align__(8) uint64_t k_full[NSK], k_empty[NSK], v_full[NSV], v_empty[NSV], v_raw[NSV];
    __shared__ __align__(8) uint64_t raw_full[NRAW], raw_empty[NRAW];
    __shared__ __align__(8) uint64_t s_full[2], p_full[2][2], o_done[2];
    __shared__ uint32_t tmem_base_smem;
    __shared__ int abort_word, poison;
    __shared__ PagedScratch scratch;
    __shared__ PagedPiece s_piece[2];                   // of this round and the next
    __shared__ int s_place[2];                          // where it goes if it is not the whole item; -1: no piece, the share is done

    const int tid  = threadIdx.x;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const int lane = tid & 31;

    if (tid == 0) {
        abort_word = 0;
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
    }
    if (warp == 9) tmem_alloc(&tmem_base_smem, 512);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, tmem_base_smem, 0);
    pdl_wait();
    pdl_trigger();

    // ---- this block's share: thread FINDER goes through it, a piece ahead of the others
    constexpr int FINDER = 352;
    PagedAt at{}, first;
    int left;
    const bool cut = a.parts.cut != nullptr;
    if (cut) {
        left = paged_part<C::THREADS>(c, a.w, blockIdx.x, gridDim.x, scratch, at, 53);
    } else {                                            // an item per block, of all sequences those of the last rows first: they are the longest
        const int group = c.H_kv * c.num_seqs, level = blockIdx.x / group, rest = blockIdx.x - level * group;
        at = PagedAt{rest % c.H_kv, rest / c.H_kv, a.w.max_tiles - 1 - level, 0};
        left = at.rt < paged_tiles(a.w, paged_seq(c, at.b)) ? INT_MAX : 0;
    }
    first = at;
    auto find_piece = [&](int slot) {
        s_place[slot] = -1;
        while (left > 0) {
            const PagedPiece p = paged_piece(c, a.w, at, left);
            const int other = at.h == first.h && at.b == first.b && at.rt == first.rt ? 0 : 1;
            if (!cut) left = 0;
            if (left > 0) paged_next(c, a.w, at);
            if (p.u_hi == p.u_lo) continue;
            s_piece[slot] = p;
            s_place[slot] = (int)blockIdx.x * 2 + other;
            return;
        }
    };
    if (tid == FINDER) {
        if (cut) {
            PagedCut here{};
            if (left > 0) here = PagedCut{at.h, at.b, at.rt, max(0, at.off - a.w.extra), paged_units(a.w, paged_seq(c, at.b), at.rt), 0, 0, 0};
            a.parts.cut[blockIdx.x] = here;
        } else if (at.rt == 0 && at.h == 0) {
            paged_seq<true>(c, at.b, 53);
        }
        find_piece(0);
    }

    struct Item { PagedPiece p; int r0, rows_q[2], nblk[2], nblk_max, jm; };
    auto fetch_item = [&](int round, Item& it) -> bool {
        if (tid == 0) {
            poison = 0;
            if (round > 0) {
                for (int q = 0; q < 2; q++) { mbar_inval(&q_full[q]); mbar_inval(&s_full[q]); mbar_inval(&p_full[q][0]); mbar_inval(&p_full[q][1]); mbar_inval(&o_done[q]); }
                for (int s = 0; s < NSK; s++) { mbar_inval(&k_full[s]); mbar_inval(&k_empty[s]); }
                for (int s = 0; s < NSV; s++) { mbar_inval(&v_full[s]); mbar_inval(&v_empty[s]); mbar_inval(&v_raw[s]); }
                for (int s = 0; s < NRAW; s++) { mbar_inval(&raw_full[s]); mbar_inval(&raw_empty[s]); }
            }
            for (int q = 0; q < 2; q++) {
                mbar_init(&q_full[q], WS_BM / 32);
                mbar_init(&s_full[q], 1);
                mbar_init(&p_full[q][0], WS_BM / 32);
                mbar_init(&p_full[q][1], WS_BM / 32);
                mbar_init(&o_done[q], 1);
            }
            for (int s = 0; s < NSK; s++) { mbar_init(&k_full[s], F8 ? 4 : 1); mbar_init(&k_empty[s], 1); }
            for (int s = 0; s < NSV; s++) { mbar_init(&v_full[s], F8 ? 4 : 2); mbar_init(&v_empty[s], 1); mbar_init(&v_raw[s], 1); }
            for (int s = 0; s < NRAW; s++) { mbar_init(&raw_full[s], 1); mbar_init(&raw_empty[s], 4); }
            mbar_fence_init();
        }
        __syncthreads();
        if (__shfl_sync(0xffffffffu, s_place[round & 1], 0) < 0 || abort_word != 0) return false;
        it.p = s_piece[round & 1];
        it.r0 = it.p.rt * 2 * WS_BM;
        const int rows = it.p.q.n * a.w.G - it.r0;
        #pragma unroll
        for (int q = 0; q < 2; q++) {
            it.rows_q[q] = max(0, min(WS_BM, rows - q * WS_BM));
            const int sees = it.rows_q[q] > 0 ? paged_visible(a.w, it.p.q, it.r0 + q * WS_BM + it.rows_q[q] - 1) : 0;
            it.nblk[q] = max(0, min((sees + WS_BN - 1) / WS_BN, it.p.u_hi) - it.p.u_lo);
        }
        it.nblk_max = max(it.nblk[0], it.nblk[1]);
        // Stages from jm on (of this piece) have keys that some row does not see, or that are not there.
        const int all_see = max(0, min(paged_visible(a.w, it.p.q, it.r0), it.p.q.kv));
        it.jm = max(0, all_see / WS_BN - it.p.u_lo);
        return true;
    };
    auto end_item = [&]() {
        __syncwarp();
        tc_fence_before_sync();
        __syncthreads();
        tc_fence_after_sync();
    };

    if (warp >= 8) {
        if (warp >= 12) setmaxnreg_dec<C::REG_CONVERT>(); else setmaxnreg_dec<C::REG_ISSUE>();
        for (int round = 0; ; round++) {
            Item it;
            if (!fetch_item(round, it)) break;
            const int nblk_max = it.nblk_max, u_lo = it.p.u_lo, kv = it.p.q.kv, jm = it.jm;
            const int* nblk = it.nblk;
            if (warp == 8) {
                // ---- producer: the lanes issue a stage's boxes side by side. Rows of a box: a page's, at most 128.
                const int box_rows = min(1 << c.page_shift, WS_BN), boxes = WS_BN / box_rows;
                const int box = lane % boxes, colb = lane / boxes;            // colb: up to NBOX column boxes (fp16)
                auto page_at = [&](int j) -> int {                            // c.num_pages: nothing there
                    const int key = (u_lo + j) * WS_BN + box * box_rows;
                    if (j >= nblk_max || key >= kv) return c.num_pages;
                    const int page = paged_page(c, it.p.b, key, 54);
                    return page < 0 ? c.num_pages : page;
                };
                int page = page_at(0);
                bool ok = true;
                for (int j = 0; j < nblk_max && ok; j++) {
                    const int slot = ((u_lo + j) * WS_BN + box * box_rows) & ((1 << c.page_shift) - 1);
                    const int row = (it.p.h << c.page_shift) + slot;
                    const int next = page_at(j + 1);
                    if constexpr (F8) {
                        #pragma unroll
                        for (int kv2 = 0; kv2 < 2; kv2++) {
                            const int n = 2 * j + kv2, s = n % NRAW, u = n / NRAW;
                            if (u > 0) ok = ok && __all_sync(0xffffffffu, mbar_wait(&raw_empty[s], (uint32_t)((u - 1) & 1), &abort_word, 61));
                            if (!ok) break;
                            const bool there = colb == 0 && page < c.num_pages;
                            const uint32_t exps = (uint32_t)__popc(__ballot_sync(0xffffffffu, there)) * (uint32_t)box_rows;
                            if (lane == 0) mbar_expect_tx(&raw_full[s], 128 * D + exps);
                            __syncwarp();
                            uint8_t* dst = sRaw + s * C::RAW_BYTES;
                            if (colb == 0) tma_load_3d(dst + box * box_rows * D, kv2 ? &tmV : &tmK, &raw_full[s], 0, row, page);
                            if (there) bulk_load(smem_u32(dst) + 128 * D + box * box_rows, (kv2 ? c.v_exp : c.k_exp) + ((long long)page * c.H_kv << c.page_shift) + row, (uint32_t)box_rows, &raw_full[s]);
                        }
                    } else {
                        const int sk = j % NSK, uk = j / NSK, sv = j % NSV, uv = j / NSV;
                        if (uk > 0) ok = __all_sync(0xffffffffu, mbar_wait(&k_empty[sk], (uint32_t)((uk - 1) & 1), &abort_word, 21));
                        if (!ok) break;
                        if (lane == 0) mbar_expect_tx(&k_full[sk], C::TILE_BYTES);
                        __syncwarp();
                        if (colb < C::NBOX) tma_load_3d(sK + sk * C::TILE_BYTES + colb * C::BOX_BYTES + box * box_rows * C::SWB, &tmK, &k_full[sk], colb * C::BOXC, row, page);
                        if (uv > 0) ok = __all_sync(0xffffffffu, mbar_wait(&v_empty[sv], (uint32_t)((uv - 1) & 1), &abort_word, 22));
                        if (!ok) break;
                        uint64_t* bar = j >= jm ? &v_raw[sv] : &v_full[sv];       // v_full: two arrivals, those of warps 10 and 11, or both here
                        if (lane == 0) mbar_expect_tx(bar, C::TILE_BYTES);
                        if (lane == 0 && j < jm) mbar_arrive(bar);
                        __syncwarp();
                        if (colb < C::NBOX) tma_load_3d(sV + sv * C::TILE_BYTES + colb * C::BOX_BYTES + box * box_rows * C::SWB, &tmV, bar, colb * C::BOXC, row, page);
                    }
                    page = next;
                }
            } else if (warp == 9) {
                // ---- MMA issuer, as in fa_fwd_ws_kernel
                const uint64_t dq0 = smem_desc(smem_u32(sQ), 16, 8 * C::SWB, SWZ);
                const uint64_t dk0 = smem_desc(smem_u32(sK), 16, 8 * C::SWB, SWZ);
                const uint64_t dv0 = smem_desc(smem_u32(sV), C::BOX_BYTES, 8 * C::SWB, SWZ);
                const uint32_t dq_lo = (uint32_t)dq0, dq_hi = (uint32_t)(dq0 >> 32);
                const uint32_t dk_lo = (uint32_t)dk0, dk_hi = (uint32_t)(dk0 >> 32);
                const uint32_t dv_lo = (uint32_t)dv0, dv_hi = (uint32_t)(dv0 >> 32);
                auto wait = [&](uint64_t* bar, int phase, int site) -> bool {
                    const bool done = __all_sync(0xffffffffu, mbar_wait(bar, (uint32_t)(phase & 1), &abort_word, site));
                    tc_fence_after_sync();
                    return done;
                };
                auto issue_qk = [&](int q, int slot) {
                    const uint32_t qa = dq_lo + (uint32_t)q * (C::TILE_BYTES >> 4);
                    const uint32_t ka = dk_lo + (uint32_t)slot * (C::TILE_BYTES >> 4);
                    const uint32_t tS = tmem_base + q * 128;
                    if (elect_one()) {
                        #pragma unroll
                        for (int ks = 0; ks < D / 16; ks++) {
                            const uint32_t off = ((uint32_t)((ks * 16) / C::BOXC) * C::BOX_BYTES + (uint32_t)((ks * 16) % C::BOXC) * 2u) >> 4;
                            tc_mma_ss_lh(tS, qa + off, dq_hi, ka + off, dk_hi, IDESC_QK, ks > 0 ? 1u : 0u);
                        }
                        tc_commit(&s_full[q]);
                    }
                };
                auto issue_pv = [&](int q, int slot, uint32_t acc0, int half, bool last) {
                    const uint32_t va = dv_lo + (uint32_t)slot * (C::TILE_BYTES >> 4);
                    const uint32_t tP = tmem_base + q * 128, tO = tmem_base + 256 + q * 128;
                    if (elect_one()) {
                        #pragma unroll
                        for (int ks = half * 4; ks < half * 4 + 4; ks++)
                            tc_mma_ts_lh(tO, tP + ks * 8, va + ((ks * 16 * C::SWB) >> 4), dv_hi, IDESC_PV, ks > 0 ? 1u : acc0);
                        if (last) tc_commit(&o_done[q]);
                    }
                };
                bool ok = true;
                if (nblk_max > 0) {
                    ok = wait(&k_full[0], 0, 23);
                    #pragma unroll
                    for (int q = 0; q < 2; q++) {
                        if (nblk[q] == 0 || !ok) continue;
                        ok = wait(&q_full[q], 0, 24);
                        if (ok) issue_qk(q, 0);
                    }
                }
                for (int j = 0; j < nblk_max && ok; j++) {
                    const int sv = j % NSV, sk = (j + 1) % NSK;
                    ok = wait(&v_full[sv], j / NSV, 25);
                    if (ok && j + 1 < nblk_max) ok = wait(&k_full[sk], (j + 1) / NSK, 27);
                    #pragma unroll
                    for (int q = 0; q < 2; q++) {
                        if (j >= nblk[q] || !ok) continue;
                        ok = wait(&p_full[q][0], j, 26);
                        if (!ok) continue;
                        issue_pv(q, sv, j > 0 ? 1u : 0u, 0, false);
                        ok = wait(&p_full[q][1], j, 29);
                        if (!ok) continue;
                        issue_pv(q, sv, 1u, 1, j + 1 == nblk[q]);
                        if (j + 1 < nblk[q]) issue_qk(q, sk);
                    }
                }
            } else {
                if (tid == FINDER) find_piece((round + 1) & 1);
                __syncwarp();
                bool bad_seen = false;
                auto clean = [&](uint4& x, int key) {            // what lies behind the last key is nobody's to see
                    uint32_t* w = &x.x;
                    uint32_t any = 0u;
                    #pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t bad = nonfinite_f16x2(w[i]);
                        any |= bad;
                        w[i] &= ~bad;
                    }
                    bad_seen |= any != 0u && key < kv;
                };
                bool ok = true;
                if constexpr (F8) {
                    // ---- warps 12 to 15: all codes to fp16. A thread has one 16-byte chunk of RPT rows behind one another. Every second thread (hi) takes its rows
                    // in the order 1, 0, 3, 2, ..., so that eight lanes' stores lie in eight different bank groups: shared memory is what the
                    // warps here, and the MMAs, contend for (Q K^T alone takes all of it for 512 cycles a tile).
                    constexpr int CH = D / 16, RPT = CH, HALF = RPT > 4 ? 4 : RPT;
                    const int ch = tid % CH, row0 = (tid & 127) / CH * RPT;
                    const int hi = CH == 8 ? ch >> 2 : CH == 4 ? (lane >> 2) & 1 : 0;
                    const uint32_t col = (uint32_t)(ch * 16 / C::BOXC) * C::BOX_BYTES, byte = (uint32_t)(ch * 16 % C::BOXC) * 2u;
                    // Rows of 128 bytes: row0 + (i ^ hi), chunk byte / 16 of it under the swizzle, as an exclusive or of what is known for i with the thread's own.
                    const uint32_t own = (uint32_t)row0 * 128u + (byte ^ (uint32_t)(hi * 0x90) ^ (uint32_t)(row0 & 4 ? 0x40 : 0));
                    auto place_of = [&](int i) { return RPT >= 4 ? own ^ (uint32_t)(i * 0x90) : swizzled<C::SWB>((uint32_t)(row0 + i) * C::SWB + byte); };
                    for (int n = 0; n < 2 * nblk_max && ok && warp >= 12; n++) {
                        const int j = n >> 1, isv = n & 1, s = n % NRAW;
                        const int NS = isv ? NSV : NSK, slot = j % NS, use = j / NS;
                        ok = __all_sync(0xffffffffu, (use == 0 || mbar_wait(isv ? &v_empty[slot] : &k_empty[slot], (uint32_t)((use - 1) & 1), &abort_word, 63)) &&
                                                     mbar_wait(&raw_full[s], (uint32_t)((n / NRAW) & 1), &abort_word, 62));
                        if (!ok) break;
                        const uint32_t raw = smem_u32(sRaw + s * C::RAW_BYTES);
                        const uint32_t dst = smem_u32((isv ? sV : sK) + slot * C::TILE_BYTES) + col;
                        #pragma unroll 1       // small: the softmax's code and this are more than the instruction caches hold (unrolled 115 us, so 86: 512 tokens x 32 heads, 8192 keys)
                        for (int i0 = 0; i0 < RPT; i0 += HALF) {
                            uint4 x[HALF];
                            uint32_t exps;
                            if constexpr (HALF == 4) asm volatile("ld.shared.b32 %0, [%1];" : "=r"(exps) : "r"(raw + 128 * D + row0 + i0) : "memory");
                            if constexpr (HALF == 2) asm volatile("{\n.reg .b16 x;\nld.shared.b16 x, [%1];\ncvt.u32.u16 %0, x;\n}\n" : "=r"(exps) : "r"(raw + 128 * D + row0) : "memory");
                            if constexpr (HALF == 1) asm volatile("ld.shared.u8 %0, [%1];" : "=r"(exps) : "r"(raw + 128 * D + row0) : "memory");
                            #pragma unroll
                            for (int i = 0; i < HALF; i++) x[i] = lds128(raw + ((row0 + (i0 + i ^ hi)) * CH + ch) * 16);
                            if (HALF == 4 && hi) exps = __byte_perm(exps, 0, 0x2301);
                            #pragma unroll
                            for (int i = 0; i < HALF; i++) {
                                const uint32_t e = exp_byte_f16x2((exps >> (8 * i)) & 0xffu);
                                uint4 lo, up;
                                e4m3x4_to_f16x4(x[i].x, lo.x, lo.y); e4m3x4_to_f16x4(x[i].y, lo.z, lo.w);
                                e4m3x4_to_f16x4(x[i].z, up.x, up.y); e4m3x4_to_f16x4(x[i].w, up.z, up.w);
                                lo = make_uint4(mul_f16x2(lo.x, e), mul_f16x2(lo.y, e), mul_f16x2(lo.z, e), mul_f16x2(lo.w, e));
                                up = make_uint4(mul_f16x2(up.x, e), mul_f16x2(up.y, e), mul_f16x2(up.z, e), mul_f16x2(up.w, e));
                                sts128(dst + place_of(i0 + i), lo);
                                sts128(dst + (place_of(i0 + i) ^ 16u), up);
                            }
                        }
                        if (isv && j >= jm) {
                            #pragma unroll 1
                            for (int i = 0; i < 2 * RPT; i++) {
                                const uint32_t at = dst + (place_of(i >> 1) ^ (i & 1 ? 16u : 0u));
                                uint4 x = lds128(at);
                                clean(x, (u_lo + j) * WS_BN + row0 + ((i >> 1) ^ hi));
                                sts128(at, x);
                            }
                            if (bad_seen) *(volatile int*)&poison = 1;
                        }
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) {
                            mbar_arrive(&raw_empty[s]);
                            mbar_arrive(isv ? &v_full[slot] : &k_full[slot]);
                        }
                    }
                } else {
                    // ---- warps 10 and 11: values that are not finite, where the mask needs it
                    const int t64 = tid - 320;
                    for (int j = jm; j < nblk_max && ok; j++) {
                        const int slot = j % NSV;
                        ok = __all_sync(0xffffffffu, mbar_wait(&v_raw[slot], (uint32_t)(((j - jm) / NSV) & 1), &abort_word, 64));
                        if (!ok) break;
                        const uint32_t v = smem_u32(sV + slot * C::TILE_BYTES);
                        #pragma unroll 4
                        for (int i = 0; i < C::TILE_BYTES / 16 / 64; i++) {
                            uint4 x = lds128(v + (i * 64 + t64) * 16);
                            clean(x, (u_lo + j) * WS_BN + (i * 64 + t64) % (C::BOX_BYTES / 16) / (C::SWB / 16));
                            sts128(v + (i * 64 + t64) * 16, x);
                        }
                        if (bad_seen) *(volatile int*)&poison = 1;
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&v_full[slot]);
                    }
                }
            }
            end_item();
        }
    } else {
        setmaxnreg_inc<C::REG_SOFTMAX>();
        for (int round = 0; ; round++) {
            Item it;
            if (!fetch_item(round, it)) break;
            const int q = warp >> 2;
            const int row = tid - q * WS_BM;
            const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
            const uint32_t tmem_S = tmem_base + q * 128 + lane_base;
            const uint32_t tmem_O = tmem_base + 256 + q * 128 + lane_base;
            const int my_nblk = q ? it.nblk[1] : it.nblk[0], u_lo = it.p.u_lo, jm = it.jm;
            const bool gives_back = (warp & 3) == 0 && lane == 0 && q == (it.nblk[1] > 0 ? 1 : 0);
            const bool valid = row < (q ? it.rows_q[1] : it.rows_q[0]);
            const int r = it.r0 + q * WS_BM + row, token = valid ? r / a.w.G : 0;
            const int sees = valid ? min(a.w.causal ? it.p.q.kv - it.p.q.n + token + 1 : it.p.q.kv, it.p.q.kv) : it.p.q.kv;
            const int head = it.p.h * a.w.G + (valid ? r - token * a.w.G : 0);

            // ---- the warp's 32 rows of Q into the tile, as many lanes to a row as it has chunks of 16 bytes
            bool far = false;
            if (my_nblk > 0) {
                const long long off = (long long)head * a.q_head + (long long)(it.p.q.row0 + token) * a.q_token;
                const uint32_t dst = smem_u32(sQ + q * C::TILE_BYTES);
                constexpr int CH = D / 8;
                uint4 x[CH];
                uint32_t top = 0u;
                #pragma unroll
                for (int i = 0; i < CH; i++) {
                    const int rr = (i * 32 + lane) / CH, ch = (i * 32 + lane) % CH;
                    const long long from = __shfl_sync(0xffffffffu, off, rr);
                    x[i] = (row & ~31) + rr < (q ? it.rows_q[1] : it.rows_q[0]) ? *reinterpret_cast<const uint4*>(a.Q + from + ch * 8) : make_uint4(0u, 0u, 0u, 0u);
                }
                #pragma unroll
                for (int i = 0; i < CH; i++) {
                    const int rr = (row & ~31) + (i * 32 + lane) / CH, ch = (i * 32 + lane) % CH;
                    sts128(dst + (uint32_t)(ch * 8 / C::BOXC) * C::BOX_BYTES + swizzled<C::SWB>((uint32_t)rr * C::SWB + (uint32_t)(ch * 8 % C::BOXC) * 2u), x[i]);
                    top = max_abs_f16x2(max_abs_f16x2(max_abs_f16x2(max_abs_f16x2(top, x[i].x), x[i].y), x[i].z), x[i].w);
                }
                far = __any_sync(0xffffffffu, scores_far<D>(top, a.scale_log2e));
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_full[q]);
            }

            const float scale = far ? 1.f : a.scale_log2e;              // of the scores as the loop has them
            const int slow_from = far ? 0 : jm;                         // stages that are masked or scaled
            float m_ref = kNegInfW, m_true = kNegInfW, l_run = 0.f;     // as in fa_fwd_ws_kernel
            bool ok = true;
            for (int j = 0; j < my_nblk; j++) {
                ok = __all_sync(0xffffffffu, mbar_wait(&s_full[q], (uint32_t)(j & 1), &abort_word, 31));
                if (!ok) break;
                tc_fence_after_sync();
                if (gives_back) {
                    mbar_arrive(&k_empty[j % NSK]);
                    if (j > 0) mbar_arrive(&v_empty[(j - 1) % NSV]);
                }

                uint32_t su[4][32];
                #pragma unroll
                for (int x = 0; x < 4; x++) tmem_ld32(tmem_S + x * 32, su[x]);
                tmem_wait_ld();

                if (j >= slow_from) {
                    if (far) {
                        #pragma unroll
                        for (int x = 0; x < 4; x++)
                            #pragma unroll
                            for (int i = 0; i < 32; i++) su[x][i] = __float_as_uint(__uint_as_float(su[x][i]) * a.scale_log2e);
                    }
                    const int lim = sees - (u_lo + j) * WS_BN;           // keys of the stage that the row sees
                    #pragma unroll
                    for (int x = 0; x < 4; x++)
                        #pragma unroll
                        for (int i = 0; i < 32; i++)
                            if (x * 32 + i >= lim) su[x][i] = 0xff800000u;
                }

                float mx0 = kNegInfW, mx1 = kNegInfW, mx2 = kNegInfW, mx3 = kNegInfW;
                #pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    mx0 = max3(mx0, __uint_as_float(su[0][i]), __uint_as_float(su[0][i + 1]));
                    mx1 = max3(mx1, __uint_as_float(su[1][i]), __uint_as_float(su[1][i + 1]));
                    mx2 = max3(mx2, __uint_as_float(su[2][i]), __uint_as_float(su[2][i + 1]));
                    mx3 = max3(mx3, __uint_as_float(su[3][i]), __uint_as_float(su[3][i + 1]));
                }
                const float mx = fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3));
                m_true = fmaxf(m_true, mx * scale);

                float alpha = 1.f;
                if (m_true - m_ref > a.rescale_above || m_ref == kNegInfW) {
                    const float m_new = m_true;
                    const float m_use = (m_new == kNegInfW) ? 0.f : m_new;
                    alpha = (m_ref == kNegInfW) ? 0.f : ex2(m_ref - m_use);
                    m_ref = m_new;
                }
                const float m_off = (m_ref == kNegInfW) ? 0.f : m_ref;

                const uint64_t scale2 = pack2(scale, scale), off2 = pack2(-m_off, -m_off);
                uint64_t psum2[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)};
                auto weights = [&](int x, uint32_t (&pk)[16]) {
                    #pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const uint64_t e2 = fma2(pack2(__uint_as_float(su[x][2 * i]), __uint_as_float(su[x][2 * i + 1])), scale2, off2);
                        float e0, e1;
                        if (POLY && i % 4 == 3) {
                            const uint64_t e = exp2_poly2(e2);
                            unpack2(e, e0, e1);
                            psum2[i & 1] = add2(psum2[i & 1], e);
                        } else {
                            unpack2(e2, e0, e1);
                            e0 = ex2(e0);
                            e1 = ex2(e1);
                            psum2[i & 1] = add2(psum2[i & 1], pack2(e0, e1));
                        }
                        pk[i] = pack_f16x2(e0, e1);
                    }
                };
                uint32_t pk[2][16];

                // PV(j-1) is complete when S(j) is (the tensor pipe runs in issue order). alpha is 0, which must not meet what is not
                // finite, only where nothing has been added yet (m_ref was -inf), and what was added then is 0 or NaN.
                if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
                    #pragma unroll
                    for (int x = 0; x < D / 16; x++) {
                        uint32_t o[16];
                        tmem_ld16(tmem_O + x * 16, o);
                        tmem_wait_ld();
                        #pragma unroll
                        for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                        tmem_st16(tmem_O + x * 16, o);
                    }
                }

                #pragma unroll
                for (int x = 0; x < 4; x++) {
                    weights(x, pk[x & 1]);
                    tmem_st16(tmem_S + x * 16, pk[x & 1]);
                    if (x == 1 || x == 3) {
                        tmem_wait_st();
                        tc_fence_before_sync();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&p_full[q][x >> 1]);
                    }
                }
                float s0, s1, s2, s3;
                unpack2(psum2[0], s0, s1);
                unpack2(psum2[1], s2, s3);
                l_run = l_run * alpha + ((s0 + s2) + (s1 + s3));
            }

            if (ok && my_nblk > 0) {
                ok = __all_sync(0xffffffffu, mbar_wait(&o_done[q], 0u, &abort_word, 32));
                tc_fence_after_sync();
            }

            // ---- epilogue (warps take it as a whole: the loads from tensor memory are collective)
            if (ok && (warp & 3) * 32 < (q ? it.rows_q[1] : it.rows_q[0])) {
                const bool whole = it.p.u_lo == 0 && it.p.u_hi == it.p.units;
                const bool none = sees <= 0;
                float mult = none ? 0.f : 1.f / l_run;
                if (!whole) mult = m_true == kNegInfW ? 1.f : ex2(m_ref - m_true);       // relative to the row's own maximum
                const long long place = s_place[round & 1];
                if (!whole && valid) a.parts.ml[place * (2 * WS_BM) + q * WS_BM + row] = make_float2(m_true, l_run * mult);
                const bool patch = *(volatile int*)&poison != 0;
                const int k0 = (u_lo + jm) * WS_BN, k1 = min(sees, it.p.u_hi * WS_BN);
                #pragma unroll 1
                for (int x = 0; x < D / 16; x++) {
                    uint32_t o[16];
                    if (my_nblk > 0) {
                        tmem_ld16(tmem_O + x * 16, o);
                        tmem_wait_ld();
                    } else {
                        #pragma unroll
                        for (int i = 0; i < 16; i++) o[i] = 0u;
                    }
                    if (patch && valid) {
                        // Rare: the values that warps 10 and 11 left out, for the keys that this row sees.
                        for (int key = k0; key < k1; key++) {
                            const int page = paged_page(c, it.p.b, key, 54);
                            if (page < 0) continue;
                            const long long at_row = (long long)(it.p.h << c.page_shift) + (key & ((1 << c.page_shift) - 1));
                            const uint8_t* src = c.v + (long long)page * c.page_stride + at_row * D * (F8 ? 1 : 2);
                            #pragma unroll
                            for (int i = 0; i < 16; i++) {
                                float v;
                                if constexpr (F8) v = (src[x * 16 + i] & 0x7f) == 0x7f ? NAN : 0.f;
                                else v = __half2float(reinterpret_cast<const __half*>(src)[x * 16 + i]);
                                if (!isfinite(v)) o[i] = __float_as_uint(__uint_as_float(o[i]) + v);
                            }
                        }
                    }
                    if (!valid) continue;
                    if (whole) {
                        uint4 w[2];
                        uint32_t* p = &w[0].x;
                        #pragma unroll
                        for (int i = 0; i < 8; i++) p[i] = none ? 0u : pack_f16x2(__uint_as_float(o[2 * i]) * mult, __uint_as_float(o[2 * i + 1]) * mult);
                        uint4* dst = reinterpret_cast<uint4*>(a.O + (long long)(it.p.q.row0 + token) * a.o_token + (long long)head * D + x * 16);
                        dst[0] = w[0];
                        dst[1] = w[1];
                    } else {
                        float4* dst = a.parts.o + (place * (D / 4) + x * 4) * (2 * WS_BM) + q * WS_BM + row;
                        #pragma unroll
                        for (int i = 0; i < 4; i++)
                            dst[i * 2 * WS_BM] = make_float4(__uint_as_float(o[4 * i]) * mult, __uint_as_float(o[4 * i + 1]) * mult,
                                                 __uint_as_float(o[4 * i + 2]) * mult, __uint_as_float(o[4 * i + 3]) * mult);
                    }
                }
            }
            end_item();
        }
    }
    __syncthreads();

    // ---- teardown
    if (abort_word != 0) {
        for (int i = 0; i < 64; i++) __nanosleep(100000);
        if (tid == 0 && c.status != nullptr && atomicCAS(c.status, 0, (int)KS_WAIT_TIMEOUT) == 0) {
            c.status[1] = blockIdx.x;
            c.status[2] = abort_word;
        }
        __syncthreads();
    }
    if (warp == 9) tmem_dealloc(tmem_base, 512);
}
