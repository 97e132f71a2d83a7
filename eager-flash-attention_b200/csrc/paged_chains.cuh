// Attention of long chunks over a paged cache of fp16 heads of 16, 32 and 64, where the exponentials are the work: the four chains of fa_fwd_chains_kernel (two to
// each 128-row tile, one for the lower and one for the upper 64 keys of every 128-key stage; the reasons stand there), with the pages, rows, masks and shares
// of paged_chunk_kernel (the reasons stand there). Included by fa_fwd_ws_sm100.cu behind both.
//
// 768 threads: warps 0-15 softmax of chain 0 to 3, 16-19 the chains' issuers, 20 producer, 21 owner of the tensor memory and, with one lane, finder of the pieces,
// 22 and 23 put zeros for values that are not finite where the mask needs it.
//
// What bounds it: the special-function unit (63 % busy in ncu at 2048 tokens x 16 heads over 8192 keys, tensor pipe 35 %), and per item about 7 us besides its units of
// 1.45 us (256 rows x 128 keys; two chains of 128 keys 1.63): us, two chains / this: 16 heads of 64, 4096 tokens 59.0 / 56.7, 8192 196 / 181; 64 rows, 16 x 16000 keys
// 159 / 129 (since then 1 to 2 % for scores far from zero and slots behind the last key). Prompts of 1024 tokens and less are the same or 5 % slower, and mostly go to the small tiles.
#pragma once

template <int D>
struct PagedChainCfg {
    static constexpr int THREADS    = 768;
    static constexpr int REG_SOFTMAX = 104, REG_ISSUE = 40, REG_REST = 24;
    static constexpr int REGS       = 512 * REG_SOFTMAX + 128 * REG_ISSUE + 128 * REG_REST;
    static constexpr int SWB        = D >= 64 ? 128 : D * 2;
    static constexpr int TILE_BYTES = 128 * D * 2;
    static constexpr int NS         = 4;                          // slots of K, and of V
    static constexpr int SMEM_BYTES = TILE_BYTES * (2 + 2 * NS) + 1024;
    static_assert(D <= 64, "one column box to a row");
};

template <int D>
__global__ void __launch_bounds__(768, 1)
paged_chains_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const PagedArgs c, const PagedAttnArgs a)
{
    using C = PagedChainCfg<D>;
    constexpr int NS = C::NS;
    constexpr uint32_t SWZ = swizzle_code(C::SWB);
    constexpr uint32_t IDESC_QK = idesc_f16_f32(WS_BM, 64, 0, 0);
    constexpr uint32_t IDESC_PV = idesc_f16_f32(WS_BM, D, 0, 1);
    constexpr bool LATE = D == 64;                                // where O is rescaled, as in fa_fwd_chains_kernel

    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* sQ = smem;
    uint8_t* sK = sQ + 2 * C::TILE_BYTES;
    uint8_t* sV = sK + NS * C::TILE_BYTES;

    __shared__ __align__(8) uint64_t q_full[2];
    __shared__ __align__(8) uint64_t k_full[NS], k_empty[NS], v_full[NS], v_empty[NS], v_raw[NS];
    __shared__ __align__(8) uint64_t s_full[4], p_full[4], o_done[4];
    __shared__ float ends[4][2][WS_BM];                           // offset and sum of every chain's rows
    __shared__ uint32_t tmem_base_smem;
    __shared__ int abort_word, poison, far_word;
    __shared__ PagedScratch scratch;
    __shared__ PagedPiece s_piece[2];
    __shared__ int s_place[2];

    const int tid  = threadIdx.x;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const int lane = tid & 31;

    if (tid == 0) {
        abort_word = 0;
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
    }
    if (warp == 21) tmem_alloc(&tmem_base_smem, 512);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, tmem_base_smem, 0);
    pdl_wait();
    pdl_trigger();

    // ---- this block's share, as in paged_chunk_kernel
    constexpr int FINDER = 21 * 32;
    PagedAt at{}, first;
    int left;
    const bool cut = a.parts.cut != nullptr;
    if (cut) {
        left = paged_part<C::THREADS>(c, a.w, blockIdx.x, gridDim.x, scratch, at, 53);
    } else {
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

    auto fetch_item = [&](int round) -> bool {
        if (tid == 0) {
            poison = 0;
            far_word = 0;
            if (round > 0) {
                for (int t = 0; t < 2; t++) mbar_inval(&q_full[t]);
                for (int s = 0; s < NS; s++) { mbar_inval(&k_full[s]); mbar_inval(&k_empty[s]); mbar_inval(&v_full[s]); mbar_inval(&v_empty[s]); mbar_inval(&v_raw[s]); }
                for (int x = 0; x < 4; x++) { mbar_inval(&s_full[x]); mbar_inval(&p_full[x]); mbar_inval(&o_done[x]); }
            }
            for (int t = 0; t < 2; t++) mbar_init(&q_full[t], 8);
            for (int s = 0; s < NS; s++) { mbar_init(&k_full[s], 1); mbar_init(&k_empty[s], 4); mbar_init(&v_full[s], 2); mbar_init(&v_empty[s], 4); mbar_init(&v_raw[s], 1); }
            for (int x = 0; x < 4; x++) { mbar_init(&s_full[x], 1); mbar_init(&p_full[x], WS_BM / 32); mbar_init(&o_done[x], 1); }
            mbar_fence_init();
        }
        __syncthreads();
        return __shfl_sync(0xffffffffu, s_place[round & 1], 0) >= 0 && abort_word == 0;
    };
    auto end_item = [&]() {
        __syncwarp();
        tc_fence_before_sync();
        __syncthreads();
        tc_fence_after_sync();
    };
    // Of the piece of this round: rows of a tile, and its 64-key blocks; block b is half b & 1 of stage b / 2 and belongs to chain b % 2 of the tile.
    auto rows_of = [&](const PagedPiece& p, int t) { return max(0, min(WS_BM, p.q.n * a.w.G - p.rt * 2 * WS_BM - t * WS_BM)); };
    auto blocks_of = [&](const PagedPiece& p, int t) {
        const int rows = rows_of(p, t);
        const int end = rows > 0 ? min(paged_visible(a.w, p.q, p.rt * 2 * WS_BM + t * WS_BM + rows - 1), p.u_hi * WS_BN) - p.u_lo * WS_BN : 0;
        return end > 0 ? (end + 63) >> 6 : 0;
    };
    // Stages from here on have keys that some row does not see, or that are not there.
    auto masked_from = [&](const PagedPiece& p) { return max(0, max(0, min(paged_visible(a.w, p.q, p.rt * 2 * WS_BM), p.q.kv)) / WS_BN - p.u_lo); };

    if (warp >= 20) {
        setmaxnreg_dec<C::REG_REST>();
        for (int round = 0; fetch_item(round); round++) {
            const PagedPiece& p = s_piece[round & 1];
            const int n0 = blocks_of(p, 0), n1 = blocks_of(p, 1), stages = (max(n0, n1) + 1) >> 1, jm = masked_from(p);
            if (warp == 20) {
                // ---- producer: the lanes issue a stage's boxes, a page's rows each, side by side
                const int box_rows = min(1 << c.page_shift, WS_BN), key0 = p.u_lo * WS_BN + lane * box_rows, b = p.b, kv = p.q.kv, h = p.h;
                const bool mine = lane < WS_BN / box_rows;
                auto page_at = [&](int j) -> int {                            // c.num_pages: nothing there
                    const int key = key0 + j * WS_BN;
                    if (!mine || j >= stages || key >= kv) return c.num_pages;
                    const int page = paged_page(c, b, key, 54);
                    return page < 0 ? c.num_pages : page;
                };
                int page = page_at(0);
                bool ok = true;
                for (int j = 0; j < stages; j++) {
                    const int s = j % NS, u = j / NS, row = (h << c.page_shift) + ((key0 + j * WS_BN) & ((1 << c.page_shift) - 1));
                    const int next = page_at(j + 1);
                    if (u > 0) ok = __all_sync(0xffffffffu, mbar_wait(&k_empty[s], (uint32_t)((u - 1) & 1), &abort_word, 21));
                    if (!ok) break;
                    if (lane == 0) mbar_expect_tx(&k_full[s], C::TILE_BYTES);
                    __syncwarp();
                    if (mine) tma_load_3d(sK + s * C::TILE_BYTES + lane * box_rows * C::SWB, &tmK, &k_full[s], 0, row, page);
                    if (u > 0) ok = __all_sync(0xffffffffu, mbar_wait(&v_empty[s], (uint32_t)((u - 1) & 1), &abort_word, 22));
                    if (!ok) break;
                    uint64_t* bar = j >= jm ? &v_raw[s] : &v_full[s];         // v_full: two arrivals, those of warps 22 and 23, or both here
                    if (lane == 0) {
                        mbar_expect_tx(bar, C::TILE_BYTES);
                        if (j < jm) mbar_arrive(bar);
                        for (int users = max(0, min(2, n0 - 2 * j)) + max(0, min(2, n1 - 2 * j)); users < 4; users++) {       // for chains that end before this stage
                            mbar_arrive(&k_empty[s]);
                            mbar_arrive(&v_empty[s]);
                        }
                    }
                    __syncwarp();
                    if (mine) tma_load_3d(sV + s * C::TILE_BYTES + lane * box_rows * C::SWB, &tmV, bar, 0, row, page);
                    page = next;
                }
            } else if (warp == 21) {
                if (tid == FINDER) find_piece((round + 1) & 1);
            } else {
                // ---- warps 22 and 23
                bool bad_seen = false;
                for (int j = jm; j < stages; j++) {
                    const int s = j % NS;
                    if (!__all_sync(0xffffffffu, mbar_wait(&v_raw[s], (uint32_t)(((j - jm) / NS) & 1), &abort_word, 64))) break;
                    const uint32_t v = smem_u32(sV + s * C::TILE_BYTES) + (tid & 63) * 16;
                    const int there = p.q.kv - (p.u_lo + j) * WS_BN;
                    #pragma unroll 2
                    for (int i = 0; i < C::TILE_BYTES / 16 / 64; i++) {
                        uint4 x = lds128(v + i * 1024);
                        uint32_t* w = &x.x;
                        uint32_t any = 0u;
                        #pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const uint32_t bad = nonfinite_f16x2(w[k]);
                            any |= bad;
                            w[k] &= ~bad;
                        }
                        bad_seen |= any != 0u && (i * 64 + (tid & 63)) / (C::SWB / 16) < there;      // what lies behind the last key is nobody's to see
                        sts128(v + i * 1024, x);
                    }
                    if (bad_seen) *(volatile int*)&poison = 1;
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&v_full[s]);
                }
            }
            end_item();
        }
    } else if (warp >= 16) {
        setmaxnreg_dec<C::REG_ISSUE>();
        for (int round = 0; fetch_item(round); round++) {
            // ---- MMA issuers, one to a chain, as in fa_fwd_chains_kernel
            const int ch = warp - 16, tile = ch >> 1, way = ch & 1;
            const uint64_t dq = smem_desc(smem_u32(sQ), 16, 8 * C::SWB, SWZ);
            const uint64_t dk = smem_desc(smem_u32(sK), 16, 8 * C::SWB, SWZ);
            const uint64_t dv = smem_desc(smem_u32(sV), 128 * C::SWB, 8 * C::SWB, SWZ);
            constexpr uint32_t HALF = (64 * C::SWB) >> 4;             // 64 keys further
            const uint32_t dq_lo = (uint32_t)dq + tile * (C::TILE_BYTES >> 4), dq_hi = (uint32_t)(dq >> 32);
            const uint32_t dk_lo = (uint32_t)dk + way * HALF, dk_hi = (uint32_t)(dk >> 32);
            const uint32_t dv_lo = (uint32_t)dv + way * HALF, dv_hi = (uint32_t)(dv >> 32);
            const uint32_t tS = tmem_base + ch * 64, tO = tmem_base + 256 + ch * 64;
            auto wait = [&](uint64_t* bar, int phase, int site) -> bool {
                return __all_sync(0xffffffffu, mbar_wait(bar, (uint32_t)(phase & 1), &abort_word, site));
            };
            auto issue_qk = [&](int slot) {
                #pragma unroll
                for (int ks = 0; ks < D / 16; ks++)
                    tc_mma_ss_lh(tS, dq_lo + ks * 2, dq_hi, dk_lo + slot * (C::TILE_BYTES >> 4) + ks * 2, dk_hi, IDESC_QK, ks > 0 ? 1u : 0u);
                tc_commit(&s_full[ch]);
            };
            const int n = (blocks_of(s_piece[round & 1], tile) - way + 1) >> 1;
            bool ok = n > 0 && wait(&q_full[tile], 0, 24);
            if (ok) {
                ok = wait(&k_full[0], 0, 27);
                tc_fence_after_sync();
                if (ok && elect_one()) issue_qk(0);
                __syncwarp();
            }
            for (int i = 0; i < n && ok; i++) {
                const int s = i % NS, next = (i + 1) % NS;
                const bool more = i + 1 < n;
                ok = wait(&s_full[ch], i, 22);                        // so QK(i) and PV(i-1) are complete
                if (!ok) break;
                if (lane == 0) {
                    mbar_arrive(&k_empty[s]);
                    if (i > 0) mbar_arrive(&v_empty[(i - 1) % NS]);
                }
                __syncwarp();
                ok = wait(&v_full[s], i / NS, 25) && (!more || wait(&k_full[next], (i + 1) / NS, 28)) && wait(&p_full[ch], i, 26);
                tc_fence_after_sync();
                if (!ok) break;
                if (elect_one()) {
                    #pragma unroll
                    for (int ks = 0; ks < 4; ks++)
                        tc_mma_ts_lh(tO, tS + ks * 8, dv_lo + s * (C::TILE_BYTES >> 4) + ((ks * 16 * C::SWB) >> 4), dv_hi, IDESC_PV, ks > 0 || i > 0 ? 1u : 0u);
                    if (more) issue_qk(next); else tc_commit(&o_done[ch]);
                }
                __syncwarp();
            }
            end_item();
        }
    } else {
        setmaxnreg_inc<C::REG_SOFTMAX>();
        for (int round = 0; fetch_item(round); round++) {
            // =====================================================================================
            // Softmax: chain ch = warp / 4, row = thread index within the warpgroup
            // =====================================================================================
            const int ch = warp >> 2, tile = ch >> 1, way = ch & 1;
            const int row = tid & (WS_BM - 1);
            const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
            const uint32_t tmem_S = tmem_base + ch * 64 + lane_base;
            const uint32_t tmem_O = tmem_base + 256 + ch * 64 + lane_base;
            const int blocks = blocks_of(s_piece[round & 1], tile), n = (blocks - way + 1) >> 1;
            const int jm = masked_from(s_piece[round & 1]);
            // Little is kept in registers through the loop: what the end needs is found again.
            auto sees_below = [&](const PagedPiece& p) {           // keys that this thread's row sees; with no such row all that there are
                return row < rows_of(p, tile) ? min(paged_visible(a.w, p.q, p.rt * 2 * WS_BM + tile * WS_BM + row), p.q.kv) : p.q.kv;
            };
            const int lim0 = sees_below(s_piece[round & 1]) - (s_piece[round & 1].u_lo * 2 + way) * 64;
            {
                const PagedPiece& p = s_piece[round & 1];
                const int rows = rows_of(p, tile);
                const bool valid = row < rows;
                const int r = p.rt * 2 * WS_BM + tile * WS_BM + row;
                // ---- half of the warp's 32 rows of Q into the tile (the other chain's warp takes the rest), as many lanes to a row as it has chunks of 16 bytes
                if (blocks > 0) {
                    const int token = valid ? r / a.w.G : 0;
                    const long long off = (long long)(p.h * a.w.G + (valid ? r - token * a.w.G : 0)) * a.q_head + (long long)(p.q.row0 + token) * a.q_token;
                    const uint32_t dst = smem_u32(sQ + tile * C::TILE_BYTES);
                    constexpr int CH = D / 8, STEPS = CH / 2 > 0 ? CH / 2 : 1;
                    uint4 x[STEPS];
                    uint32_t top = 0u;
                    #pragma unroll
                    for (int i = 0; i < STEPS; i++) {
                        const int rr = way * 16 + (i * 32 + lane) / CH, k = (i * 32 + lane) % CH;
                        const long long from = __shfl_sync(0xffffffffu, off, rr);
                        x[i] = (row & ~31) + rr < rows ? *reinterpret_cast<const uint4*>(a.Q + from + k * 8) : make_uint4(0u, 0u, 0u, 0u);
                    }
                    #pragma unroll
                    for (int i = 0; i < STEPS; i++) {
                        const int rr = (row & ~31) + way * 16 + (i * 32 + lane) / CH, k = (i * 32 + lane) % CH;
                        sts128(dst + swizzled<C::SWB>((uint32_t)rr * C::SWB + (uint32_t)k * 16u), x[i]);
                        top = max_abs_f16x2(max_abs_f16x2(max_abs_f16x2(max_abs_f16x2(top, x[i].x), x[i].y), x[i].z), x[i].w);
                    }
                    if (scores_far<D>(top, a.scale_log2e)) *(volatile int*)&far_word = 1;      // for the other chain's warps too
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&q_full[tile]);
                }
            }

            bool ok = n == 0 || __all_sync(0xffffffffu, mbar_wait(&q_full[tile], 0u, &abort_word, 33));
            const bool far = __shfl_sync(0xffffffffu, *(volatile int*)&far_word, 0) != 0;
            const float scale = far ? 1.f : a.scale_log2e;            // of the scores as the loop has them
            const int slow_from = far ? 0 : jm;                       // stages that are masked or scaled
            float m_ref = kNegInfW;     // exponent offset in use (a past row maximum), scaled by scale*log2(e)
            float l_run = 0.f;          // running denominator relative to m_ref
            for (int i = 0; i < n && ok; i++) {
                ok = __all_sync(0xffffffffu, mbar_wait(&s_full[ch], (uint32_t)(i & 1), &abort_word, 31));
                if (!ok) break;
                tc_fence_after_sync();
                uint32_t su[2][32];
                tmem_ld32(tmem_S, su[0]);
                tmem_ld32(tmem_S + 32, su[1]);
                tmem_wait_ld();

                if (i >= slow_from) {
                    if (far) {
                        #pragma unroll
                        for (int x = 0; x < 2; x++)
                            #pragma unroll
                            for (int k = 0; k < 32; k++) su[x][k] = __float_as_uint(__uint_as_float(su[x][k]) * a.scale_log2e);
                    }
                    const int lim = lim0 - i * WS_BN;
                    #pragma unroll
                    for (int x = 0; x < 2; x++)
                        #pragma unroll
                        for (int k = 0; k < 32; k++)
                            if (x * 32 + k >= lim) su[x][k] = 0xff800000u;
                }

                float mx0 = kNegInfW, mx1 = kNegInfW, mx2 = kNegInfW, mx3 = kNegInfW;
                #pragma unroll
                for (int k = 0; k < 16; k += 2) {
                    mx0 = max3(mx0, __uint_as_float(su[0][k]), __uint_as_float(su[0][k + 1]));
                    mx1 = max3(mx1, __uint_as_float(su[0][16 + k]), __uint_as_float(su[0][17 + k]));
                    mx2 = max3(mx2, __uint_as_float(su[1][k]), __uint_as_float(su[1][k + 1]));
                    mx3 = max3(mx3, __uint_as_float(su[1][16 + k]), __uint_as_float(su[1][17 + k]));
                }
                const float mx = fmaxf(max3(mx0, mx1, mx2), mx3) * scale;

                // Move the exponent offset only when the maximum grew by more than the threshold.
                float alpha = 1.f;
                if (mx > m_ref + a.rescale_above) {                   // also the first finite one
                    alpha = ex2(m_ref - mx);
                    m_ref = mx;
                }
                const float m_off = (m_ref == kNegInfW) ? 0.f : m_ref;
                const uint64_t scale2 = pack2(scale, scale), off2 = pack2(-m_off, -m_off);
                uint64_t psum2[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)};
                // Complete with S(i): PV(i-1), so O may be rescaled and P take the place of S.
                auto rescale = [&]() {
                    if (i == 0 || !__any_sync(0xffffffffu, alpha != 1.f)) return;
                    constexpr int PART = D < 32 ? D : 32;
                    #pragma unroll 1
                    for (int x = 0; x < D; x += PART) {
                        uint32_t o[PART];
                        if constexpr (PART == 32) tmem_ld32(tmem_O + x, o); else tmem_ld16(tmem_O + x, o);
                        tmem_wait_ld();
                        #pragma unroll
                        for (int k = 0; k < PART; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
                        if constexpr (PART == 32) tmem_st32(tmem_O + x, o); else tmem_st16(tmem_O + x, o);
                    }
                };
                if constexpr (!LATE) rescale();
                #pragma unroll
                for (int x = 0; x < 2; x++) {
                    uint32_t pk[16];
                    #pragma unroll
                    for (int k = 0; k < 16; k++) {
                        const uint64_t e = fma2(pack2(__uint_as_float(su[x][2 * k]), __uint_as_float(su[x][2 * k + 1])), scale2, off2);
                        float p0, p1;
                        if (k % 8 == 7) {
                            unpack2(exp2_poly2(e), p0, p1);
                        } else {
                            unpack2(e, p0, p1);
                            p0 = ex2(p0);
                            p1 = ex2(p1);
                        }
                        psum2[k & 1] = add2(psum2[k & 1], pack2(p0, p1));
                        pk[k] = pack_f16x2(p0, p1);
                    }
                    if constexpr (LATE) { if (x == 0) rescale(); }
                    tmem_st16(tmem_S + x * 16, pk);
                }
                tmem_wait_st();
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[ch]);
                float s0, s1, s2, s3;
                unpack2(psum2[0], s0, s1);
                unpack2(psum2[1], s2, s3);
                l_run = l_run * alpha + ((s0 + s2) + (s1 + s3));
            }
            if (ok && n > 0) {
                ok = __all_sync(0xffffffffu, mbar_wait(&o_done[ch], 0u, &abort_word, 32));
                tc_fence_after_sync();
            }

            // ---- the chains of a tile learn each other's offset and sum; each then merges and stores its share of the columns
            ends[ch][0][row] = m_ref; ends[ch][1][row] = l_run;
            tc_fence_before_sync();
            asm volatile("bar.sync %0, 256;" :: "r"(1 + tile) : "memory");
            tc_fence_after_sync();
            ok = __all_sync(0xffffffffu, ok && *(volatile int*)&abort_word == 0);
            float w[2];
            {
                const float m0 = ends[tile * 2][0][row], m1 = ends[tile * 2 + 1][0][row];
                m_ref = fmaxf(m0, m1);
                w[0] = m0 == m_ref ? 1.f : ex2(m0 - m_ref);
                w[1] = m1 == m_ref ? 1.f : ex2(m1 - m_ref);
                l_run = w[0] * ends[tile * 2][1][row] + w[1] * ends[tile * 2 + 1][1][row];
            }
            constexpr int PER = D / 2 < 16 ? 16 : D / 2;              // columns; of 16 one chain has all
            const int c_lo = way * PER;

            if (ok && (warp & 3) * 32 < rows_of(s_piece[round & 1], tile)) {
                const PagedPiece& p = s_piece[round & 1];
                const int sees = sees_below(p), u_lo = p.u_lo;
                const bool whole = u_lo == 0 && p.u_hi == p.units, valid = row < rows_of(p, tile), none = sees <= 0;
                const int r = p.rt * 2 * WS_BM + tile * WS_BM + row, token = valid ? r / a.w.G : 0;
                const float mult = !whole ? 1.f : none ? 0.f : 1.f / l_run;
                const long long place = s_place[round & 1];
                if (!whole && valid && way == 0) a.parts.ml[place * (2 * WS_BM) + tile * WS_BM + row] = make_float2(m_ref, l_run);
                const bool patch = *(volatile int*)&poison != 0;
                if (c_lo < D) {
                    #pragma unroll 1
                    for (int x = c_lo; x < c_lo + PER; x += 16) {
                        uint32_t o[16];
                        #pragma unroll
                        for (int k = 0; k < 16; k++) o[k] = 0u;
                        #pragma unroll
                        for (int k = 0; k < 2; k++) {
                            if (k >= blocks) break;                   // that chain has not run
                            uint32_t part[16];
                            tmem_ld16(tmem_base + 256 + (tile * 2 + k) * 64 + lane_base + x, part);
                            tmem_wait_ld();
                            #pragma unroll
                            for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) + __uint_as_float(part[e]) * w[k]);
                        }
                        if (!valid) continue;
                        if (patch) {
                            // Rare: the values that warps 22 and 23 left out, for the keys that this row sees.
                            for (int key = (u_lo + jm) * WS_BN; key < min(sees, p.u_hi * WS_BN); key++) {
                                const int page = paged_page(c, p.b, key, 54);
                                if (page < 0) continue;
                                const long long at_row = (long long)(p.h << c.page_shift) + (key & ((1 << c.page_shift) - 1));
                                const __half* src = reinterpret_cast<const __half*>(c.v + (long long)page * c.page_stride) + at_row * D + x;
                                #pragma unroll
                                for (int k = 0; k < 16; k++) {
                                    const float v = __half2float(src[k]);
                                    if (!isfinite(v)) o[k] = __float_as_uint(__uint_as_float(o[k]) + v);
                                }
                            }
                        }
                        if (whole) {
                            uint4 v[2];
                            uint32_t* d = &v[0].x;
                            #pragma unroll
                            for (int k = 0; k < 8; k++) d[k] = none ? 0u : pack_f16x2(__uint_as_float(o[2 * k]) * mult, __uint_as_float(o[2 * k + 1]) * mult);
                            uint4* dst = reinterpret_cast<uint4*>(a.O + (long long)(p.q.row0 + token) * a.o_token + (long long)(p.h * a.w.G + r - token * a.w.G) * D + x);
                            dst[0] = v[0];
                            dst[1] = v[1];
                        } else {
                            float4* dst = a.parts.o + (place * (D / 4) + x / 4) * (2 * WS_BM) + tile * WS_BM + row;
                            #pragma unroll
                            for (int k = 0; k < 4; k++)
                                dst[k * 2 * WS_BM] = make_float4(__uint_as_float(o[4 * k]), __uint_as_float(o[4 * k + 1]), __uint_as_float(o[4 * k + 2]), __uint_as_float(o[4 * k + 3]));
                        }
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
    if (warp == 21) tmem_dealloc(tmem_base, 512);
}
