// The paged key/value cache: rows of keys and values into pages and out of them, the checks of its arguments, and which kernel an attention
// over it takes. fp16, or e4m3 with an exponent per row (token and head): of a row x with largest finite magnitude `top`
//     e = max(-24, smallest e with top <= 448 * 2^e),   code = x * 2^-e on the e4m3 grid, ties to even,   value = code * 2^e.
// A power of two costs no accuracy (a code has its four significant bits wherever it stands) and buys exactness: every value is an fp16, in
// the scores the exponents multiply fp32 numbers, and one rounding is all that the cache adds. With e = 8 codes end at 240: 256 * 2^8 is no fp16.
#include "paged_attention.h"
#include "paged_kernels.cuh"

#include <cuda_fp8.h>

#include <algorithm>
#include <climits>
#include <cmath>

namespace efa {

namespace {

constexpr int PC_THREADS = 256;
// Heads that a thread moves at a time: what it has in flight, against the blocks that there are. us with 1 / 2 / 4 (8): fp16, 5822 tokens x 32 heads of
// 128 in 31.9 / 32.2 / 32.2 (33.3), 73472 keys x 16 heads of 64 out 93.8 / 94.3 / 96.0 (98.4); 8 bits, 12225 tokens x 8 heads of 128 in and out 34.1 / 30.3 / 31.0 (39.4),
// 100451 keys x 8 of 128 out 113.9 / 104.3 / 101.8 (103.7).
template <bool F8, bool READ> constexpr int PC_HEADS = !F8 ? 1 : READ ? 4 : 2;

struct PagedRows {
    __half* k;
    __half* v;
    long long head, token;           // strides in elements
};

// The sequence that a row belongs to: the last b with q_start[b] <= row. -1: none.
__device__ __forceinline__ int sequence_of(const PagedArgs& c, int row)
{
    int lo = 0, hi = c.num_seqs;                           // q_start[lo] <= row < q_start[hi], if anywhere
    if (row < c.q_start[0] || row >= c.q_start[hi]) return -1;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (c.q_start[mid] <= row) lo = mid; else hi = mid;
    }
    return lo;
}

// The exponent of a row whose largest magnitude has the fp16 bits `top` (finite).
__device__ __forceinline__ int exponent_of(uint32_t top)
{
    const uint32_t bits = __float_as_uint(__half2float(__ushort_as_half((unsigned short)top)));
    return max(-24, (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0));     // 448 = 1.75 * 2^8
}

// Eight fp16 of a row of LANES * 8, spread over LANES lanes, to eight codes; the row's exponent byte. Rows of any kind: with values that are not finite, or
// of exponent 8.
template <int LANES>
__device__ __noinline__ uint2 to_e4m3_any(uint4 x, unsigned& byte)
{
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    uint32_t top2 = 0;
    #pragma unroll
    for (int i = 0; i < 4; i++) top2 = __vmaxu2(top2, w[i] & 0x7fff7fffu & ~nonfinite_f16x2(w[i]));
    uint32_t top = max(top2 & 0xffffu, top2 >> 16);        // magnitudes of fp16 order like their bits
    #pragma unroll
    for (int d = 1; d < LANES; d *= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
    const int e = exponent_of(top);
    byte = (unsigned)(e + 127);
    const float scale = __uint_as_float((unsigned)(127 - e) << 23), most = e == 8 ? 240.f : 448.f;
    uint32_t code[4];
    #pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        float2 y = make_float2(fminf(fmaxf(f.x * scale, -most), most), fminf(fmaxf(f.y * scale, -most), most));
        const uint32_t bad = nonfinite_f16x2(w[i]);        // e4m3 has no infinity: stored as NaN
        if (bad & 0xffffu) y.x = NAN;
        if (bad >> 16) y.y = NAN;
        code[i] = __nv_cvt_float2_to_fp8x2(y, __NV_SATFINITE, __NV_E4M3);
    }
    return make_uint2(code[0] | code[1] << 16, code[2] | code[3] << 16);
}

// The same. Rows that are finite and below 57344 without leaving fp16: x * 2^-e is exact there, or so small that its code is 0 whatever the rounding.
// The kernel executes 112 instructions for 16 bytes, 83 without a conversion (ncu). 12225 tokens x 8 heads of 128: 27 us the way above, so 21 (cold).
template <int LANES>
__device__ __forceinline__ uint2 to_e4m3(const uint4& x, unsigned& byte)
{
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    auto max2 = [](uint32_t a, uint32_t b) { uint32_t r; asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; };
    const uint32_t top2 = max2(max2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu), max2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu)) & 0x7fff7fffu;
    uint32_t top = max(top2 & 0xffffu, top2 >> 16);        // magnitudes order like their bits, NaN above all
    #pragma unroll
    for (int d = 1; d < LANES; d *= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
    if (__any_sync(0xffffffffu, top > 0x7b00u)) return to_e4m3_any<LANES>(x, byte);
    const int e = exponent_of(top), up = min(-e, 15);      // 2^up is an fp16; of rows below 2^-7 there is more to come
    byte = (unsigned)(e + 127);
    const uint32_t h = (uint32_t)(up + 15) << 10, scale = h | h << 16;                      // up is -7 at least
    uint32_t y[4], code[4];
    #pragma unroll
    for (int i = 0; i < 4; i++) y[i] = mul_f16x2(w[i], scale);
    if (e < -15) {
        const uint32_t g = (uint32_t)(-e) << 10, rest = g | g << 16;                // 2^(-e - 15)
        #pragma unroll
        for (int i = 0; i < 4; i++) y[i] = mul_f16x2(y[i], rest);
    }
    #pragma unroll
    for (int i = 0; i < 4; i++) code[i] = __nv_cvt_halfraw2_to_fp8x2(*reinterpret_cast<const __half2_raw*>(&y[i]), __NV_SATFINITE, __NV_E4M3);
    return make_uint2(code[0] | code[1] << 16, code[2] | code[3] << 16);
}

__device__ __forceinline__ uint4 from_e4m3(const uint2& x, unsigned byte)
{
    const uint32_t s = exp_byte_f16x2(byte);
    return make_uint4(mul_f16x2(e4m3x2_to_f16x2(x.x & 0xffffu), s), mul_f16x2(e4m3x2_to_f16x2(x.x >> 16), s),
                      mul_f16x2(e4m3x2_to_f16x2(x.y & 0xffffu), s), mul_f16x2(e4m3x2_to_f16x2(x.y >> 16), s));
}

// Rows into pages (READ: out of them). A row of a head is D / 8 lanes of 16 bytes fp16; a warp takes the 256 / D rows that it holds of one token range and up to
// PC_HEADS heads of K and V at a time. HBM-bound for prompts (5822 tokens x 32 heads of 128 in: 31.5 us, 6.1 TB/s; 73472 x 16 of 64 out 94 us, 6.4 TB/s; of 8 bits
// 100451 x 8 of 128 out 101 us, 6.1 TB/s), a chain of three loads (lengths, page, row) for single tokens, less than the 4.7 us that the host takes for the call.
template <int D, bool F8, bool READ>
__global__ void __launch_bounds__(PC_THREADS)
paged_move_kernel(const PagedArgs c, const PagedRows rows)
{
    constexpr int LANES = D / 8, PER_WARP = 32 / LANES;
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int sub = lane % LANES;
    const int row = (blockIdx.x * (PC_THREADS / 32) + warp) * PER_WARP + lane / LANES;
    const int h0 = blockIdx.y * PC_HEADS<F8, READ>;
    const bool there = row < c.tokens;
    __half* const rk = rows.k + h0 * rows.head + (long long)row * rows.token + sub * 8;
    __half* const rv = rows.v + h0 * rows.head + (long long)row * rows.token + sub * 8;
    const int heads = min(PC_HEADS<F8, READ>, c.H_kv - h0);

    uint4 k[PC_HEADS<F8, READ>], v[PC_HEADS<F8, READ>];
    if constexpr (!READ) {                                 // asked for ahead of the search for their place
        #pragma unroll
        for (int i = 0; i < PC_HEADS<F8, READ>; i++)
            if (there && i < heads) {
                k[i] = *reinterpret_cast<const uint4*>(rk + i * rows.head);
                v[i] = *reinterpret_cast<const uint4*>(rv + i * rows.head);
            } else k[i] = v[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    int page = -1, slot = 0;
    bool owned = false;                                    // a row of some sequence
    if (there) {
        const int b = sequence_of(c, row);
        if (b >= 0) {
            const PagedSeq q = paged_seq(c, b);
            const int i = row - q.row0, position = q.kv - q.n + i;
            owned = i >= 0 && i < q.n;
            if (owned && position >= 0) {
                page = paged_page(c, b, position, 50);
                slot = position & ((1 << c.page_shift) - 1);
            }
        }
    }
    // Of head h0: where the row's chunk lies in the cache, and its exponents; from a head to the next.
    const long long in_page = ((long long)h0 << c.page_shift) + slot, to = max(page, 0) * c.page_stride + (in_page * D + sub * 8) * (F8 ? 1 : 2);
    const long long e = ((long long)max(page, 0) * c.H_kv << c.page_shift) + in_page;
    const int to_step = (D * (F8 ? 1 : 2)) << c.page_shift, e_step = 1 << c.page_shift;
    uint8_t* const pk = c.k + to;
    uint8_t* const pv = c.v + to;
    #pragma unroll
    for (int i = 0; i < PC_HEADS<F8, READ>; i++) {
        if (i >= heads) break;
        const long long o = (long long)i * to_step;
        if constexpr (READ) {
            uint4 x = make_uint4(0u, 0u, 0u, 0u), y = x;
            if (page >= 0) {
                if constexpr (F8) {
                    x = from_e4m3(*reinterpret_cast<const uint2*>(pk + o), c.k_exp[e + i * e_step]);
                    y = from_e4m3(*reinterpret_cast<const uint2*>(pv + o), c.v_exp[e + i * e_step]);
                } else {
                    x = *reinterpret_cast<const uint4*>(pk + o);
                    y = *reinterpret_cast<const uint4*>(pv + o);
                }
            }
            if (owned) {
                *reinterpret_cast<uint4*>(rk + i * rows.head) = x;
                *reinterpret_cast<uint4*>(rv + i * rows.head) = y;
            }
        } else if constexpr (F8) {
            unsigned bk, bv;                               // all lanes of the warp: the row's maximum goes through shuffles
            const uint2 x = to_e4m3<LANES>(k[i], bk), y = to_e4m3<LANES>(v[i], bv);
            if (page >= 0) {
                *reinterpret_cast<uint2*>(pk + o) = x;
                *reinterpret_cast<uint2*>(pv + o) = y;
                if (sub == 0) { c.k_exp[e + i * e_step] = (uint8_t)bk; c.v_exp[e + i * e_step] = (uint8_t)bv; }
            }
        } else if (page >= 0) {
            *reinterpret_cast<uint4*>(pk + o) = k[i];
            *reinterpret_cast<uint4*>(pv + o) = v[i];
        }
    }
    // Wrong lengths, of sequences without rows as well.
    if (blockIdx.x == 0 && blockIdx.y == 0)
        for (int b = threadIdx.x; b < c.num_seqs; b += PC_THREADS) paged_seq<true>(c, b, 50);
}

PagedArgs device_args(const efa_paged_cache& c, const efa_paged_batch& b)
{
    PagedArgs a{};
    a.k = static_cast<uint8_t*>(c.k); a.v = static_cast<uint8_t*>(c.v);
    a.k_exp = c.k_exp; a.v_exp = c.v_exp;
    a.q_start = b.q_start; a.kv_len = b.kv_len; a.pages = b.pages;
    a.num_seqs = b.num_seqs; a.max_pages = b.max_pages; a.tokens = b.tokens; a.max_q = b.max_q;
    a.kv_cap = (int)std::min<long long>(b.max_kv, (long long)b.max_pages * c.page_size);
    a.num_pages = c.num_pages; a.H_kv = c.H_kv;
    while ((1 << a.page_shift) < c.page_size) a.page_shift++;
    const long long per_page = (long long)c.H_kv * c.page_size * c.d_h;
    a.page_stride = (c.page_stride ? c.page_stride : per_page) * (c.dtype == EFA_F16 ? 2 : 1);
    return a;
}

const char* check_rows(const efa_paged_cache& c, const efa_paged_batch& b, long long& head, long long& token)
{
    if (head == 0 && token == 0) { token = c.d_h; head = (long long)b.tokens * c.d_h; return nullptr; }
    if (head < c.d_h || token < c.d_h || head % 8 || token % 8) return "paged: row strides must be multiples of 8 and at least d_h";
    if (token < (c.H_kv - 1) * head + c.d_h && head < (b.tokens - 1) * token + c.d_h) return "paged: rows of these strides overlap";
    return nullptr;
}

template <int D, bool F8>
int launch_move(bool read, const PagedArgs& a, const PagedRows& rows, cudaStream_t stream)
{
    const int per_block = PC_THREADS / 32 * (256 / D), heads = read ? PC_HEADS<F8, true> : PC_HEADS<F8, false>;
    const dim3 grid((a.tokens + per_block - 1) / per_block, (a.H_kv + heads - 1) / heads);
    EFA_CUDA(read ? paged_launch(paged_move_kernel<D, F8, true>, grid, PC_THREADS, 0, stream, a, rows)
                  : paged_launch(paged_move_kernel<D, F8, false>, grid, PC_THREADS, 0, stream, a, rows));
    return 0;
}

int move_rows(const char* what, bool read, const void* K, const void* V, long long head, long long token, const efa_paged_cache& c,
              const efa_paged_batch& b, cudaStream_t stream)
{
    if (const char* why = paged_check(c, b)) { set_error("%s: %s", what, why); return 2; }
    if (const char* why = check_rows(c, b, head, token)) { set_error("%s: %s", what, why); return 2; }
    if (b.num_seqs == 0 || b.tokens == 0 || b.max_q == 0) return 0;
    if (!K || !V) { set_error("%s: K or V is null", what); return 2; }
    if (!aligned16(K) || !aligned16(V)) { set_error("%s: K and V must be 16-byte aligned", what); return 2; }
    const void* const mem[] = {K, V, c.k, b.q_start};
    if (int rc = check_memory(what, mem, 4)) return rc;
    PagedArgs a = device_args(c, b);
    a.status = kernel_status_word();
    const PagedRows rows{static_cast<__half*>(const_cast<void*>(K)), static_cast<__half*>(const_cast<void*>(V)), head, token};
    const bool f8 = c.dtype == EFA_E4M3;
    switch (c.d_h) {
        case 16:  return f8 ? launch_move<16, true>(read, a, rows, stream) : launch_move<16, false>(read, a, rows, stream);
        case 32:  return f8 ? launch_move<32, true>(read, a, rows, stream) : launch_move<32, false>(read, a, rows, stream);
        case 64:  return f8 ? launch_move<64, true>(read, a, rows, stream) : launch_move<64, false>(read, a, rows, stream);
        default:  return f8 ? launch_move<128, true>(read, a, rows, stream) : launch_move<128, false>(read, a, rows, stream);
    }
}

// Which of the two kinds of kernel, its tiles and units, and bounds: keys of a sequence, tiles of a chunk, items of a launch with one block to each, the weight of all items.
// Rows of different sequences are different rows of Q, so that however long single chunks may be their tiles are no more than `tokens` has, and one
// more for each sequence.
struct PagedKind { bool chunk; int tile, unit, extra; long long kv_cap, units; double max_tiles, items, weight; };

PagedKind kind_of(const efa_paged_cache& c, const efa_paged_batch& b, const efa_paged_attention_params& p)
{
    PagedKind k{};
    const int G = p.H_q / c.H_kv;
    const long long rows = (long long)b.max_q * G;
    k.kv_cap = std::min<long long>(b.max_kv, (long long)b.max_pages * c.page_size);
    // Up to 32 rows the keys' way to the SM is the time: small tiles. More go to the tensor cores' tiles of 256 unless there is little work, counted as 64 rows x 64 keys:
    // small tiles start and end faster, and clusters share theirs. us, small tiles / tiles of 256: 64 rows, 8 heads of 128, 1000 keys 14 / 19, 2 x 16000 keys
    // 57 / 47, 16 x 16000 304 / 190, of 8 bits 307 / 230; 32 rows, 16 x 16000 keys 171 / 186; prompts, 16 heads of 64, 128 tokens 7.8 / 8.6, 512 12.9 / 14.0,
    // of 8 bits 256 11.2 / 12.0, 512 19.3 / 14.9; 8 heads of 16, 200 tokens over 400 keys 6.9 / 11.9; 32 heads of 128 on 8, 4 x 64 tokens 9.5 / 11.4, 128 11.2 / 11.3,
    // 256 16.1 / 12.8.
    const bool f8 = c.dtype == EFA_E4M3;
    const double work = (double)b.num_seqs * c.H_kv * (double)((rows + 63) / 64) * (double)((k.kv_cap + 63) / 64);
    k.chunk = rows > 32 && work > (rows <= 64 ? 1024 : c.d_h == 128 ? 128 : c.d_h == 64 ? (f8 ? 256 : 1024) : 2048);
    k.tile = k.chunk ? PAGED_CHUNK_TILE : paged_rows_tile((int)std::min<long long>(rows, INT_MAX));
    k.unit = k.chunk ? PAGED_CHUNK_UNIT : paged_rows_unit(f8);
    k.extra = k.chunk ? PAGED_CHUNK_EXTRA : PAGED_ROWS_EXTRA;
    k.units = std::max<long long>(1, (k.kv_cap + k.unit - 1) / k.unit);
    k.max_tiles = (double)((rows + k.tile - 1) / k.tile);
    k.items = (double)b.num_seqs * c.H_kv * k.max_tiles;
    k.weight = std::min((double)b.num_seqs * k.max_tiles, std::floor((double)b.tokens * G / k.tile) + b.num_seqs) * c.H_kv * (double)(k.units + k.extra);
    return k;
}

struct PagedPlan { PagedShape w; int blocks, cluster; bool cut, chunk; size_t cut_bytes, ml_bytes, o_bytes; };

PagedPlan plan_attention(const efa_paged_cache& c, const efa_paged_batch& b, const efa_paged_attention_params& p)
{
    PagedPlan plan{};
    const PagedKind k = kind_of(c, b, p);
    const int G = p.H_q / c.H_kv, tile = k.tile, unit = k.unit;
    const bool f8 = c.dtype == EFA_E4M3;
    plan.chunk = k.chunk;
    plan.w = PagedShape{G, p.causal ? 1 : 0, tile, unit, k.extra, (int)k.max_tiles, 0, (int)k.weight};
    const long long items = (long long)k.items, units = k.units;
    plan.cluster = 1;
    int parts = device_sms();
    if (plan.chunk) {
        // A block per item, those of the last rows first, or equal shares of everything with a merge behind: in units of 128 keys (about 2 us), for chunks and
        // sequences as long as the bounds allow. Items of about one length go in waves; else, longest first, they come out even. Shares pay for the
        // merge, for pieces half of which begin and end within an item, and for reading keys at different places at a time: blocks in step on many tiles of one
        // sequence find them in the L2. Below MIN_SHARE a block spends its time on anything but keys. us, items / shares: prompts, 16 heads of 64, 1024 tokens
        // 19 / 21, 4096 59 / 68; 32 heads of 128 on 8, 2048 45 / 61, 8192 516 / 559; 2048 tokens over 32768 keys 1004 / 1070, of 8 bits 1099 / 1039; eight
        // sequences, 512 tokens over 4096 keys 310 / 279; one, 64 tokens over 2000 keys 34 / 30. Tiles of max_q that a sequence does not have are blocks as well,
        // of 1.7 us each (tensor memory, lengths): one chunk with single tokens beside it, 32 heads of 128 on 8, 4096 keys, 512 tokens and 63 sequences 276 / 247,
        // 4096 and 127 1286 / 610, 4096 and 255 of 300 keys 1819 / 322.
        constexpr double MIN_SHARE = 6, MERGE = 6, EMPTY = 0.85;
        const double tiles = std::min<double>((double)b.num_seqs * plan.w.max_tiles, (double)b.tokens * G / tile + b.num_seqs) * c.H_kv;
        const double longest = (double)units + PAGED_CHUNK_EXTRA;
        const double first = p.causal ? std::max<double>(1, ((double)k.kv_cap - b.max_q + (double)tile / G) / unit) + PAGED_CHUNK_EXTRA : longest;
        const bool even = first * 2 >= longest;
        const double each = tiles * (first + longest) / 2 / parts;
        const double by_item = (even ? std::ceil(tiles / parts) * longest : std::max(longest, each * 1.05)) + std::max(0.0, k.items - tiles) / parts * EMPTY;
        const double by_share = std::max(MIN_SHARE, each) * 1.05 + MERGE;
        plan.cut = by_item > by_share * (!f8 && plan.w.max_tiles >= 16 ? 1.15 : 1.0);
        parts = (int)std::min<double>(parts, std::max(1.0, each * parts / MIN_SHARE));
    } else {
        // Few rows: a block per item, or where there are few items a cluster of up to eight that shares one, merged in shared memory, as long as a block's part of
        // the longest item stays short; else equal shares of everything, which cost a merge in a launch of its own but leave no SM idle, whatever the
        // lengths. us, clusters / shares, one token: 16 heads of 64 1000 keys 5.6 / 10.2, 8000 12.4 / 14.4, 16000 20.3 / 18.9; 32 heads of 128 on 8,
        // 1000 keys 6.8 / 10.6, 8000 15.8 / 17.2, 16000 26.4 / 19.9; 8 bits (with the host's part) 8.8 / 13.1, 18.1 / 21.6, 29.0 / 27.3; 64 such sequences (no clusters) 1000 keys 45 / 50.
        parts *= paged_rows_blocks_per_sm(c.d_h, f8);
        while (plan.cluster < 8 && plan.cluster * 2 <= units && items * plan.cluster * 2 <= parts) plan.cluster *= 2;
        plan.cut = units * unit > (c.d_h == 128 ? 1024 : 1536) * plan.cluster;
        if (plan.cut) {
            plan.cluster = 1;
            // Where memory is the time: us without / with, 64 sequences of 4096 keys, 16 heads of 64 176.6 / 167.0, of up to 8192, 8 heads of 128 176.5 / 172.0; but
            // of 8 bits 121.7 / 126.8, 105.7 / 110.
            if (!f8 && c.d_h >= 64 && items * units >= (long long)parts * LATE_RATIO * LATE_UNITS) plan.w.late = parts * 3 / 4;
            parts += plan.w.late;
        }
    }
    plan.blocks = (int)(plan.cut ? std::min<long long>(parts, items * units) : items);
    if (plan.cut) {
        plan.cut_bytes = ((size_t)plan.blocks * sizeof(PagedCut) + 255) / 256 * 256;
        plan.ml_bytes = (size_t)plan.blocks * 2 * tile * sizeof(float2);
        plan.o_bytes = (size_t)plan.blocks * 2 * tile * c.d_h * sizeof(float);
    }
    return plan;
}

}  // namespace

const char* paged_check(const efa_paged_cache& c, const efa_paged_batch& b)
{
    if (c.dtype != EFA_F16 && c.dtype != EFA_E4M3) return "paged: the cache must be EFA_F16 or EFA_E4M3";
    if (c.d_h != 16 && c.d_h != 32 && c.d_h != 64 && c.d_h != 128) return "paged: d_h must be 16, 32, 64 or 128";
    if (c.page_size < 16 || c.page_size > 256 || (c.page_size & (c.page_size - 1))) return "paged: page_size must be 16, 32, 64, 128 or 256";
    if (c.H_kv < 1 || c.H_kv > 65535) return "paged: H_kv must be positive";
    if (c.num_pages < 1) return "paged: num_pages must be positive";
    if (!c.k || !c.v || !aligned16(c.k) || !aligned16(c.v)) return "paged: k and v must be 16-byte aligned memory";
    if (c.dtype == EFA_E4M3 && (!c.k_exp || !c.v_exp || !aligned16(c.k_exp) || !aligned16(c.v_exp))) return "paged: an e4m3 cache needs k_exp and v_exp, 16-byte aligned";
    if (c.page_stride != 0 && (c.page_stride < (long long)c.H_kv * c.page_size * c.d_h || c.page_stride % 16)) return "paged: page_stride must be 0 or a multiple of 16 that holds a page";
    if (b.num_seqs < 0 || b.tokens < 0 || b.max_q < 0 || b.max_kv < 0) return "paged: negative size";
    if (b.max_pages < 1) return "paged: max_pages must be positive";
    if (b.num_seqs > 0 && (!b.q_start || !b.kv_len || !b.pages)) return "paged: q_start, kv_len and pages must not be null";
    if (b.tokens > 1 << 30 || b.max_q > 1 << 30 || b.max_kv > 1 << 30 || (long long)b.num_seqs * b.max_pages > INT_MAX || (long long)c.H_kv * c.page_size * c.d_h > INT_MAX) return "paged: sizes too large";
    return nullptr;
}

const char* paged_attention_check(const efa_paged_cache& c, const efa_paged_batch& b, const efa_paged_attention_params& p)
{
    if (const char* why = paged_check(c, b)) return why;
    if (p.H_q < 1 || p.H_q % c.H_kv) return "paged: H_q must be a positive multiple of H_kv";
    if (!std::isfinite(p.scale) || p.scale <= 0.f) return "paged: scale must be positive and finite";
    if (p.q_head_stride || p.q_token_stride) {
        if (p.q_head_stride < c.d_h || p.q_token_stride < c.d_h || p.q_head_stride % 8 || p.q_token_stride % 8) return "paged: row strides must be multiples of 8 and at least d_h";
    }
    if (p.o_token_stride != 0 && (p.o_token_stride < (long long)p.H_q * c.d_h || p.o_token_stride % 8)) return "paged: o_token_stride must be 0 or a multiple of 8 that holds H_q * d_h";
    const PagedKind k = kind_of(c, b, p);                  // counted in 31 bits; of items and rows the kernels add a block's to the number
    if ((long long)b.max_q * (p.H_q / c.H_kv) > INT_MAX / 2 || k.items > (double)(INT_MAX / 2) || k.weight > (double)INT_MAX) return "paged: sizes too large";
    return nullptr;
}

size_t paged_attention_bytes(const efa_paged_cache& c, const efa_paged_batch& b, const efa_paged_attention_params& p)
{
    const PagedPlan plan = plan_attention(c, b, p);
    return plan.cut_bytes + plan.ml_bytes + plan.o_bytes;
}

int cache_write(const void* K, const void* V, long long head_stride, long long token_stride, const efa_paged_cache& c, const efa_paged_batch& b, cudaStream_t stream)
{
    return move_rows("cache_write", false, K, V, head_stride, token_stride, c, b, stream);
}

int cache_read(void* K, void* V, long long head_stride, long long token_stride, const efa_paged_cache& c, const efa_paged_batch& b, cudaStream_t stream)
{
    return move_rows("cache_read", true, K, V, head_stride, token_stride, c, b, stream);
}

int paged_attention(const void* Q, void* O, const efa_paged_cache& c, const efa_paged_batch& b, const efa_paged_attention_params& p,
                    void* workspace, size_t workspace_bytes, cudaStream_t stream)
{
    if (const char* why = paged_attention_check(c, b, p)) { set_error("paged_attention: %s", why); return 2; }
    if (b.num_seqs == 0 || b.tokens == 0 || b.max_q == 0) return 0;
    if (!Q || !O) { set_error("paged_attention: Q or O is null"); return 2; }
    if (!aligned16(Q) || !aligned16(O)) { set_error("paged_attention: Q and O must be 16-byte aligned"); return 2; }
    const PagedPlan plan = plan_attention(c, b, p);
    const size_t need = plan.cut_bytes + plan.ml_bytes + plan.o_bytes;
    if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace))) {
        set_error("paged_attention: needs a workspace of %zu bytes, 16-byte aligned (got %zu)", need, workspace ? workspace_bytes : 0);
        return 2;
    }
    const void* const mem[] = {Q, O, c.k, b.q_start, need ? workspace : nullptr};
    if (int rc = check_memory("paged_attention", mem, 5)) return rc;
    PagedArgs args = device_args(c, b);
    args.status = kernel_status_word();
    PagedAttnArgs a{};
    a.Q = static_cast<const __half*>(Q);
    a.O = static_cast<__half*>(O);
    const bool dense = p.q_head_stride == 0 && p.q_token_stride == 0;
    a.q_head = dense ? (long long)b.tokens * c.d_h : p.q_head_stride;
    a.q_token = dense ? c.d_h : p.q_token_stride;
    a.o_token = p.o_token_stride ? p.o_token_stride : (long long)p.H_q * c.d_h;
    a.scale_log2e = p.scale * 1.4426950408889634f;
    a.rescale_above = c.d_h >= 64 ? 8.f : 0.f;             // as the attention over contiguous keys has it
    a.w = plan.w;
    if (plan.cut) {
        uint8_t* at = static_cast<uint8_t*>(workspace);
        a.parts.cut = reinterpret_cast<PagedCut*>(at);
        a.parts.ml = reinterpret_cast<float2*>(at + plan.cut_bytes);
        a.parts.o = reinterpret_cast<float4*>(at + plan.cut_bytes + plan.ml_bytes);
    }
    const bool f8 = c.dtype == EFA_E4M3;
    if (int rc = plan.chunk ? paged_chunk_launch(args, a, c.d_h, f8, plan.blocks, stream) : paged_rows_launch(args, a, c.d_h, f8, plan.blocks, plan.cluster, stream)) return rc;
    if (!plan.cut || plan.blocks < 2) return 0;
    return paged_merge_launch(args, a, c.d_h, plan.blocks, (int)std::min<long long>(plan.w.tile, (long long)b.max_q * plan.w.G), stream);
}

}  // namespace efa
