// What the kernels of the paged key/value cache share: the cache and the ragged batch as they see them, where a key lies,
// and how work is laid out over the GPU when only the device knows the lengths.
//
// Everything that comes from device memory (lengths, page numbers) is brought into range before it is used as an index: a call whose
// lengths or pages are wrong stays inside its buffers and reports it in the status word.
#pragma once

#include "sm100_ptx.cuh"

namespace efa {

struct PagedArgs {
    uint8_t* k;             // [num_pages][H_kv][page][d_h], fp16 or e4m3
    uint8_t* v;
    uint8_t* k_exp;         // [num_pages][H_kv][page], e4m3 only: 127 + exponent of a row
    uint8_t* v_exp;
    const int* q_start;     // [num_seqs + 1]
    const int* kv_len;      // [num_seqs]
    const int* pages;       // [num_seqs][max_pages]
    int num_seqs, max_pages, tokens, max_q, kv_cap /* min(max_kv, what a row of `pages` holds) */;
    int num_pages, page_shift, H_kv;
    long long page_stride;  // bytes from a page of k or v to the next
    int* status;
};

// The first thing that is wrong stays in the status word (code, sequence, site).
__device__ __forceinline__ void paged_report(const PagedArgs& c, int code, int seq, int site)
{
    if (c.status != nullptr && atomicCAS(c.status, 0, code) == 0) {
        c.status[1] = seq;
        c.status[2] = site;
    }
}

struct PagedSeq { int row0, n, kv; };      // first row of the chunk, its rows, keys in the cache (the chunk's included)

template <bool REPORT = false>
__device__ __forceinline__ PagedSeq paged_seq(const PagedArgs& c, int b, int site = 0)
{
    const int s0 = c.q_start[b], s1 = c.q_start[b + 1], kv = c.kv_len[b];
    PagedSeq s;
    s.row0 = min(max(s0, 0), c.tokens);
    s.n = min(min(max(s1, s.row0), c.tokens) - s.row0, c.max_q);
    s.kv = min(max(kv, 0), c.kv_cap);
    if (REPORT && (s.row0 != s0 || s.n != s1 - s0 || s.kv != kv)) paged_report(c, KS_BAD_LENGTH, b, site);
    return s;
}

// The page that holds key `key` (below kv_cap) of sequence b; -1, and a report, if there is no such page.
__device__ __forceinline__ int paged_page(const PagedArgs& c, int b, int key, int site)
{
    const int page = c.pages[(long long)b * c.max_pages + (key >> c.page_shift)];
    if ((unsigned)page < (unsigned)c.num_pages) return page;
    paged_report(c, KS_BAD_PAGE, b, site);
    return -1;
}

// ---------------------------------------------------------------------------------------------
// e4m3 with an exponent per row: value = code * 2^(byte - 127). The writer's exponents are -24 to 8, for which every value is an fp16
// exactly (a code has four significant bits; 2^-24 is fp16's smallest step).
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ float exp_byte_f32(unsigned byte) { return __uint_as_float(byte << 23); }     // byte 0, which nothing is stored with, as 0

// 2^(byte - 127) twice as fp16. Of bytes that the writer does not store (below 103, above 142) something finite.
__device__ __forceinline__ uint32_t exp_byte_f16x2(unsigned byte)
{
    const uint32_t normal = (min(byte, 142u) - 112u) << 10, h = byte > 112u ? normal : 1u << ((byte - 103u) & 15u);
    return __byte_perm(h, h, 0x1010);
}

// The same of two bytes, one to a half.
__device__ __forceinline__ uint32_t exp_bytes_f16x2(uint32_t two)
{
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(exp_byte_f32(min(two >> 8, 142u))), "f"(exp_byte_f32(min(two & 0xffu, 142u))));
    return r;
}

__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two)
{
    uint32_t r;
    asm("{\n.reg .b16 x;\ncvt.u16.u32 x, %1;\ncvt.rn.f16x2.e4m3x2 %0, x;\n}\n" : "=r"(r) : "r"(two));
    return r;
}

__device__ __forceinline__ void e4m3x4_to_f16x4(uint32_t four, uint32_t& lo, uint32_t& hi)
{
    asm("{\n.reg .b16 x, y;\nmov.b32 {x, y}, %2;\ncvt.rn.f16x2.e4m3x2 %0, x;\ncvt.rn.f16x2.e4m3x2 %1, y;\n}\n" : "=r"(lo), "=r"(hi) : "r"(four));
}

__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b)
{
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// Halves of x that are infinite or NaN as a mask.
__device__ __forceinline__ uint32_t nonfinite_f16x2(uint32_t x)
{
    return __vcmpeq2(x & 0x7c007c00u, 0x7c007c00u);
}

// ---------------------------------------------------------------------------------------------
// Work over the GPU
// ---------------------------------------------------------------------------------------------
// An item is a tile of rows of one sequence and kv head: the rows (token, query head of the group) in that order, `tile` of them
// at a time, so that all heads of a group, and several tokens, share what is loaded of the keys. Its keys are units of
// `unit` keys, as many as its last row sees, and its weight is its units plus `extra` for what an item costs besides them. All items
// in a row (heads outermost) are cut into as many shares of equal weight as there are blocks: no length of any sequence leaves an SM idle.
// An item that a cut goes through is merged afterwards (paged_merge_kernel).
// Equal shares of what memory has to deliver do not end together: some SMs get a tenth less of it than others (64 sequences of 8000 keys, 8 heads of 128:
// blocks end between 252 and 309 us). So the last `late` blocks, which start as others end, have a tenth of a share each, if that is still
// LATE_UNITS: the faster SMs take them.
struct PagedShape {
    int G, causal, tile, unit, extra, max_tiles;   // query heads per kv head; rows of a tile; keys of a unit; ...; tiles of the longest chunk
    int late;
    int limit;              // weight of all items that a batch of these sizes may have
};
constexpr unsigned LATE_UNITS = 4, LATE_RATIO = 10;

__device__ __forceinline__ int paged_tiles(const PagedShape& w, const PagedSeq& s) { return (int)((unsigned)(s.n * w.G + w.tile - 1) / (unsigned)w.tile); }

// Keys that row r of a sequence (token r / G) sees: below this. Not above kv; at most 0: none.
__device__ __forceinline__ int paged_visible(const PagedShape& w, const PagedSeq& s, int r)
{
    return w.causal ? s.kv - s.n + (int)((unsigned)r / (unsigned)w.G) + 1 : s.kv;
}

// One unit at least: rows that see nothing are written as well.
__device__ __forceinline__ int paged_units(const PagedShape& w, const PagedSeq& s, int rt)
{
    const int last = min((rt + 1) * w.tile, s.n * w.G) - 1;
    return max(1, (paged_visible(w, s, last) + w.unit - 1) / w.unit);
}

// A place in the row of items; off: weight of the item ahead of it.
struct PagedAt { int h, b, rt, off; };

__device__ __forceinline__ void paged_next(const PagedArgs& c, const PagedShape& w, PagedAt& at)
{
    at.off = 0;
    at.rt++;
    while (at.h < c.H_kv) {
        if (at.rt < paged_tiles(w, paged_seq(c, at.b))) return;
        at.rt = 0;
        if (++at.b == c.num_seqs) { at.b = 0; at.h++; }
    }
}

// The units [u_lo, u_hi) of the item at `at` that a share with `left` weight from there on has (perhaps none); takes them off `left`.
struct PagedPiece { PagedSeq q; int h, b, rt, units, u_lo, u_hi; };
__device__ __forceinline__ PagedPiece paged_piece(const PagedArgs& c, const PagedShape& w, const PagedAt& at, int& left)
{
    PagedPiece p;
    p.q = paged_seq(c, at.b);
    p.h = at.h; p.b = at.b; p.rt = at.rt;
    p.units = paged_units(w, p.q, at.rt);
    const int take = min(p.units + w.extra - at.off, left);
    p.u_lo = max(0, at.off - w.extra);
    p.u_hi = max(0, at.off + take - w.extra);
    left -= take;
    return p;
}

struct PagedScratch { int warp_sum[32]; PagedAt at; };

// The weight of share `part` of `parts` and where it begins, found by all THREADS threads of a block together; 0: there is less weight
// than shares, and none for this one. Block 0, which like all others looks at every sequence, reports lengths that are wrong. Sequences that overlap
// (q_start falls) may add up to more than any legal batch of these sizes; sums stop at 2^31 - 1, and nobody has a share then.
template <int THREADS>
__device__ int paged_part(const PagedArgs& c, const PagedShape& w, int part, int parts, PagedScratch& s, PagedAt& at, int site)
{
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int entries = c.num_seqs * w.max_tiles, per = (int)((unsigned)(entries + THREADS - 1) / THREADS);
    const int e0 = min(tid * per, entries), e1 = min(e0 + per, entries);
    auto add = [](int x, int y) { return (int)min((unsigned)x + (unsigned)y, 0x7fffffffu); };
    int sum = 0;
    for (int e = e0; e < e1; ) {
        const int b = (int)((unsigned)e / (unsigned)w.max_tiles), rt0 = e - b * w.max_tiles;
        const PagedSeq q = part == 0 ? paged_seq<true>(c, b, site) : paged_seq(c, b);
        const int stop = min(paged_tiles(w, q), rt0 + e1 - e);
        for (int rt = rt0; rt < stop; rt++) sum = add(sum, paged_units(w, q, rt) + w.extra);
        e = (b + 1) * w.max_tiles;
    }
    int before = sum;
    #pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int o = __shfl_up_sync(0xffffffffu, before, d);
        if (lane >= d) before = add(before, o);
    }
    if (lane == 31) s.warp_sum[warp] = before;
    __syncthreads();
    int total = 0;
    #pragma unroll
    for (int i = 0; i < THREADS / 32; i++) {
        if (i < warp) before = add(before, s.warp_sum[i]);
        total = add(total, s.warp_sum[i]);
    }
    if ((long long)total * c.H_kv > w.limit) return 0;
    before -= sum;
    const unsigned all = (unsigned)total * (unsigned)c.H_kv;
    const unsigned big = (unsigned)(parts - w.late), weights = big * LATE_RATIO + (unsigned)w.late;
    unsigned begin, end;
    if (w.late > 0 && all / LATE_UNITS >= weights) {
        auto at_part = [&](unsigned p) { return (unsigned)((unsigned long long)all * (min(p, big) * LATE_RATIO + (p > big ? p - big : 0)) / weights); };
        begin = at_part((unsigned)part);
        end = at_part((unsigned)part + 1);
    } else {
        const unsigned n = min(all, big);
        if ((unsigned)part >= n) return 0;
        const unsigned each = all / n, more = all - each * n;               // the first `more` shares have one more
        begin = (unsigned)part * each + min((unsigned)part, more);
        end = begin + each + ((unsigned)part < more ? 1 : 0);
    }
    const int h = (int)(begin / (unsigned)total), rest = (int)begin - h * total;
    if (rest >= before && rest < before + sum) {
        int left = rest - before;
        for (int e = e0; e < e1; ) {
            const int b = (int)((unsigned)e / (unsigned)w.max_tiles), rt0 = e - b * w.max_tiles;
            const PagedSeq q = paged_seq(c, b);
            const int stop = min(paged_tiles(w, q), rt0 + e1 - e);
            for (int rt = rt0; rt < stop; rt++) {
                const int n = paged_units(w, q, rt) + w.extra;
                if (left < n) { s.at = PagedAt{h, b, rt, left}; e = entries; break; }
                left -= n;
            }
            if (e < entries) e = (b + 1) * w.max_tiles;
        }
    }
    __syncthreads();
    at = s.at;
    return (int)(end - begin);
}

// Where blocks leave their pieces of items that a cut goes through: two places a block, one for the item that its share begins with and one
// for the other (the last). A place is `tile` rows of (maximum in the log2 domain, denominator), and of O without the division as [d_h / 4][tile] float4, so that
// neighbouring rows lie side by side for writer and reader.
struct PagedCut { int h, b, rt, off /* units of that item ahead of the share */, units /* 0: no share */, pad0, pad1, pad2; };
struct PagedParts {
    PagedCut* cut;      // [parts]: what each share begins with
    float2* ml;         // [parts][2][tile]
    float4* o;          // [parts][2][d_h / 4][tile]
};

}  // namespace efa
