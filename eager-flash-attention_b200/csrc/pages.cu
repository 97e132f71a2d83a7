// The pages of a paged cache: taken, shared, given back, moved. All of it goes by device memory: the host knows the sizes only.
//
// Which pages are free is a scan over their counts. One block does it, or for large pools and long lists a cluster of eight, a segment of the pages to each block: 512
// neighbouring pages to a warp, whose votes stay in registers from the counting to the ranking; so the lowest free pages are found in one pass and one launch,
// in an order that nothing but the arrays decides. What moves keys is a kernel of its own over all SMs.
//
// What bounds them, GPU time: the scan is a chain of steps that wait for memory or for one another: arrays, counts, ranks, list, entries (pages of 16 for 180 prompts of up to 2048 tokens taken and
// given back 13.2 us, with the votes in memory instead of registers 26.7; forking one sequence 9.6). Moves are memory's: 68.5 us of bytes in 68 at 6.5 TB/s, compaction 76.9 with its
// plan; 24.2 in 27.3 for copies of 8-bit pages. The table and the counts are renamed beside the moves: after them 83.8.
//
// Everything that comes from device memory is brought into range before it is an index; what was out of range is reported in the status word.
#include "host_util.h"
#include "serving.h"
#include "paged_attention.h"
#include "sm100_ptx.cuh"

#include <algorithm>
#include <climits>

namespace efa {

namespace {

constexpr int PG_CLUSTER = 8, PG_THREADS = 1024, PG_WARPS = PG_THREADS / 32;
constexpr int PG_VOTES = 16, PG_TILE = PG_THREADS * PG_VOTES;  // of 32 pages to a warp; pages that a block looks at in one pass
constexpr int PG_MOVE_THREADS = 256, PG_SEGMENT = 32768;       // bytes of a page that a block moves at a time
enum { SITE_TAKE = 60, SITE_FORK = 61, SITE_FREE = 62, SITE_COMPACT = 63, SITE_COPY = 64 };

struct PoolArgs {
    int* refs;
    int* pages;
    int* kv_len;
    int num_pages, page_size, num_seqs, max_pages;
    int* status;
};

__device__ __forceinline__ void report(int* status, int code, int who, int site)
{
    if (status != nullptr && atomicCAS(status, 0, code) == 0) {
        status[1] = who;
        status[2] = site;
    }
}

__device__ __forceinline__ long long capacity(const PoolArgs& p) { return (long long)p.max_pages * p.page_size; }

// Keys of a slot, brought into what its table holds.
__device__ __forceinline__ int keys_that_fit(const PoolArgs& p, int kv) { return (int)min(max((long long)kv, 0ll), min(capacity(p), (long long)INT_MAX)); }
__device__ __forceinline__ int keys_in_table(const PoolArgs& p, int kv, int b, int site)
{
    const int cut = keys_that_fit(p, kv);
    if (cut != kv) report(p.status, KS_BAD_LENGTH, b, site);
    return cut;
}
__device__ __forceinline__ int keys_of(const PoolArgs& p, int b, int site) { return keys_in_table(p, p.kv_len[b], b, site); }
__device__ __forceinline__ int pages_of(const PoolArgs& p, int keys) { return (int)(((long long)keys + p.page_size - 1) / p.page_size); }

// Sum of the values of the threads before this one, and of all of them in `total`; `part` [PG_WARPS] in shared memory.
__device__ __forceinline__ int block_scan(int v, int* part, int& total)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int run = v;
    #pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int o = __shfl_up_sync(0xffffffffu, run, d);
        if (lane >= d) run += o;
    }
    __syncthreads();
    if (lane == 31) part[warp] = run;
    __syncthreads();
    int w = part[lane], all = w;
    #pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int o = __shfl_up_sync(0xffffffffu, all, d);
        if (lane >= d) all += o;
    }
    total = __shfl_sync(0xffffffffu, all, 31);
    return run - v + __shfl_sync(0xffffffffu, all - w, warp);
}

// All blocks of the cluster, or of the one block there is.
__device__ __forceinline__ void sync_all() { if (gridDim.z > 1) cluster_sync(); else __syncthreads(); }
__device__ __forceinline__ int rank_of_block() { return gridDim.z > 1 ? (int)cluster_rank() : 0; }
__device__ __forceinline__ int shared_of(const int* p, int block)
{
    if (gridDim.z == 1) return *p;
    int x;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(x) : "r"(cluster_addr(p, (uint32_t)block)));
    return x;
}

struct Range { int lo, hi; };
__device__ __forceinline__ Range segment(int n)
{
    const int each = (int)(((long long)n + gridDim.z - 1) / gridDim.z), lo = (int)min((long long)n, (long long)each * rank_of_block());
    return Range{lo, (int)min((long long)n, (long long)lo + each)};
}

// A warp's pages of the tile at `base`: votes[j] says which of base + warp * 512 + 32 j + (0 .. 31) satisfy the predicate; their number.
template <class F>
__device__ __forceinline__ int vote(int base, int hi, uint32_t (&votes)[PG_VOTES], F predicate)
{
    const int first = base + (int)(threadIdx.x >> 5) * (32 * PG_VOTES) + (int)(threadIdx.x & 31);
    bool yes[PG_VOTES];
    #pragma unroll
    for (int j = 0; j < PG_VOTES; j++) yes[j] = first + 32 * j < hi && predicate(first + 32 * j);
    int n = 0;
    #pragma unroll
    for (int j = 0; j < PG_VOTES; j++) {
        votes[j] = __ballot_sync(0xffffffffu, yes[j]);
        n += __popc(votes[j]);
    }
    return n;
}

// Sums of a warp's numbers over the block: of the warps before, and of all.
__device__ __forceinline__ int warp_scan(int n, int* part, int& total)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __syncthreads();
    if (lane == 0) part[warp] = n;
    __syncthreads();
    const int w = part[lane];
    int all = w;
    #pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int o = __shfl_up_sync(0xffffffffu, all, d);
        if (lane >= d) all += o;
    }
    total = __shfl_sync(0xffffffffu, all, 31);
    return __shfl_sync(0xffffffffu, all - w, warp);
}

// Calls f(page, rank) for the pages that the votes name; rank: that of the warp's first.
template <class F>
__device__ __forceinline__ void ranked(int base, const uint32_t (&votes)[PG_VOTES], int rank, F f)
{
    const int lane = threadIdx.x & 31, first = base + (int)(threadIdx.x >> 5) * (32 * PG_VOTES) + lane;
    #pragma unroll
    for (int j = 0; j < PG_VOTES; j++) {
        if (votes[j] >> lane & 1u) f(first + 32 * j, rank + __popc(votes[j] & ((1u << lane) - 1u)));
        rank += __popc(votes[j]);
    }
}

// The numbers that the blocks have put into `mine` (shared memory), a block's to a lane, and their sums: of the blocks before, and of all. A word from another SM takes 400 cycles: all at once.
struct Sums { int own, before, all; };
__device__ __forceinline__ Sums sums_of(const int* mine)
{
    const int lane = threadIdx.x & 31, x = lane < (int)gridDim.z ? shared_of(mine, lane) : 0;
    return Sums{x, (int)__reduce_add_sync(0xffffffffu, lane < rank_of_block() ? x : 0), (int)__reduce_add_sync(0xffffffffu, x)};
}
// The same of v. Ends with everything that was written visible to all.
__device__ __forceinline__ int over_blocks(int v, int* mine, int& total)
{
    if (threadIdx.x == 0) *mine = v;
    sync_all();
    const Sums s = sums_of(mine);
    total = s.all;
    return s.before;
}

// The free pages of a block's segment: found (their number), and listed: those of a rank below `wanted` go to list[rank] and have a count of 1 from then on.
struct FreePages {
    Range own;
    uint32_t votes[PG_VOTES];            // of the segment's first tile, which is mostly all of it
    int n;                               // free pages of that, of this warp

    // `meanwhile`: what has to be asked for too, while the counts are on their way.
    template <class F>
    __device__ __forceinline__ int find(const int* refs, int num_pages, int* part, F meanwhile)
    {
        own = segment(num_pages);
        const auto free = [&](int p) { return refs[p] <= 0; };
        const int first = own.lo + (int)(threadIdx.x >> 5) * (32 * PG_VOTES) + (int)(threadIdx.x & 31);
        int count[PG_VOTES];
        #pragma unroll
        for (int j = 0; j < PG_VOTES; j++) count[j] = first + 32 * j < own.hi ? refs[first + 32 * j] : 1;
        meanwhile();
        n = 0;
        #pragma unroll
        for (int j = 0; j < PG_VOTES; j++) {
            votes[j] = __ballot_sync(0xffffffffu, count[j] <= 0);
            n += __popc(votes[j]);
        }
        int total, all;
        warp_scan(n, part, total);
        for (int base = own.lo + PG_TILE; base < own.hi; base += PG_TILE) {
            uint32_t v[PG_VOTES];
            warp_scan(vote(base, own.hi, v, free), part, all);
            total += all;
        }
        return total;
    }
    __device__ __forceinline__ void list(int* refs, int before, int wanted, int* to, int* part)
    {
        const auto take = [&](int p, int rank) { if (rank < wanted) { to[rank] = p; refs[p] = 1; } };
        int total;
        int rank = before + warp_scan(n, part, total);
        ranked(own.lo, votes, rank, take);
        before += total;
        for (int base = own.lo + PG_TILE; base < own.hi && before < wanted; base += PG_TILE) {
            uint32_t v[PG_VOTES];
            const int m = vote(base, own.hi, v, [&](int p) { return refs[p] <= 0; });
            rank = before + warp_scan(m, part, total);
            ranked(base, v, rank, take);
            before += total;
        }
    }
};

// workspace: list [num_pages]; of slots behind a block's first PG_THREADS the pages they have, those they get, and how many the block's slots before them get.
struct TakeArgs { PoolArgs p; const int* q_start; int* list; int* have; int* gets; int* rank; };

__global__ void __launch_bounds__(PG_THREADS)
pages_take_kernel(const TakeArgs a)
{
    __shared__ int part[PG_WARPS], need_of, free_of;
    __shared__ int have_of[PG_THREADS], gets_of[PG_THREADS], rank_of[PG_THREADS];      // of the block's first slots; of others in the workspace
    pdl_wait();
    pdl_trigger();
    const PoolArgs& p = a.p;
    const Range seqs = segment(p.num_seqs);
    FreePages pages;
    struct Slot { int kv, from, to; } first{0, 0, 0};
    auto ask = [&](int b) { return b < seqs.hi ? Slot{p.kv_len[b], a.q_start[b], a.q_start[b + 1]} : Slot{0, 0, 0}; };
    const int found = pages.find(p.refs, p.num_pages, part, [&]() { first = ask(seqs.lo + (int)threadIdx.x); });
    int need = 0;
    for (int base = seqs.lo; base < seqs.hi; base += PG_THREADS) {
        const int b = base + (int)threadIdx.x;
        const Slot slot = base == seqs.lo ? first : ask(b);
        int have = 0, gets = 0, total;
        if (b < seqs.hi) {
            const int kv = keys_in_table(p, slot.kv, b, SITE_TAKE);
            const long long n = (long long)slot.to - slot.from;
            const long long after = min((long long)kv + max(n, 0ll), min(capacity(p), (long long)INT_MAX));
            if (n < 0 || after != kv + n) report(p.status, KS_BAD_LENGTH, b, SITE_TAKE);
            have = pages_of(p, kv);
            gets = pages_of(p, (int)after) - have;
            p.kv_len[b] = (int)after;                          // no other thread looks at it
        }
        const int rank = need + block_scan(gets, part, total);
        if (base == seqs.lo) { have_of[threadIdx.x] = have; gets_of[threadIdx.x] = gets; rank_of[threadIdx.x] = rank; }
        else if (b < seqs.hi) { a.have[b] = have; a.gets[b] = gets; a.rank[b] = rank; }
        need += total;
    }
    if (threadIdx.x == 0) { need_of = need; free_of = found; }
    sync_all();
    const Sums needs = sums_of(&need_of), frees = sums_of(&free_of);
    const int there = frees.all;
    pages.list(p.refs, frees.before, needs.all, a.list, part);
    sync_all();
    // Entries of the block's slots, in turn to its warps.
    for (int b = seqs.lo + (int)(threadIdx.x >> 5); b < seqs.hi; b += PG_WARPS) {
        const int at = b - seqs.lo, gets = at < PG_THREADS ? gets_of[at] : a.gets[b];
        if (gets == 0) continue;
        const int rank = needs.before + (at < PG_THREADS ? rank_of[at] : a.rank[b]);
        int* const to = p.pages + (long long)b * p.max_pages + (at < PG_THREADS ? have_of[at] : a.have[b]);
        if ((threadIdx.x & 31) == 0 && rank + gets > there) report(p.status, KS_NO_PAGE, b, SITE_TAKE);
        #pragma unroll 4
        for (int e = (int)(threadIdx.x & 31); e < gets; e += 32) to[e] = rank + e < there ? a.list[rank + e] : -1;
    }
}

// Moves: pairs of pages, whole (keys NULL) or their first keys[i] keys. count: on the device, or NULL for n of them.
struct MoveArgs {
    uint8_t* part[2];           // k, v
    uint8_t* exps[2];           // their exponents, or NULL
    long long stride;           // bytes from a page to the next
    int head_bytes, key_bytes;  // bytes of a head of a page, and of a key of it
    int heads, page_size, num_pages;
    int segments;               // of a page's k: heads, or pieces of PG_SEGMENT bytes
    const int* src;
    const int* dst;
    const int* keys;
    const int* count;
    int n, site;
    int* status;
};

// Moves first, first + step, ... of n pairs of pages, by a block.
__device__ __forceinline__ void move(const MoveArgs& a, int n, long long first, long long step)
{
    constexpr int THREADS = PG_MOVE_THREADS;
    const int thread = threadIdx.x;
    const int per_page = 2 * a.segments;
    const long long items = (long long)n * per_page;
    for (long long item = first; item < items; item += step) {
        const int i = (int)(item / per_page), of_page = (int)(item % per_page), what = of_page / a.segments, s = of_page % a.segments;
        const int src = a.src[i], dst = a.dst[i], keys = a.keys ? a.keys[i] : 0;
        if ((unsigned)src >= (unsigned)a.num_pages || (unsigned)dst >= (unsigned)a.num_pages) {
            if (thread == 0 && of_page == 0) report(a.status, KS_BAD_PAGE, i, a.site);
            continue;
        }
        // A head's first keys, or a segment of the page; with it the exponents of these keys, or, beside the first segment, all of the page's.
        const long long at = a.keys ? (long long)s * a.head_bytes : (long long)s * PG_SEGMENT;
        const int bytes = a.keys ? keys * a.key_bytes : (int)min((long long)PG_SEGMENT, (long long)a.heads * a.head_bytes - at);
        uint8_t* const part = what ? a.part[1] : a.part[0];
        uint8_t* const exps = what ? a.exps[1] : a.exps[0];
        const uint8_t* const from = part + src * a.stride + at;
        uint8_t* const to = part + dst * a.stride + at;
        const int chunks = bytes / 16;                         // a key is 16 bytes at least
        int c = thread;
        for (; c + 7 * THREADS < chunks; c += 8 * THREADS) {
            uint4 v[8];
            #pragma unroll
            for (int j = 0; j < 8; j++) v[j] = reinterpret_cast<const uint4*>(from)[c + j * THREADS];
            #pragma unroll
            for (int j = 0; j < 8; j++) reinterpret_cast<uint4*>(to)[c + j * THREADS] = v[j];
        }
        if (c < chunks) {
            uint4 v[7];
            #pragma unroll
            for (int j = 0; j < 7; j++)
                if (c + j * THREADS < chunks) v[j] = reinterpret_cast<const uint4*>(from)[c + j * THREADS];
            #pragma unroll
            for (int j = 0; j < 7; j++)
                if (c + j * THREADS < chunks) reinterpret_cast<uint4*>(to)[c + j * THREADS] = v[j];
        }
        if (exps) {                                            // of a head's keys byte by byte, of a page, beside its first segment, all
            const long long page = (long long)a.heads * a.page_size;
            const uint8_t* const es = exps + src * page + (a.keys ? (long long)s * a.page_size : 0);
            uint8_t* const ed = exps + dst * page + (a.keys ? (long long)s * a.page_size : 0);
            if (a.keys)
                for (int k = thread; k < keys; k += THREADS) ed[k] = es[k];
            else if (s == 0)
                for (long long l = thread; l * 16 < page; l += THREADS) reinterpret_cast<uint4*>(ed)[l] = reinterpret_cast<const uint4*>(es)[l];
        }
    }
}

// workspace of a fork: list [num_pages], then [num_seqs] each of claim, keys of the child and rank of its page (behind a block's first PG_THREADS), and the moves: source, target, keys; then their count.
struct ForkArgs { PoolArgs p; const int* parents; const int* children; int n; int* list; int* claim; int* keys; int* rank; int* src; int* dst; int* rest; int* count; };

constexpr int PG_FEW = 512;             // forks whose children are compared with one another, without the claims' round trip through memory

__global__ void __launch_bounds__(PG_THREADS)
pages_fork_kernel(const ForkArgs a)
{
    __shared__ int part[PG_WARPS], mine[2], named[PG_FEW];
    __shared__ int keys_of_fork[PG_THREADS], rank_of_fork[PG_THREADS];                 // of the block's first forks; of others in the workspace
    pdl_wait();
    pdl_trigger();
    const PoolArgs& p = a.p;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Range forks = segment(a.n);
    auto slot = [&](int b) { return (unsigned)b < (unsigned)p.num_seqs; };
    FreePages pages;
    struct Pair { int child, parent, child_keys, parent_keys, source; };
    // source: the page that is not full, of a parent that has one.
    auto ask = [&](int i) {
        Pair x{-1, -1, 0, 0, -1};
        if (i >= forks.hi) return x;
        x.child = a.children[i];
        x.parent = a.parents[i];
        if (slot(x.child)) x.child_keys = p.kv_len[x.child];
        if (slot(x.parent)) {
            x.parent_keys = p.kv_len[x.parent];
            const int keys = keys_that_fit(p, x.parent_keys);
            if (keys % p.page_size) x.source = p.pages[(long long)x.parent * p.max_pages + keys / p.page_size];
        }
        return x;
    };
    const int found = pages.find(p.refs, p.num_pages, part, []() {});

    // The first entry that names a child has it.
    const bool few = a.n <= PG_FEW;
    if (few) {
        if ((int)threadIdx.x < a.n) named[threadIdx.x] = a.children[threadIdx.x];
        __syncthreads();
    } else {
        for (int i = forks.lo + (int)threadIdx.x; i < forks.hi; i += PG_THREADS)
            if (slot(a.children[i])) a.claim[a.children[i]] = INT_MAX;
        sync_all();
        for (int i = forks.lo + (int)threadIdx.x; i < forks.hi; i += PG_THREADS)
            if (slot(a.children[i])) atomicMin(&a.claim[a.children[i]], i);
        sync_all();
    }
    // Keys of the children (-1: an entry that changes nothing) and the ranks of the pages that they get.
    int need = 0;
    for (int base = forks.lo; base < forks.hi; base += PG_THREADS) {
        const int i = base + (int)threadIdx.x;
        const Pair x = ask(i);
        int keys = -1, wants = 0, total;
        if (i < forks.hi) {
            const int c = x.child, b = x.parent;
            bool original = true;
            if (few) {
                #pragma unroll 8
                for (int j = 0; j < i; j++) original &= named[j] != c;
            } else original = slot(c) && a.claim[c] == i;
            if (!original || !slot(c) || !slot(b) || x.child_keys != 0) report(p.status, KS_BAD_SLOT, slot(c) ? c : i, SITE_FORK);
            else {
                keys = keys_in_table(p, x.parent_keys, b, SITE_FORK);
                if (keys % p.page_size) {
                    if ((unsigned)x.source < (unsigned)p.num_pages) wants = 1;
                    else report(p.status, KS_BAD_PAGE, b, SITE_FORK);
                }
            }
        }
        const int before = need + block_scan(wants, part, total), rank = wants ? before : -1;
        if (base == forks.lo) { keys_of_fork[threadIdx.x] = keys; rank_of_fork[threadIdx.x] = rank; }
        else if (i < forks.hi) { a.keys[i] = keys; a.rank[i] = rank; }
        need += total;
    }
    if (threadIdx.x == 0) mine[1] = found;
    int wanted;
    const int need_before = over_blocks(need, &mine[0], wanted);
    const Sums frees = sums_of(&mine[1]);
    const int there = frees.all;
    pages.list(p.refs, frees.before, wanted, a.list, part);
    if (rank_of_block() == 0 && threadIdx.x == 0) *a.count = min(wanted, there);
    sync_all();
    for (int i = forks.lo + warp; i < forks.hi; i += PG_WARPS) {
        const int at = i - forks.lo, keys = at < PG_THREADS ? keys_of_fork[at] : a.keys[i];
        if (keys < 0) continue;
        const int rank_here = at < PG_THREADS ? rank_of_fork[at] : a.rank[i], rank = rank_here < 0 ? -1 : need_before + rank_here;
        const int c = a.children[i], full = keys / p.page_size;
        const int* const from = p.pages + (long long)a.parents[i] * p.max_pages;
        int* const to = p.pages + (long long)c * p.max_pages;
        #pragma unroll 4
        for (int e = lane; e < full; e += 32) {
            const int page = from[e];
            const bool good = (unsigned)page < (unsigned)p.num_pages;
            to[e] = good ? page : -1;
            if (good) atomicAdd(&p.refs[page], 1);
            else report(p.status, KS_BAD_PAGE, a.parents[i], SITE_FORK);
        }
        if (lane == 0) {
            if (keys % p.page_size) {
                const bool got = rank >= 0 && rank < there;
                const int page = got ? a.list[rank] : -1;
                to[full] = page;
                if (got) {
                    a.src[rank] = from[full];
                    a.dst[rank] = page;
                    a.rest[rank] = keys % p.page_size;
                } else if (rank >= 0) report(p.status, KS_NO_PAGE, c, SITE_FORK);
            }
            p.kv_len[c] = keys;
        }
    }
}

constexpr int PG_FREE_THREADS = 128;

__global__ void __launch_bounds__(PG_FREE_THREADS)
pages_free_kernel(const PoolArgs p, const int* seqs)
{
    __shared__ int keys_of_slot;
    pdl_wait();
    pdl_trigger();
    const int i = blockIdx.x, b = seqs[i];
    if ((unsigned)b >= (unsigned)p.num_seqs) {
        if (threadIdx.x == 0) report(p.status, KS_BAD_SLOT, i, SITE_FREE);
        return;
    }
    if (threadIdx.x == 0) keys_of_slot = atomicExch(&p.kv_len[b], 0);          // whoever names the slot again finds it empty
    __syncthreads();
    const int keys = keys_of_slot, cut = keys_that_fit(p, keys);
    if (cut != keys && threadIdx.x == 0) report(p.status, KS_BAD_LENGTH, b, SITE_FREE);
    const int held = pages_of(p, cut);
    #pragma unroll 4
    for (int e = threadIdx.x; e < held; e += PG_FREE_THREADS) {
        const int page = p.pages[(long long)b * p.max_pages + e];
        if ((unsigned)page >= (unsigned)p.num_pages) {
            if (page != -1) report(p.status, KS_BAD_PAGE, b, SITE_FREE);       // -1: there was no page to be had
        } else if (atomicSub(&p.refs[page], 1) <= 0) {
            atomicAdd(&p.refs[page], 1);
            report(p.status, KS_BAD_PAGE, b, SITE_FREE);
        }
    }
}

// workspace: moves from and to [num_pages / 2 + 1] each, and their count.
struct CompactArgs { PoolArgs p; int* pages_out; int* refs_out; int* moved; int* from; int* to; int* count; };

__global__ void __launch_bounds__(PG_THREADS)
pages_compact_kernel(const CompactArgs a)
{
    __shared__ int part[PG_WARPS], mine[2];
    pdl_wait();
    pdl_trigger();
    const PoolArgs& p = a.p;
    FreePages pages;
    const int found = pages.find(p.refs, p.num_pages, part, []() {});
    int free_all;
    const int free_before = over_blocks(found, &mine[0], free_all);
    const int live = p.num_pages - free_all;
    // Free pages before L, in this segment: as many as pages in use at or behind L. Rank of a free page before L: of its hole.
    int rank = free_before, total, holes = 0;
    auto in_front = [&](int base, const uint32_t (&votes)[PG_VOTES]) {
        int n = 0;
        const int first = base + (int)(threadIdx.x >> 5) * (32 * PG_VOTES);
        #pragma unroll
        for (int j = 0; j < PG_VOTES; j++) {
            const int left = live - (first + 32 * j);          // of the 32, those before L
            n += left >= 32 ? __popc(votes[j]) : left > 0 ? __popc(votes[j] & ((1u << left) - 1u)) : 0;
        }
        return n;
    };
    auto free = [&](int q) { return p.refs[q] <= 0; };
    for (int base = pages.own.lo; base < pages.own.hi && base < live; base += PG_TILE) {
        uint32_t v[PG_VOTES];
        if (base == pages.own.lo) {
            #pragma unroll
            for (int j = 0; j < PG_VOTES; j++) v[j] = pages.votes[j];
        } else vote(base, pages.own.hi, v, free);
        warp_scan(in_front(base, v), part, total);
        holes += total;
    }
    int moves;
    over_blocks(holes, &mine[1], moves);
    for (int base = pages.own.lo; base < pages.own.hi; base += PG_TILE) {
        uint32_t v[PG_VOTES];
        int n = pages.n;
        if (base == pages.own.lo) {
            #pragma unroll
            for (int j = 0; j < PG_VOTES; j++) v[j] = pages.votes[j];
        } else n = vote(base, pages.own.hi, v, free);
        int at = rank + warp_scan(n, part, total);             // free pages before this warp's
        const int lane = threadIdx.x & 31, first = base + (int)(threadIdx.x >> 5) * (32 * PG_VOTES) + lane;
        #pragma unroll
        for (int j = 0; j < PG_VOTES; j++) {
            const int q = first + 32 * j, frees = at + __popc(v[j] & ((1u << lane) - 1u));
            if (q < pages.own.hi) {
                const bool is_free = v[j] >> lane & 1u;
                if (!is_free && q >= live) a.from[q - frees - (live - moves)] = q;     // pages in use before q, less those before L
                else a.moved[q] = is_free ? -1 : q;
                if (is_free && q < live) a.to[frees] = q;
            }
            at += __popc(v[j]);
        }
        rank += total;
    }
    if (rank_of_block() == 0 && threadIdx.x == 0) *a.count = moves;
    sync_all();
    for (int i = rank_of_block() * PG_THREADS + threadIdx.x; i < moves; i += (int)gridDim.z * PG_THREADS) a.moved[a.from[i]] = a.to[i];
}

// The table and the counts of the pool after the moves, by `blocks` blocks of 256 threads.
__device__ __forceinline__ void rename(const CompactArgs& a, int block, int blocks)
{
    const PoolArgs& p = a.p;
    const int lane = threadIdx.x & 31, warps = blocks * 8, warp = block * 8 + (threadIdx.x >> 5);
    for (int b = warp; b < p.num_seqs; b += warps) {
        const int held = pages_of(p, keys_of(p, b, SITE_COMPACT));
        #pragma unroll 4
        for (int e = lane; e < held; e += 32) {
            const long long at = (long long)b * p.max_pages + e;
            const int page = p.pages[at], to = (unsigned)page < (unsigned)p.num_pages ? a.moved[page] : -1;
            if (to < 0 && page != -1) report(p.status, KS_BAD_PAGE, b, SITE_COMPACT);
            a.pages_out[at] = to;
        }
    }
    // A place before L that was free is written by the page that moves there, every other by itself.
    const int moves = *a.count, last = moves ? a.to[moves - 1] : -1;
    for (int q = warp * 32 + lane; q < p.num_pages; q += warps * 32) {
        const int to = a.moved[q], n = p.refs[q];
        if (to == q) a.refs_out[q] = n;
        else if (to >= 0) { a.refs_out[to] = n; a.refs_out[q] = 0; }
        else if (q > last) a.refs_out[q] = 0;                  // behind the last free place that is filled
    }
}

// RENAME: first the table and the counts, by the grid's first `renamers` blocks, which take part in the moves last.
template <bool RENAME>
__global__ void __launch_bounds__(PG_MOVE_THREADS)
pages_move_kernel(const MoveArgs a, const CompactArgs names, int renamers)
{
    pdl_wait();
    pdl_trigger();
    if (RENAME && (int)blockIdx.x < renamers) rename(names, blockIdx.x, renamers);
    move(a, a.count ? min(*a.count, a.n) : a.n, RENAME ? ((int)blockIdx.x + (int)gridDim.x - renamers) % (int)gridDim.x : blockIdx.x, gridDim.x);
}

MoveArgs move_args(const efa_paged_cache& c, const int* src, const int* dst, const int* keys, const int* count, int n, int site, int* status)
{
    MoveArgs a{};
    const int elem = c.dtype == EFA_F16 ? 2 : 1;
    const long long dense = (long long)c.H_kv * c.page_size * c.d_h;
    a.part[0] = static_cast<uint8_t*>(c.k); a.part[1] = static_cast<uint8_t*>(c.v);
    if (c.dtype == EFA_E4M3) { a.exps[0] = c.k_exp; a.exps[1] = c.v_exp; }
    a.stride = (c.page_stride ? c.page_stride : dense) * elem;
    a.key_bytes = c.d_h * elem;
    a.head_bytes = a.key_bytes * c.page_size;
    a.page_size = c.page_size;
    a.heads = c.H_kv; a.num_pages = c.num_pages;
    a.src = src; a.dst = dst; a.keys = keys; a.count = count;
    a.n = n; a.site = site; a.status = status;
    a.segments = keys ? c.H_kv : (int)(((long long)c.H_kv * a.head_bytes + PG_SEGMENT - 1) / PG_SEGMENT);
    return a;
}

int launch_moves(const MoveArgs& a, const CompactArgs* names, cudaStream_t stream)
{
    const long long items = (long long)a.n * 2 * a.segments, most = 8ll * device_sms();
    if (names) {
        const int work = std::max(names->p.num_seqs, (names->p.num_pages + 31) / 32), renamers = std::min((work + 7) / 8, device_sms());
        const unsigned blocks = (unsigned)std::max<long long>(renamers, std::min(items, most));
        EFA_CUDA(launch_value(pages_move_kernel<true>, dim3(blocks), PG_MOVE_THREADS, 0, stream, a, *names, renamers));
    } else EFA_CUDA(launch_value(pages_move_kernel<false>, dim3((unsigned)std::min(items, most)), PG_MOVE_THREADS, 0, stream, a, CompactArgs{}, 0));
    return 0;
}

// Blocks of a launch that looks at all pages and at n slots: one while that is little, as eight wait for one another. GPU time, us, one / eight: fork of one sequence 9.8 / 12.1, of 192 32.5 /
// 29.8; pages for 180 prompts 27.3 / 13.9.
int blocks_of(const efa_page_pool& p, int n) { return p.num_pages > PG_TILE || n > PG_WARPS ? PG_CLUSTER : 1; }

PoolArgs device_pool(const efa_page_pool& p) { return PoolArgs{p.refs, p.pages, p.kv_len, p.num_pages, p.page_size, p.num_seqs, p.max_pages, kernel_status_word()}; }

size_t words(int n) { return ((size_t)n + 3) / 4 * 4; }

int check_workspace(const char* what, const efa_page_pool& p, const void* workspace, size_t bytes)
{
    const size_t need = pages_bytes(p);
    if (!workspace || bytes < need || !aligned16(workspace)) {
        set_error("%s: needs a workspace of %zu bytes, 16-byte aligned (got %zu)", what, need, workspace ? bytes : 0);
        return 2;
    }
    return 0;
}

const char* check_cache(const efa_paged_cache& c, const efa_page_pool* p)
{
    const efa_paged_batch none{nullptr, nullptr, nullptr, 0, 1, 0, 0, 0};
    if (const char* why = paged_check(c, none)) return why;
    if (p && (c.num_pages != p->num_pages || c.page_size != p->page_size)) return "pages: pool and cache must have the same number of pages of the same size";
    return nullptr;
}

}  // namespace

const char* page_pool_check(const efa_page_pool& p)
{
    if (p.page_size < 16 || p.page_size > 256 || (p.page_size & (p.page_size - 1))) return "pages: page_size must be 16, 32, 64, 128 or 256";
    if (p.num_pages < 1 || p.max_pages < 1) return "pages: num_pages and max_pages must be positive";
    if (p.num_seqs < 0) return "pages: negative number of slots";
    if (!p.refs) return "pages: refs must not be null";
    if (p.num_seqs > 0 && (!p.pages || !p.kv_len)) return "pages: pages and kv_len must not be null";
    if (!aligned(p.refs, 4) || !aligned(p.pages, 4) || !aligned(p.kv_len, 4)) return "pages: arrays must be aligned to their numbers";
    if (p.num_pages > 1 << 30 || p.num_seqs > 1 << 30 || (long long)p.num_seqs * p.max_pages > INT_MAX) return "pages: sizes too large";
    return nullptr;
}

size_t pages_bytes(const efa_page_pool& p) { return 4 * (words(p.num_pages + 2) + 6 * words(p.num_seqs) + 4); }

int pages_take(const efa_page_pool& p, const int* q_start, void* workspace, size_t workspace_bytes, cudaStream_t stream)
{
    if (const char* why = page_pool_check(p)) { set_error("pages_take: %s", why); return 2; }
    if (p.num_seqs == 0) return 0;
    if (!q_start || !aligned(q_start, 4)) { set_error("pages_take: q_start is null or not aligned"); return 2; }
    if (int rc = check_workspace("pages_take", p, workspace, workspace_bytes)) return rc;
    const void* const mem[] = {p.refs, p.pages, p.kv_len, q_start, workspace};
    if (int rc = check_memory("pages_take", mem, 5)) return rc;
    int* const list = static_cast<int*>(workspace);
    int* const slots = list + words(p.num_pages + 2);
    const TakeArgs a{device_pool(p), q_start, list, slots, slots + words(p.num_seqs), slots + 2 * words(p.num_seqs)};
    EFA_CUDA(launch_value(pages_take_kernel, dim3(1, 1, blocks_of(p, p.num_seqs)), PG_THREADS, 0, stream, a));
    return 0;
}

int pages_fork(const efa_page_pool& p, const efa_paged_cache& c, const int* parents, const int* children, int n, void* workspace, size_t workspace_bytes, cudaStream_t stream)
{
    if (const char* why = page_pool_check(p)) { set_error("pages_fork: %s", why); return 2; }
    if (const char* why = check_cache(c, &p)) { set_error("pages_fork: %s", why); return 2; }
    if (n < 0 || n > p.num_seqs) { set_error("pages_fork: n must be from 0 to the number of slots (got %d)", n); return 2; }
    if (n == 0) return 0;
    if (!parents || !children || !aligned(parents, 4) || !aligned(children, 4)) { set_error("pages_fork: parents or children is null or not aligned"); return 2; }
    if (int rc = check_workspace("pages_fork", p, workspace, workspace_bytes)) return rc;
    const void* const mem[] = {p.refs, p.pages, p.kv_len, c.k, parents, children, workspace};
    if (int rc = check_memory("pages_fork", mem, 7)) return rc;
    int* at = static_cast<int*>(workspace);
    ForkArgs a{device_pool(p), parents, children, n};
    a.list = at; at += words(p.num_pages + 2);
    for (int** q : {&a.claim, &a.keys, &a.rank, &a.src, &a.dst, &a.rest}) { *q = at; at += words(p.num_seqs); }
    a.count = at;
    EFA_CUDA(launch_value(pages_fork_kernel, dim3(1, 1, blocks_of(p, n)), PG_THREADS, 0, stream, a));
    return launch_moves(move_args(c, a.src, a.dst, a.rest, a.count, n, SITE_FORK, a.p.status), nullptr, stream);
}

int pages_free(const efa_page_pool& p, const int* seqs, int n, cudaStream_t stream)
{
    if (const char* why = page_pool_check(p)) { set_error("pages_free: %s", why); return 2; }
    if (n < 0 || n > 1 << 24) { set_error("pages_free: n must be from 0 to 2^24 (got %d)", n); return 2; }
    if (n == 0) return 0;
    if (!seqs || !aligned(seqs, 4)) { set_error("pages_free: seqs is null or not aligned"); return 2; }
    const void* const mem[] = {p.refs, p.pages, p.kv_len, seqs};
    if (int rc = check_memory("pages_free", mem, 4)) return rc;
    EFA_CUDA(launch_value(pages_free_kernel, dim3(n), PG_FREE_THREADS, 0, stream, device_pool(p), seqs));
    return 0;
}

int pages_compact(const efa_page_pool& p, const efa_paged_cache& c, int* pages_out, int* refs_out, int* moved, void* workspace, size_t workspace_bytes, cudaStream_t stream)
{
    if (const char* why = page_pool_check(p)) { set_error("pages_compact: %s", why); return 2; }
    if (const char* why = check_cache(c, &p)) { set_error("pages_compact: %s", why); return 2; }
    if (!refs_out || !moved || (!pages_out && p.num_seqs > 0)) { set_error("pages_compact: pages_out, refs_out or moved is null"); return 2; }
    if (!aligned(pages_out, 4) || !aligned(refs_out, 4) || !aligned(moved, 4)) { set_error("pages_compact: arrays must be aligned to their numbers"); return 2; }
    if (int rc = check_workspace("pages_compact", p, workspace, workspace_bytes)) return rc;
    const void* const mem[] = {p.refs, p.pages, p.kv_len, c.k, pages_out, refs_out, moved, workspace};
    if (int rc = check_memory("pages_compact", mem, 8)) return rc;
    const int half = p.num_pages / 2 + 1;                      // no more pages can move than there are free ones before L
    int* const at = static_cast<int*>(workspace);
    const CompactArgs a{device_pool(p), pages_out, refs_out, moved, at, at + half, at + words(p.num_pages + 2)};
    EFA_CUDA(launch_value(pages_compact_kernel, dim3(1, 1, blocks_of(p, 0)), PG_THREADS, 0, stream, a));
    return launch_moves(move_args(c, a.from, a.to, nullptr, a.count, half, SITE_COMPACT, a.p.status), &a, stream);
}

int pages_copy(const efa_paged_cache& c, const int* src, const int* dst, int n, cudaStream_t stream)
{
    if (const char* why = check_cache(c, nullptr)) { set_error("pages_copy: %s", why); return 2; }
    if (n < 0 || n > c.num_pages) { set_error("pages_copy: n must be from 0 to the number of pages (got %d)", n); return 2; }
    if (n == 0) return 0;
    if (!src || !dst || !aligned(src, 4) || !aligned(dst, 4)) { set_error("pages_copy: src or dst is null or not aligned"); return 2; }
    const void* const mem[] = {c.k, src, dst};
    if (int rc = check_memory("pages_copy", mem, 3)) return rc;
    return launch_moves(move_args(c, src, dst, nullptr, nullptr, n, SITE_COPY, kernel_status_word()), nullptr, stream);
}

}  // namespace efa
