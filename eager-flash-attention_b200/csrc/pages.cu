// The pages of a paged cache: taken, shared, given back, moved. All of it goes by device memory: the host knows the sizes only.
//
// Which pages are free is a scan over their counts. One cluster of eight blocks does it, a segment of the pages to each block: counts per block, exchanged
// through the cluster's shared memory, then ranks within the segment; so the lowest free pages are found in one launch, in an order that nothing but the arrays
// decides. What moves keys is a kernel of its own over all SMs.
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
__device__ __forceinline__ int keys_of(const PoolArgs& p, int b, int site)
{
    const int kv = p.kv_len[b];
    const int cut = (int)min(max((long long)kv, 0ll), min(capacity(p), (long long)INT_MAX));
    if (cut != kv) report(p.status, KS_BAD_LENGTH, b, site);
    return cut;
}
__device__ __forceinline__ int pages_of(const PoolArgs& p, int keys) { return (int)(((long long)keys + p.page_size - 1) / p.page_size); }

// Sum over the block; `part` [PG_WARPS] in shared memory.
__device__ __forceinline__ int block_sum(int v, int* part)
{
    #pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = part[threadIdx.x & 31];
    #pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}

// Sum of the values of the threads before this one, and of all of them in `total`.
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

// Sums over the cluster: of what the blocks before this one, and all of them, put into `mine` (shared memory, one word a block).
__device__ __forceinline__ int cluster_scan(int v, int* mine, int& total)
{
    if (threadIdx.x == 0) *mine = v;
    cluster_sync();
    int before = 0;
    total = 0;
    const int rank = (int)cluster_rank();
    #pragma unroll
    for (int q = 0; q < PG_CLUSTER; q++) {
        int x;
        asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(x) : "r"(cluster_addr(mine, q)));
        before += q < rank ? x : 0;
        total += x;
    }
    return before;
}

struct Range { int lo, hi; };
__device__ __forceinline__ Range segment(int n)
{
    const int each = (n + PG_CLUSTER - 1) / PG_CLUSTER, lo = min(n, each * (int)cluster_rank());
    return Range{lo, min(n, lo + each)};
}

// Free pages [lo, hi) get their ranks among all free pages; those below `wanted` go into list[rank] and get a count of 1.
__device__ __forceinline__ int count_free(const int* refs, Range r, int* part)
{
    int n = 0;
    for (int p = r.lo + (int)threadIdx.x; p < r.hi; p += PG_THREADS) n += refs[p] <= 0 ? 1 : 0;
    return block_sum(n, part);
}
__device__ __forceinline__ void list_free(int* refs, Range r, int before, int wanted, int* list, int* part)
{
    for (int base = r.lo; base < r.hi && before < wanted; base += PG_THREADS) {
        const int p = base + (int)threadIdx.x;
        const int free = p < r.hi && refs[p] <= 0 ? 1 : 0;
        int total;
        const int rank = before + block_scan(free, part, total);
        if (free && rank < wanted) { list[rank] = p; refs[p] = 1; }
        before += total;
    }
}

// workspace: list [num_pages], then what the kernels say of it.
struct TakeArgs { PoolArgs p; const int* q_start; int* list; };

__global__ void __launch_bounds__(PG_THREADS)
pages_take_kernel(const TakeArgs a)
{
    __shared__ int part[PG_WARPS], mine[2];
    __shared__ int3 todo[PG_THREADS];
    pdl_wait();
    pdl_trigger();
    const PoolArgs& p = a.p;
    const Range seqs = segment(p.num_seqs), own = segment(p.num_pages);

    // A slot's new length, and the pages that it has and wants.
    auto grown = [&](int b, int& have, int& want) {
        const int kv = keys_of(p, b, SITE_TAKE);
        const long long n = (long long)a.q_start[b + 1] - a.q_start[b];
        const long long after = min((long long)kv + max(n, 0ll), min(capacity(p), (long long)INT_MAX));
        if (n < 0 || after != kv + n) report(p.status, KS_BAD_LENGTH, b, SITE_TAKE);
        have = pages_of(p, kv);
        want = pages_of(p, (int)after);
        return (int)after;
    };
    int need = 0;
    for (int b = seqs.lo + (int)threadIdx.x; b < seqs.hi; b += PG_THREADS) {
        int have, want;
        grown(b, have, want);
        need += want - have;
    }
    need = block_sum(need, part);
    int wanted, there;
    int first = cluster_scan(need, &mine[0], wanted);
    const int before = cluster_scan(count_free(p.refs, own, part), &mine[1], there);
    list_free(p.refs, own, before, wanted, a.list, part);
    cluster_sync();
    for (int base = seqs.lo; base < seqs.hi; base += PG_THREADS) {
        const int b = base + (int)threadIdx.x;
        int have = 0, want = 0, after = 0, total;
        if (b < seqs.hi) after = grown(b, have, want);
        const int rank = first + block_scan(want - have, part, total);
        todo[threadIdx.x] = make_int3(have, want, rank);
        __syncthreads();
        for (int i = threadIdx.x >> 5; i < PG_THREADS; i += PG_WARPS) {
            const int3 d = todo[i];
            for (int e = d.x + (int)(threadIdx.x & 31); e < d.y; e += 32) {
                const int r = d.z + e - d.x;
                p.pages[(long long)(base + i) * p.max_pages + e] = r < there ? a.list[r] : -1;
                if (r >= there) report(p.status, KS_NO_PAGE, base + i, SITE_TAKE);
            }
        }
        __syncthreads();
        if (b < seqs.hi) p.kv_len[b] = after;
        first += total;
    }
}

// Moves: pairs of pages, whole (keys NULL) or their first keys[i] keys. count: on the device, or NULL for n of them.
struct MoveArgs {
    uint8_t* part[4];           // k, v, k_exp, v_exp
    long long stride[4];        // bytes from a page to the next
    int head_bytes[4];          // bytes of a head of a page
    int key_bytes[4];
    int heads, num_pages;
    const int* src;
    const int* dst;
    const int* keys;
    const int* count;
    int n, site;
    int* status;
};

// workspace of a fork: list [num_pages], then [num_seqs] each of claim, keys of the child, rank of its page, and the moves: source, target, keys; then their count.
struct ForkArgs { PoolArgs p; const int* parents; const int* children; int n; int* list; int* claim; int* keys; int* rank; int* src; int* dst; int* rest; int* count; };

__global__ void __launch_bounds__(PG_THREADS)
pages_fork_kernel(const ForkArgs a)
{
    __shared__ int part[PG_WARPS], mine[2];
    pdl_wait();
    pdl_trigger();
    const PoolArgs& p = a.p;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Range forks = segment(a.n), own = segment(p.num_pages);
    auto slot = [&](int b) { return (unsigned)b < (unsigned)p.num_seqs; };

    // The first entry that names a child has it.
    for (int i = forks.lo + (int)threadIdx.x; i < forks.hi; i += PG_THREADS)
        if (slot(a.children[i])) a.claim[a.children[i]] = INT_MAX;
    cluster_sync();
    for (int i = forks.lo + (int)threadIdx.x; i < forks.hi; i += PG_THREADS)
        if (slot(a.children[i])) atomicMin(&a.claim[a.children[i]], i);
    cluster_sync();
    int need = 0;
    for (int i = forks.lo + (int)threadIdx.x; i < forks.hi; i += PG_THREADS) {
        const int c = a.children[i], b = a.parents[i];
        int keys = -1;
        if (!slot(c) || !slot(b) || a.claim[c] != i || p.kv_len[c] != 0) report(p.status, KS_BAD_SLOT, slot(c) ? c : i, SITE_FORK);
        else {
            keys = keys_of(p, b, SITE_FORK);
            if (keys % p.page_size) {
                const int source = p.pages[(long long)b * p.max_pages + keys / p.page_size];
                if ((unsigned)source < (unsigned)p.num_pages) need++;
                else report(p.status, KS_BAD_PAGE, b, SITE_FORK);
            }
        }
        a.keys[i] = keys;
    }
    need = block_sum(need, part);
    int wanted, there;
    int first = cluster_scan(need, &mine[0], wanted);
    const int before = cluster_scan(count_free(p.refs, own, part), &mine[1], there);
    list_free(p.refs, own, before, wanted, a.list, part);
    if (cluster_rank() == 0 && threadIdx.x == 0) *a.count = min(wanted, there);
    // Ranks of the children's pages.
    for (int base = forks.lo; base < forks.hi; base += PG_THREADS) {
        const int i = base + (int)threadIdx.x;
        int wants = 0, total;
        if (i < forks.hi && a.keys[i] > 0 && a.keys[i] % p.page_size) {
            const int source = p.pages[(long long)a.parents[i] * p.max_pages + a.keys[i] / p.page_size];
            wants = (unsigned)source < (unsigned)p.num_pages ? 1 : 0;
        }
        const int rank = first + block_scan(wants, part, total);
        if (i < forks.hi) a.rank[i] = wants ? rank : -1;
        first += total;
    }
    cluster_sync();
    for (int i = forks.lo + warp; i < forks.hi; i += PG_WARPS) {
        const int keys = a.keys[i];
        if (keys < 0) continue;
        const int c = a.children[i], full = keys / p.page_size, rank = a.rank[i];
        const int* const from = p.pages + (long long)a.parents[i] * p.max_pages;
        int* const to = p.pages + (long long)c * p.max_pages;
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
                to[full] = got ? a.list[rank] : -1;
                if (got) {
                    a.src[rank] = from[full];
                    a.dst[rank] = a.list[rank];
                    a.rest[rank] = keys % p.page_size;
                } else if (rank >= 0) report(p.status, KS_NO_PAGE, c, SITE_FORK);
            }
            p.kv_len[c] = keys;
        }
    }
}

__global__ void __launch_bounds__(256)
pages_free_kernel(const PoolArgs p, const int* seqs, int n)
{
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, i = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (i >= n) return;
    const int b = seqs[i];
    if ((unsigned)b >= (unsigned)p.num_seqs) {
        if (lane == 0) report(p.status, KS_BAD_SLOT, i, SITE_FREE);
        return;
    }
    int keys = 0;
    if (lane == 0) keys = atomicExch(&p.kv_len[b], 0);         // whoever names the slot again finds it empty
    keys = __shfl_sync(0xffffffffu, keys, 0);
    const int cut = (int)min(max((long long)keys, 0ll), min(capacity(p), (long long)INT_MAX));
    if (cut != keys && lane == 0) report(p.status, KS_BAD_LENGTH, b, SITE_FREE);
    const int held = pages_of(p, cut);
    for (int e = lane; e < held; e += 32) {
        const int page = p.pages[(long long)b * p.max_pages + e];
        if ((unsigned)page >= (unsigned)p.num_pages) {
            if (page != -1) report(p.status, KS_BAD_PAGE, b, SITE_FREE);     // -1: there was no page to be had
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
    const Range own = segment(p.num_pages);
    int n = own.hi - own.lo - count_free(p.refs, own, part), live;
    int before = cluster_scan(n, &mine[0], live);
    n = 0;
    for (int q = own.lo + (int)threadIdx.x; q < min(own.hi, live); q += PG_THREADS) n += p.refs[q] > 0 ? 1 : 0;
    int stay;                                                  // pages in use before L
    cluster_scan(block_sum(n, part), &mine[1], stay);
    for (int base = own.lo; base < own.hi; base += PG_THREADS) {
        const int q = base + (int)threadIdx.x;
        const bool used = q < own.hi && p.refs[q] > 0;
        int total;
        const int rank = before + block_scan(used ? 1 : 0, part, total);       // pages in use before q
        if (q < own.hi) {
            if (used && q >= live) a.from[rank - stay] = q;
            else a.moved[q] = used ? q : -1;
            if (!used && q < live) a.to[q - rank] = q;
        }
        before += total;
    }
    cluster_sync();
    if (cluster_rank() == 0 && threadIdx.x == 0) *a.count = live - stay;
    for (int i = (int)cluster_rank() * PG_THREADS + threadIdx.x; i < live - stay; i += PG_CLUSTER * PG_THREADS) a.moved[a.from[i]] = a.to[i];
}

// The table and the counts of the pool after the moves.
__global__ void __launch_bounds__(256)
pages_rename_kernel(const CompactArgs a)
{
    pdl_wait();
    pdl_trigger();
    const PoolArgs& p = a.p;
    const int lane = threadIdx.x & 31, warps = gridDim.x * 8, warp = blockIdx.x * 8 + (threadIdx.x >> 5);
    for (int b = warp; b < p.num_seqs; b += warps) {
        const int held = pages_of(p, keys_of(p, b, SITE_COMPACT));
        for (int e = lane; e < held; e += 32) {
            const long long at = (long long)b * p.max_pages + e;
            const int page = p.pages[at], to = (unsigned)page < (unsigned)p.num_pages ? a.moved[page] : -1;
            if (to < 0 && page != -1) report(p.status, KS_BAD_PAGE, b, SITE_COMPACT);
            a.pages_out[at] = to;
        }
    }
    // A place before L that was free is written by the page that moves there, every other by itself.
    const int moves = *a.count;
    for (int q = warp * 32 + lane; q < p.num_pages; q += warps * 32) {
        const int to = a.moved[q], n = p.refs[q];
        if (to == q) a.refs_out[q] = n;
        else if (to >= 0) { a.refs_out[to] = n; a.refs_out[q] = 0; }
        else if (moves == 0 || q > a.to[moves - 1]) a.refs_out[q] = 0;      // behind the last free place that is filled
    }
}

__global__ void __launch_bounds__(PG_MOVE_THREADS)
pages_move_kernel(const MoveArgs a, int segments /* of a page's k */, int exp_segments)
{
    pdl_wait();
    pdl_trigger();
    const int n = a.count ? min(*a.count, a.n) : a.n;
    const int per_page = 2 * (segments + exp_segments);
    for (long long item = blockIdx.x; item < (long long)n * per_page; item += gridDim.x) {
        const int i = (int)(item / per_page);
        int s = (int)(item % per_page);
        const int src = a.src[i], dst = a.dst[i];
        if ((unsigned)src >= (unsigned)a.num_pages || (unsigned)dst >= (unsigned)a.num_pages) {
            if (threadIdx.x == 0 && s == 0) report(a.status, KS_BAD_PAGE, i, a.site);
            continue;
        }
        const bool exps = s >= 2 * segments;
        if (exps) s -= 2 * segments;
        const int per = exps ? exp_segments : segments, what = (exps ? 2 : 0) + s / per;
        s %= per;
        long long at, bytes;
        if (a.keys) {                                          // a head's first keys
            at = (long long)s * a.head_bytes[what];
            bytes = (long long)a.keys[i] * a.key_bytes[what];
        } else {
            const long long all = (long long)a.heads * a.head_bytes[what];
            at = (long long)s * PG_SEGMENT;
            bytes = min((long long)PG_SEGMENT, all - at);
        }
        const uint8_t* const from = a.part[what] + src * a.stride[what] + at;
        uint8_t* const to = a.part[what] + dst * a.stride[what] + at;
        const int chunks = (int)(bytes / 16);
        int c = threadIdx.x;
        for (; c + 7 * PG_MOVE_THREADS < chunks; c += 8 * PG_MOVE_THREADS) {
            uint4 v[8];
            #pragma unroll
            for (int j = 0; j < 8; j++) v[j] = reinterpret_cast<const uint4*>(from)[c + j * PG_MOVE_THREADS];
            #pragma unroll
            for (int j = 0; j < 8; j++) reinterpret_cast<uint4*>(to)[c + j * PG_MOVE_THREADS] = v[j];
        }
        for (; c < chunks; c += PG_MOVE_THREADS) reinterpret_cast<uint4*>(to)[c] = reinterpret_cast<const uint4*>(from)[c];
        for (long long b = (long long)chunks * 16 + threadIdx.x; b < bytes; b += PG_MOVE_THREADS) to[b] = from[b];
    }
}

int launch_moves(const efa_paged_cache& c, const int* src, const int* dst, const int* keys, const int* count, int n, int site, int* status, cudaStream_t stream)
{
    MoveArgs a{};
    const int elem = c.dtype == EFA_F16 ? 2 : 1;
    const long long dense = (long long)c.H_kv * c.page_size * c.d_h;
    a.part[0] = static_cast<uint8_t*>(c.k); a.part[1] = static_cast<uint8_t*>(c.v);
    a.part[2] = c.k_exp; a.part[3] = c.v_exp;
    for (int i = 0; i < 4; i++) {
        a.key_bytes[i] = i < 2 ? c.d_h * elem : 1;
        a.head_bytes[i] = a.key_bytes[i] * c.page_size;
        a.stride[i] = i < 2 ? (c.page_stride ? c.page_stride : dense) * elem : (long long)c.H_kv * c.page_size;
    }
    a.heads = c.H_kv; a.num_pages = c.num_pages;
    a.src = src; a.dst = dst; a.keys = keys; a.count = count;
    a.n = n; a.site = site; a.status = status;
    const auto pieces = [&](int i) { return keys ? c.H_kv : (int)(((long long)c.H_kv * a.head_bytes[i] + PG_SEGMENT - 1) / PG_SEGMENT); };
    const int segments = pieces(0), exp_segments = c.dtype == EFA_E4M3 ? pieces(2) : 0;
    const long long items = (long long)n * 2 * (segments + exp_segments);
    const unsigned blocks = (unsigned)std::min<long long>(items, 8ll * device_sms());
    EFA_CUDA(launch_value(pages_move_kernel, dim3(blocks), PG_MOVE_THREADS, 0, stream, a, segments, exp_segments));
    return 0;
}

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
    if (p.num_pages > 1 << 30 || p.num_seqs > 1 << 30 || (long long)p.num_seqs * p.max_pages > INT_MAX) return "pages: sizes too large";
    return nullptr;
}

size_t pages_bytes(const efa_page_pool& p) { return 4 * (words(p.num_pages + 2) + 6 * words(p.num_seqs) + 4); }

int pages_take(const efa_page_pool& p, const int* q_start, void* workspace, size_t workspace_bytes, cudaStream_t stream)
{
    if (const char* why = page_pool_check(p)) { set_error("pages_take: %s", why); return 2; }
    if (p.num_seqs == 0) return 0;
    if (!q_start) { set_error("pages_take: q_start is null"); return 2; }
    if (int rc = check_workspace("pages_take", p, workspace, workspace_bytes)) return rc;
    const void* const mem[] = {p.refs, p.pages, p.kv_len, q_start, workspace};
    if (int rc = check_memory("pages_take", mem, 5)) return rc;
    const TakeArgs a{device_pool(p), q_start, static_cast<int*>(workspace)};
    EFA_CUDA(launch_value(pages_take_kernel, dim3(1, 1, PG_CLUSTER), PG_THREADS, 0, stream, a));
    return 0;
}

int pages_fork(const efa_page_pool& p, const efa_paged_cache& c, const int* parents, const int* children, int n, void* workspace, size_t workspace_bytes, cudaStream_t stream)
{
    if (const char* why = page_pool_check(p)) { set_error("pages_fork: %s", why); return 2; }
    if (const char* why = check_cache(c, &p)) { set_error("pages_fork: %s", why); return 2; }
    if (n < 0 || n > p.num_seqs) { set_error("pages_fork: n must be from 0 to the number of slots (got %d)", n); return 2; }
    if (n == 0) return 0;
    if (!parents || !children) { set_error("pages_fork: parents or children is null"); return 2; }
    if (int rc = check_workspace("pages_fork", p, workspace, workspace_bytes)) return rc;
    const void* const mem[] = {p.refs, p.pages, p.kv_len, c.k, parents, children, workspace};
    if (int rc = check_memory("pages_fork", mem, 7)) return rc;
    int* at = static_cast<int*>(workspace);
    ForkArgs a{device_pool(p), parents, children, n};
    a.list = at; at += words(p.num_pages + 2);
    for (int** q : {&a.claim, &a.keys, &a.rank, &a.src, &a.dst, &a.rest}) { *q = at; at += words(p.num_seqs); }
    a.count = at;
    EFA_CUDA(launch_value(pages_fork_kernel, dim3(1, 1, PG_CLUSTER), PG_THREADS, 0, stream, a));
    return launch_moves(c, a.src, a.dst, a.rest, a.count, n, SITE_FORK, a.p.status, stream);
}

int pages_free(const efa_page_pool& p, const int* seqs, int n, cudaStream_t stream)
{
    if (const char* why = page_pool_check(p)) { set_error("pages_free: %s", why); return 2; }
    if (n < 0 || n > 1 << 24) { set_error("pages_free: n must be from 0 to 2^24 (got %d)", n); return 2; }
    if (n == 0) return 0;
    if (!seqs) { set_error("pages_free: seqs is null"); return 2; }
    const void* const mem[] = {p.refs, p.pages, p.kv_len, seqs};
    if (int rc = check_memory("pages_free", mem, 4)) return rc;
    EFA_CUDA(launch_value(pages_free_kernel, dim3((n + 7) / 8), 256, 0, stream, device_pool(p), seqs, n));
    return 0;
}

int pages_compact(const efa_page_pool& p, const efa_paged_cache& c, int* pages_out, int* refs_out, int* moved, void* workspace, size_t workspace_bytes, cudaStream_t stream)
{
    if (const char* why = page_pool_check(p)) { set_error("pages_compact: %s", why); return 2; }
    if (const char* why = check_cache(c, &p)) { set_error("pages_compact: %s", why); return 2; }
    if (!refs_out || !moved || (!pages_out && p.num_seqs > 0)) { set_error("pages_compact: pages_out, refs_out or moved is null"); return 2; }
    if (int rc = check_workspace("pages_compact", p, workspace, workspace_bytes)) return rc;
    const void* const mem[] = {p.refs, p.pages, p.kv_len, c.k, pages_out, refs_out, moved, workspace};
    if (int rc = check_memory("pages_compact", mem, 8)) return rc;
    const int half = p.num_pages / 2 + 1;                      // no more pages can move than there are free ones before L
    int* const at = static_cast<int*>(workspace);
    const CompactArgs a{device_pool(p), pages_out, refs_out, moved, at, at + half, at + words(p.num_pages + 2)};
    EFA_CUDA(launch_value(pages_compact_kernel, dim3(1, 1, PG_CLUSTER), PG_THREADS, 0, stream, a));
    const int work = std::max(p.num_seqs, (p.num_pages + 31) / 32);
    EFA_CUDA(launch_value(pages_rename_kernel, dim3(std::min((work + 7) / 8, 2 * device_sms())), 256, 0, stream, a));
    return launch_moves(c, a.from, a.to, nullptr, a.count, half, SITE_COMPACT, a.p.status, stream);
}

int pages_copy(const efa_paged_cache& c, const int* src, const int* dst, int n, cudaStream_t stream)
{
    if (const char* why = check_cache(c, nullptr)) { set_error("pages_copy: %s", why); return 2; }
    if (n < 0 || n > c.num_pages) { set_error("pages_copy: n must be from 0 to the number of pages (got %d)", n); return 2; }
    if (n == 0) return 0;
    if (!src || !dst) { set_error("pages_copy: src or dst is null"); return 2; }
    const void* const mem[] = {c.k, src, dst};
    if (int rc = check_memory("pages_copy", mem, 3)) return rc;
    return launch_moves(c, src, dst, nullptr, nullptr, n, SITE_COPY, kernel_status_word(), stream);
}

}  // namespace efa
