// Launch arguments of the attention kernels over the paged cache, and their launchers.
#pragma once

#include "host_util.h"
#include "paged_args.cuh"

namespace efa {

struct PagedAttnArgs {
    const __half* Q;
    __half* O;
    long long q_head, q_token, o_token;     // strides in elements
    float scale_log2e, rescale_above;       // log2 units by which a maximum may outgrow the exponent offset in use
    PagedShape w;
    PagedParts parts;                       // all null: nothing is cut, one block per item
};

// mma.sync over tiles of up to 64 rows (paged_rows_sm100.cu).
int paged_rows_tile(int rows);              // rows of a tile for chunks of up to `rows` rows (tokens x heads of a group)
constexpr int PAGED_ROWS_EXTRA = 1;
int paged_rows_unit(bool f8);               // keys of a unit
int paged_rows_blocks_per_sm(int d_h, bool f8);
// blocks: items, or shares; cluster: blocks that share an item (items only).
int paged_rows_launch(const PagedArgs& c, const PagedAttnArgs& a, int d_h, bool f8, int blocks, int cluster, cudaStream_t stream);

// tcgen05 over tiles of 256 rows (paged_chunk.cuh); blocks: items, or shares.
constexpr int PAGED_CHUNK_TILE = 256, PAGED_CHUNK_UNIT = 128, PAGED_CHUNK_EXTRA = 3;
int paged_chunk_launch(const PagedArgs& c, const PagedAttnArgs& a, int d_h, bool f8, int blocks, cudaStream_t stream);

// Merge of the items that the cuts of `blocks` parts go through.
int paged_merge_launch(const PagedArgs& c, const PagedAttnArgs& a, int d_h, int blocks, int most_rows, cudaStream_t stream);

// A launch like launch_early's (host_util.h) of a kernel whose name the caller has as a value. grid.z: a cluster's blocks.
template <class... P, class... A>
cudaError_t paged_launch(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t stream, const A&... args)
{
    return launch_kernel(true, (int)grid.z, kernel, grid, threads, smem, stream, args...);
}

}  // namespace efa
