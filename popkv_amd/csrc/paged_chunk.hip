// Attention of a chunk of new tokens a sequence over its paged 4-bit cache and,
// causally, over the chunk itself: how a call is cut, and its launches.
#include "kernels.h"
#include "popkv_hip.h"

namespace popkv {

hipError_t launch_paged_chunk_bf16(const PagedChunk& a, const PagedView& c, int64_t max_tokens, int dim_group,
                                   hipStream_t stream);
hipError_t launch_paged_chunk_f16(const PagedChunk& a, const PagedView& c, int64_t max_tokens, int dim_group,
                                  hipStream_t stream);
hipError_t launch_paged_chunk_f32(const PagedChunk& a, const PagedView& c, int64_t max_tokens, int dim_group,
                                  hipStream_t stream);

namespace {

constexpr int kChunkCus = 256;
// Fewest tiles of a workgroup, and what a block of rows costs beside its tiles: its
// queries, first reads, state or output.  us by the fewest tiles, 1, 2, 4, 8: a
// verification of 6 tokens behind 2000 19.7, 18.0, 21.0, 27.9, eight of up to 8201 33.8,
// 33.9, 33.6, 39.4, small ragged fp32 chunks 40.5, 40.5, 44.2, 57.0; longer calls the same.
// By the cost, 0, 1, 2, 4, 8: the eight verifications 36.9, 34.8, 33.7, 34.0, 33.7, 16
// decode steps with weights 69.4, 63.7, 62.6, 65.3, 70.6, 64 verifications behind up to 900
// 41.0, 37.4, 37.7, 40.2, 40.1, six ragged fp16 prompts 668, 641, 594, 539, 545.
constexpr int kLeastTiles = 4, kBlockCost = 2;
int64_t ceil_of(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace

// As many rows a workgroup as there are, up to 256 (fp32 128: two terms of everything
// fill its registers), which share a tile's dequantisation.  Two workgroups a CU where
// their LDS allows it (eight verifications of 6 tokens behind up to 8201 38 us, with one a
// CU 40), and no more than fit at once (the first pass of 16 decode steps with weights,
// whose LDS holds one, 41 us, in two rounds 51).
ChunkPlan paged_chunk_plan(int dtype, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t rows, int64_t max_tokens,
                           bool weights) {
    ChunkPlan p{};
    const bool f32 = dtype == POPKV_DTYPE_F32;
    const int64_t all = rows * (q_heads / kv_heads);
    p.shape = all <= 32 && !f32 ? 1 : all <= 64 ? 2 : all <= 128 || f32 ? 4 : 8;
    p.row_blocks = ceil_of(all, 32 * p.shape);
    p.least = kLeastTiles;
    p.item_cost = kBlockCost;
    const bool alone = p.shape == 8 || f32 || (p.shape == 1 && (weights || dtype != POPKV_DTYPE_BF16));
    const int64_t tile = p.shape == 1 ? 128 : 64;
    const int64_t tiles = ceil_of(max_tokens, tile) + ceil_of(rows, tile) + p.item_cost;
    const int64_t target = ceil_of(kChunkCus * (alone ? 1 : 2), kv_heads);
    const int64_t most = ceil_of(batch * p.row_blocks * tiles, p.least);
    p.groups = static_cast<int>(most < target ? most : target);
    p.states = p.groups > 1 ? 2 * static_cast<int64_t>(p.groups) * kv_heads * p.shape * (32 * 128 + 64) : 0;
    p.stored = f32 ? kChunkStored32 : kChunkStored16;
    p.places = batch * p.row_blocks * tiles;
    return p;
}

hipError_t launch_paged_chunk(const PagedChunk& a, const PagedView& c, int64_t max_tokens, int dtype, int dim_group,
                              hipStream_t stream) {
    switch (dtype) {
        case POPKV_DTYPE_F32: return launch_paged_chunk_f32(a, c, max_tokens, dim_group, stream);
        case POPKV_DTYPE_F16: return launch_paged_chunk_f16(a, c, max_tokens, dim_group, stream);
        default: return launch_paged_chunk_bf16(a, c, max_tokens, dim_group, stream);
    }
}

}  // namespace popkv
