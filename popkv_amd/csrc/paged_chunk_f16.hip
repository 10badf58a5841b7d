// The chunk attention's kernels in fp16.
#include "paged_chunk.h"

namespace popkv {

hipError_t launch_paged_chunk_f16(const PagedChunk& a, const PagedView& c, int64_t max_tokens, int dim_group,
                                 hipStream_t stream) {
    return launch_chunk<f16_t>(a, c, max_tokens, dim_group, stream);
}

}  // namespace popkv
