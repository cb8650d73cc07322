// kernels_paged_chunk_f16.hip — attention of long chunks over the paged cache, rows of f16
// (paged_chunk.hpp).
#include "paged_chunk.hpp"

namespace kivi {

template hipError_t launch_paged_chunk<_Float16>(const PagedAttention&, const ChunkPlan&, float*, hipStream_t);

}  // namespace kivi
