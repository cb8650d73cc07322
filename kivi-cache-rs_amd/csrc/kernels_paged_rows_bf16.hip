// kernels_paged_rows_bf16.hip — attention of few rows over the paged cache, rows of bf16
// (paged_rows.hpp).
#include "paged_rows.hpp"

namespace kivi {

template hipError_t launch_paged_rows<__bf16, false>(const PagedAttention&, const RowsPlan&, float*, hipStream_t);

}  // namespace kivi
