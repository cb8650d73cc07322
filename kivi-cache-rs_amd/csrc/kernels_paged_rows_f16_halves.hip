// kernels_paged_rows_f16_halves.hip — attention of few rows over the paged cache, rows of f16, groups of an odd multiple of 16
// (paged_rows.hpp).
#include "paged_rows.hpp"

namespace kivi {

template hipError_t launch_paged_rows<_Float16, true>(const PagedAttention&, const RowsPlan&, float*, hipStream_t);

}  // namespace kivi
