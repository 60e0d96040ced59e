// Many queries per request, mlops_paged_attend.
#include "paged_tile.cuh"

namespace paged {
PAGED_TILE(CAUSAL);
}  // namespace paged
