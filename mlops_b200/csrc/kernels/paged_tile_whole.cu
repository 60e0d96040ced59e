// Many queries per request, mlops_paged_cross_attend.
#include "paged_tile.cuh"

namespace paged {
PAGED_TILE(WHOLE);
}  // namespace paged
