// Many queries per request, mlops_paged_attend_shared.
#include "paged_tile.cuh"

namespace paged {
PAGED_TILE(SHARED);
}  // namespace paged
