// Few queries per request, mlops_paged_attend_shared.
#include "paged_stream.cuh"

namespace paged {
PAGED_STREAM(SHARED);
}  // namespace paged
