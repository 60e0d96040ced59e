// Few queries per request, mlops_paged_cross_attend.
#include "paged_stream.cuh"

namespace paged {
PAGED_STREAM(WHOLE);
}  // namespace paged
