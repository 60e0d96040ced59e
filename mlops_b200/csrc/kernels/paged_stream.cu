// Few queries per request, mlops_paged_attend.
#include "paged_stream.cuh"

namespace paged {
PAGED_STREAM(CAUSAL);
}  // namespace paged
