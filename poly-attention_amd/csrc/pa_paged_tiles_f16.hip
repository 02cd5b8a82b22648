// pa_paged_tiles_f16.hip -- attention over a paged cache, chunks of many rows, f16.
#include "pa_paged_tiles.h"

namespace pa {
template void launch_paged_tiles<f16>(const PagedDev& P, int64_t units, hipStream_t s);
}  // namespace pa
