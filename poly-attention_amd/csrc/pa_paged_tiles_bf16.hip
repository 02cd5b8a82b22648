// pa_paged_tiles_bf16.hip -- attention over a paged cache, chunks of many rows, bf16.
#include "pa_paged_tiles.h"

namespace pa {
template void launch_paged_tiles<bf16>(const PagedDev& P, int64_t units, hipStream_t s);
}  // namespace pa
