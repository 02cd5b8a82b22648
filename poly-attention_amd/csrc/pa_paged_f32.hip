// pa_paged_f32.hip -- attention over a paged cache, f32.
#include "pa_paged_rows.h"

namespace pa {
template void launch_paged_rows<float>(const PagedDev& P, int64_t units, int clear, int tiles, hipStream_t s);
}  // namespace pa
