// pa_paged_f32.hip -- attention over a paged cache, f32.
#include "pa_paged_rows.h"

namespace pa {
template void launch_paged_rows<float>(const PagedDev& P, const PagedDev& B, int64_t units, int joins, int clear, int tiles, hipStream_t s);
}  // namespace pa
