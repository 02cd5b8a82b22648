// pa_paged_bf16.hip -- attention over a paged cache, bf16.
#include "pa_paged_rows.h"

namespace pa {
template void launch_paged_rows<bf16>(const PagedDev& P, const PagedDev& B, int64_t units, int joins, int clear, int tiles, hipStream_t s);
}  // namespace pa
