// pa_draft_bf16.hip -- k_draft_partial and k_draft_wide for bf16 (a source file of its own: compile time).
#include "pa_draft_wide.h"

namespace pa {
template void launch_draft_partial<bf16>(const DraftDev& P, int units, int tiles, bool vmul, hipStream_t s);
template void launch_draft_wide<bf16>(const DraftDev& P, int units, bool vmul, hipStream_t s);
}  // namespace pa
