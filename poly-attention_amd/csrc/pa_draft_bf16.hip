// pa_draft_bf16.hip -- k_draft_partial for bf16 (a source file of its own: compile time).
#include "pa_draft_partial.h"

namespace pa {
template void launch_draft_partial<bf16>(const DraftDev& P, int units, int tiles, bool vmul, hipStream_t s);
}  // namespace pa
