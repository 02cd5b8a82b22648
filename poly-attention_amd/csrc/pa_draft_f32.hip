// pa_draft_f32.hip -- k_draft_partial for f32 (a source file of its own: compile time).
#include "pa_draft_partial.h"

namespace pa {
template void launch_draft_partial<float>(const DraftDev& P, int units, int tiles, bool vmul, hipStream_t s);
}  // namespace pa
