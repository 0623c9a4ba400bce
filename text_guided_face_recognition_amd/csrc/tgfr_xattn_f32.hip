// The f32 kernels of cross attention (tgfr_xattn.h).
#include "tgfr_xattn.h"

namespace tgfr {
int xattn_run_f32(const XArgs& a, int what, void* stream) {
  return a.D % 4 ? x_by_width<XF32Any>(a, what, stream) : x_by_width<XF32>(a, what, stream);
}
}  // namespace tgfr
