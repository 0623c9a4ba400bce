// The bf16 kernels of cross attention (tgfr_xattn.h).
#include "tgfr_xattn.h"

namespace tgfr {
int xattn_run_bf16(const XArgs& a, int what, void* stream) {
  return x_by_width<XBf16>(a, what, stream);
}
}  // namespace tgfr
