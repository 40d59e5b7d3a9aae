// hipcc-flags: -Xclang -target-feature -Xclang -packed-fp32-ops
// Shaped attention, forward: the bf16 instances (one file each: they compile in parallel).
#include "attn_shaped_fwd.h"

extern "C" int tfk_shaped_fwd_bf16(const void* p, float* ws, hipStream_t s, int D) {
  return D == 64 ? launch_fwd<bf16, 64>(*(const Shaped*)p, ws, s) : launch_fwd<bf16, 128>(*(const Shaped*)p, ws, s);
}
