// hipcc-flags: -Xclang -target-feature -Xclang -packed-fp32-ops
// Shaped attention, dQ pass: the f16 instances (one file each: they compile in parallel).
#include "attn_shaped_bwd.h"

extern "C" int tfk_shaped_dq_f16(const void* p, hipStream_t s, int D) {
  return D == 64 ? launch_dq<f16, 64>(*(const Shaped*)p, s) : launch_dq<f16, 128>(*(const Shaped*)p, s);
}
