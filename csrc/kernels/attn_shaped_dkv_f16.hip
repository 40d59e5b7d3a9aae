// hipcc-flags: -Xclang -target-feature -Xclang -packed-fp32-ops
// Shaped attention, dK/dV pass: the f16 instances (one file each: they compile in parallel).
#include "attn_shaped_bwd.h"

extern "C" int tfk_shaped_dkv_f16(const void* p, float* ws, hipStream_t s, int D) {
  return D == 64 ? launch_dkv<f16, 64>(*(const Shaped*)p, ws, s) : launch_dkv<f16, 128>(*(const Shaped*)p, ws, s);
}
