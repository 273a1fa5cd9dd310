// Attention whose scores are capped by a tanh, biased by distance or not: the kernels of
// exl3_attn_few.hpp and exl3_attn_many.hpp with kCapped and kBoth (exl3_attn.hpp says what they add).
#include <hip/hip_runtime.h>

#include "exl3_attn_launch.hpp"

namespace exl3 {

EXL3_FEW(EXL3_FEW_INST, kCapped)
EXL3_MANY(EXL3_MANY_INST, kCapped)
EXL3_MANY(EXL3_MANY_INST, kBoth)

#ifndef __HIP_DEVICE_COMPILE__
void launch_attention_capped(const AttnParams& p, const AttnShape& sh, bool both, hipStream_t s) {
  both ? launch_attention<kBoth>(p, sh, s) : launch_attention<kCapped>(p, sh, s);
}
#endif

}  // namespace exl3
