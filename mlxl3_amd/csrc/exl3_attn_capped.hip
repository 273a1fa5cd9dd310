// Attention whose scores are capped by a tanh, biased by distance or not: the kernels of
// exl3_attn_few.hpp and exl3_attn_many.hpp with kCapped (exl3_attn.hpp says what it adds).
#include <hip/hip_runtime.h>

#include "exl3_attn_launch.hpp"

namespace exl3 {

EXL3_FEW(EXL3_FEW_INST, kCapped)
EXL3_MANY(EXL3_MANY_INST, kCapped)

#ifndef __HIP_DEVICE_COMPILE__
void launch_attention_capped(const AttnParams& p, const AttnShape& sh, hipStream_t s) {
  launch_attention<kCapped>(p, sh, s);
}
#endif

}  // namespace exl3
