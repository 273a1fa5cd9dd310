// Attention whose scores are biased by distance, or whose rows see a prefix: the kernels of
// exl3_attn_few.hpp and exl3_attn_many.hpp with kEarly (exl3_attn.hpp says what it adds).
#include <hip/hip_runtime.h>

#include "exl3_attn_launch.hpp"

namespace exl3 {

EXL3_FEW(EXL3_FEW_INST, kEarly)
EXL3_MANY(EXL3_MANY_INST, kEarly)

#ifndef __HIP_DEVICE_COMPILE__
void launch_attention_early(const AttnParams& p, const AttnShape& sh, hipStream_t s) {
  launch_attention<kEarly>(p, sh, s);
}
#endif

}  // namespace exl3
