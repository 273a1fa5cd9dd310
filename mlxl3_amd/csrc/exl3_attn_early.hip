// Attention whose scores are biased by distance, or whose rows see a prefix: the kernels of
// exl3_attn_few.hpp and exl3_attn_many.hpp with kEarly and kSeen (exl3_attn.hpp says what they add).
#include <hip/hip_runtime.h>

#include "exl3_attn_launch.hpp"

namespace exl3 {

EXL3_FEW(EXL3_FEW_INST, kEarly)
EXL3_MANY(EXL3_MANY_INST, kEarly)
EXL3_MANY(EXL3_MANY_INST, kSeen)

#ifndef __HIP_DEVICE_COMPILE__
void launch_attention_early(const AttnParams& p, const AttnShape& sh, bool seen, hipStream_t s) {
  seen ? launch_attention<kSeen>(p, sh, s) : launch_attention<kEarly>(p, sh, s);
}
#endif

}  // namespace exl3
