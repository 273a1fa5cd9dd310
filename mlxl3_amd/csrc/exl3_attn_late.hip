// Attention with caps above 256 and with factors whose quotients may leave f32's range: the kernels of
// exl3_attn_few.hpp and exl3_attn_many.hpp with kLate (exl3_attn.hpp says what it adds).
#include <hip/hip_runtime.h>

#include "exl3_attn_launch.hpp"

namespace exl3 {

EXL3_FEW(EXL3_FEW_INST, kLate)
EXL3_MANY(EXL3_MANY_INST, kLate)

#ifndef __HIP_DEVICE_COMPILE__
void launch_attention_late(const AttnParams& p, const AttnShape& sh, hipStream_t s) {
  launch_attention<kLate>(p, sh, s);
}
#endif

}  // namespace exl3
