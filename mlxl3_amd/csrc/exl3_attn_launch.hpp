// Attention's kernels by format, width and rows: their instances, spelled out for the device
// pass, and their launches.  S: scores that are capped or biased, or rows that see a prefix: translation
// units of their own.
#pragma once

#include "exl3_attn_few.hpp"
#include "exl3_attn_many.hpp"

namespace exl3 {

struct AttnShape {
  bool few;       // attn_few_kernel, else attn_many_kernel
  int rows;       // rows of a workgroup
  bool one_tile;  // every sequence's rows fit one workgroup
  int64_t tiles;  // at most; the device counts the tiles that there are
  int splits;     // even ranges of the tokens that a tile sees
  int budget;     // else ranges by the batch's sum, about (as AttnParams')
  int64_t slots;  // of partial results to join, `rows` rows each
};

#define EXL3_FEW_D(M, FMT, T, PARTS, S)                                                  \
  M(FMT, T, 64, 1, PARTS, S) M(FMT, T, 64, 2, PARTS, S) M(FMT, T, 128, 1, PARTS, S)      \
  M(FMT, T, 128, 2, PARTS, S) M(FMT, T, 256, 1, PARTS, S)
#define EXL3_FEW(M, S)                                                                   \
  EXL3_FEW_D(M, KV_F16, F16, 1, S) EXL3_FEW_D(M, KV_BF16, BF16, 1, S) EXL3_FEW_D(M, KV_Q8, F16, 1, S) \
  EXL3_FEW_D(M, KV_Q8, F16, 2, S) EXL3_FEW_D(M, KV_Q4, F16, 1, S) EXL3_FEW_D(M, KV_Q4, F16, 2, S)
#define EXL3_FEW_INST(FMT, T, D, RT, PARTS, S) \
  template __global__ void attn_few_kernel<FMT, T, D, RT, PARTS, S>(AttnParams);

#define EXL3_MANY_D(M, FMT, T, PARTS, S) M(FMT, T, 64, PARTS, S) M(FMT, T, 128, PARTS, S) M(FMT, T, 256, PARTS, S)
#define EXL3_MANY(M, S)                                                                  \
  EXL3_MANY_D(M, KV_F16, F16, 1, S) EXL3_MANY_D(M, KV_BF16, BF16, 1, S) EXL3_MANY_D(M, KV_Q8, F16, 1, S) \
  EXL3_MANY_D(M, KV_Q8, F16, 2, S) EXL3_MANY_D(M, KV_Q4, F16, 1, S) EXL3_MANY_D(M, KV_Q4, F16, 2, S)
#define EXL3_MANY_INST(FMT, T, D, PARTS, S) \
  template __global__ void attn_many_kernel<FMT, T, D, PARTS, S>(AttnParams, int);

#ifndef __HIP_DEVICE_COMPILE__

template <int S, int FMT, typename T, int PARTS, int D, int RT>
void launch_few(const AttnParams& p, hipStream_t s) {
  const dim3 grid = p.budget ? dim3((unsigned)p.cache.kv_heads, (unsigned)(p.budget + p.batch.seqs + 1))
                             : dim3((unsigned)p.cache.kv_heads, (unsigned)p.splits, (unsigned)p.batch.seqs);
  constexpr size_t lds = 4 * (Few<FMT, T, D, RT, PARTS>::kWaveLds);
  hipLaunchKernelGGL((attn_few_kernel<FMT, T, D, RT, PARTS, S>), grid, dim3(256), lds, s, p);
}
template <int S, int FMT, typename T, int PARTS>
void launch_few(const AttnParams& p, int rows, hipStream_t s) {
  const int d = p.cache.head_dim;
  if (rows == 16) {
    d == 64 ? launch_few<S, FMT, T, PARTS, 64, 1>(p, s) : d == 128 ? launch_few<S, FMT, T, PARTS, 128, 1>(p, s)
                                                                : launch_few<S, FMT, T, PARTS, 256, 1>(p, s);
  } else {
    d == 64 ? launch_few<S, FMT, T, PARTS, 64, 2>(p, s) : launch_few<S, FMT, T, PARTS, 128, 2>(p, s);
  }
}

template <int S, int FMT, typename T, int PARTS, int D>
void launch_many(const AttnParams& p, int tiles, hipStream_t s) {
  constexpr size_t lds = Many<FMT, T, D, PARTS>::kLds;
  const dim3 grid((unsigned)tiles * p.splits * p.cache.kv_heads);
  hipLaunchKernelGGL((attn_many_kernel<FMT, T, D, PARTS, S>), grid, dim3(256), lds, s, p, tiles);
}
template <int S, int FMT, typename T, int PARTS>
void launch(const AttnParams& p, const AttnShape& sh, hipStream_t s) {
  const int d = p.cache.head_dim, tiles = (int)sh.tiles;
  if (sh.few)
    launch_few<S == kSeen ? kEarly : S == kBoth ? kCapped : S, FMT, T, PARTS>(p, sh.rows, s);
  else
    d == 64 ? launch_many<S, FMT, T, PARTS, 64>(p, tiles, s) : d == 128 ? launch_many<S, FMT, T, PARTS, 128>(p, tiles, s)
                                                                     : launch_many<S, FMT, T, PARTS, 256>(p, tiles, s);
}

// The kernel of a call by the cache's format and the queries' type (f16 ones: coded values in two parts).
template <int S>
void launch_attention(const AttnParams& p, const AttnShape& sh, hipStream_t s) {
  const bool fine = p.q_type == DT_F16;
  switch (p.cache.format) {
    case KV_F16: launch<S, KV_F16, F16, 1>(p, sh, s); break;
    case KV_BF16: launch<S, KV_BF16, BF16, 1>(p, sh, s); break;
    case KV_Q8: fine ? launch<S, KV_Q8, F16, 2>(p, sh, s) : launch<S, KV_Q8, F16, 1>(p, sh, s); break;
    default: fine ? launch<S, KV_Q4, F16, 2>(p, sh, s) : launch<S, KV_Q4, F16, 1>(p, sh, s);
  }
}

#endif  // __HIP_DEVICE_COMPILE__

// launch_attention<kEarly> and <kSeen>, <kCapped> and <kBoth>, <kLate>, of the other translation units.
void launch_attention_early(const AttnParams& p, const AttnShape& sh, bool seen, hipStream_t s);
void launch_attention_capped(const AttnParams& p, const AttnShape& sh, bool both, hipStream_t s);
void launch_attention_late(const AttnParams& p, const AttnShape& sh, hipStream_t s);

}  // namespace exl3
