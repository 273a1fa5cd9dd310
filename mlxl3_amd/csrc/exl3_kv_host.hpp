// Host side shared by the cache's and attention's entry points.
#pragma once

#include "../../include/exl3_hip.h"
#include "exl3_kv.hpp"

struct exl3_kv_cache {
  exl3::KvCacheView view;
};

namespace exl3 {

// Workgroups of 256 lanes that one dimension of a launch takes (2^32 lanes).
constexpr int64_t kMostBlocks = (1 << 24) - 1;

bool aligned16(const void* p);

// Checks a batch (its block table only with a cache) and fills the kernels' view.
int check_batch(const exl3_kv_cache* cache, const exl3_kv_batch* batch, int64_t tokens,
                KvBatchView* view);

// exl3_rope and exl3_kv_append; without `launch` all their checks alone, for a call that is
// made of several and refuses before its first launch.
int rope_call(const exl3_rope_spec* rope, const void* x, int32_t x_type, int64_t tokens,
              int32_t heads, int32_t head_dim, int64_t x_stride, const int32_t* positions,
              const exl3_kv_batch* batch, void* y, int32_t y_type, int64_t y_stride, void* stream,
              bool launch);
int append_call(const exl3_kv_cache* cache, const exl3_kv_batch* batch, const void* k,
                int64_t k_stride, const void* v, int64_t v_stride, int32_t type, int64_t tokens,
                const exl3_rope_spec* rope, void* stream, bool launch);

}  // namespace exl3
