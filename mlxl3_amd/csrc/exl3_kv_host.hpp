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

}  // namespace exl3
