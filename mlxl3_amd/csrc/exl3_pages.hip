// Pages of the paged cache copied (layout: exl3_kv.hpp): forked sequences' last pages, pools
// that are compacted.
//
// One launch copies up to 224 pairs of pages in up to 32 caches of one shape -- a model's layers --
// named in the kernel's arguments, so that nothing is uploaded.  Where a pair copies its first
// n slots only, a head's n slots are one run of its page (its scales n of every group's run).
// Memory bounds it: every byte is read and written once, 16 at a time.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <new>
#include <vector>

#include "../../include/exl3_hip.h"
#include "exl3_kv.hpp"
#include "exl3_kv_host.hpp"
#include "exl3_launch.hpp"

namespace exl3 {

constexpr int kMostCaches = 32, kMostPairs = 224;  // of a launch: 3.8 KB of arguments, of 4 that it takes
constexpr int kUnits = 1024;                       // 16-byte units of a workgroup, four a thread

struct CopyParams {
  uint8_t* keys[kMostCaches];
  uint8_t* values[kMostCaches];
  uint16_t* key_scales[kMostCaches];
  uint16_t* value_scales[kMostCaches];
  int32_t src[kMostPairs], dst[kMostPairs];
  uint16_t slots[kMostPairs];
  int page_shift, kv_heads, row, groups;  // row: bytes of a cached head; groups: of scales, 0 without
};

// A run of `runs` pieces of `length` 16-byte units, `pitch` units apart, copied by 256 threads from
// unit `first` on.
__device__ __forceinline__ void copy_units(const u32x4* from, u32x4* to, int runs, int length, int pitch, int first) {
  const int n = runs * length;
  u32x4 v[4];
  int at[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t u = first + i * 256 + threadIdx.x;
    at[i] = -1;
    if (u >= (uint32_t)n) continue;
    at[i] = length == pitch ? u : u / (uint32_t)length * pitch + u % (uint32_t)length;
    v[i] = from[at[i]];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (at[i] >= 0) to[at[i]] = v[i];
}

// grid (parts of a page, pairs, caches x sides): the parts of the codes, behind them those of the scales
__global__ __launch_bounds__(256) void kv_copy_kernel(CopyParams p, int parts) {
  const int pair = blockIdx.y, cache = blockIdx.z >> 1, part = blockIdx.x;
  const bool value = blockIdx.z & 1;
  const int page = 1 << p.page_shift, slots = p.slots[pair];
  const int64_t src = p.src[pair], dst = p.dst[pair];
  if (part < parts) {
    const int units = p.row / 16;  // of a slot
    uint8_t* pool = value ? p.values[cache] : p.keys[cache];
    const size_t bytes = (size_t)p.kv_heads * page * p.row;
    copy_units((const u32x4*)(pool + src * bytes), (u32x4*)(pool + dst * bytes), p.kv_heads, slots * units,
               page * units, part * kUnits);
    return;
  }
  uint16_t* pool = value ? p.value_scales[cache] : p.key_scales[cache];
  const int runs = p.kv_heads * p.groups;
  const uint16_t* from = pool + src * ((int64_t)runs << p.page_shift);
  uint16_t* to = pool + dst * ((int64_t)runs << p.page_shift);
  const int first = (part - parts) * kUnits;
  if (slots == page) {
    copy_units((const u32x4*)from, (u32x4*)to, runs, page / 8, page / 8, first);
    return;
  }
  // eight slots at a time, the last ones of a run one by one
  const uint32_t pieces = (slots + 7) / 8;
  for (int i = 0; i < 4; ++i) {
    const uint32_t u = first + i * 256 + threadIdx.x;
    if (u >= runs * pieces) return;
    const int run = u / pieces, slot = u % pieces * 8, at = (run << p.page_shift) + slot;
    if (slot + 8 <= slots) {
      *(u32x4*)(to + at) = *(const u32x4*)(from + at);
    } else {
      for (int e = 0; e < slots - slot; ++e) to[at + e] = from[at + e];
    }
  }
}

}  // namespace exl3

using namespace exl3;

#ifndef __HIP_DEVICE_COMPILE__

static_assert(sizeof(CopyParams) + 16 <= 4096, "a launch takes 4 KB of arguments");

// What a copy of pages refuses, before anything is launched: every page is in all pools, none is
// written twice or written and read.
static int check_copy(const exl3_kv_cache* const* caches, int32_t count, const int32_t* src, const int32_t* dst,
                      const int32_t* slots, int64_t pairs) {
  if (!caches || count < 1) return fail(EXL3_EINVAL, "a copy of pages needs at least one KV cache");
  for (int i = 0; i < count; ++i)
    if (!caches[i]) return fail(EXL3_EINVAL, "null KV cache");
  const KvCacheView& c = caches[0]->view;
  for (int i = 1; i < count; ++i)
    if (caches[i]->view.pages != c.pages || caches[i]->view.page_shift != c.page_shift)
      return fail(EXL3_EINVAL, "KV caches whose pages are copied together have as many pages of as many tokens");
  if (pairs < 0) return fail(EXL3_EINVAL, "negative page count");
  if (pairs == 0) return EXL3_OK;
  if (!src || !dst) return fail(EXL3_EINVAL, "null page list");
  if (pairs > c.pages)
    return fail(EXL3_EINVAL, "%lld copies among %lld pages", (long long)pairs, (long long)c.pages);
  for (int64_t i = 0; i < pairs; ++i) {
    for (const int32_t page : {src[i], dst[i]})
      if (page < 0 || page >= c.pages)
        return fail(EXL3_EINVAL, "page %d of a pool of %lld", page, (long long)c.pages);
    if (slots && (slots[i] < 0 || slots[i] > 1 << c.page_shift))
      return fail(EXL3_EINVAL, "%d slots of a page of %d", slots[i], 1 << c.page_shift);
  }
  auto clash = [&](const int32_t* from, const int32_t* to) {  // sorted
    for (int64_t i = 1; i < pairs; ++i)
      if (to[i] == to[i - 1]) return fail(EXL3_EINVAL, "page %d is copied to twice", to[i]);
    for (int64_t i = 0, j = 0; i < pairs && j < pairs;) {
      if (from[i] == to[j]) return fail(EXL3_EINVAL, "page %d is copied and copied to", to[j]);
      from[i] < to[j] ? ++i : ++j;
    }
    return (int)EXL3_OK;
  };
  constexpr int kFew = 64;
  if (pairs <= kFew) {
    int32_t from[kFew], to[kFew];
    std::copy(src, src + pairs, from);
    std::copy(dst, dst + pairs, to);
    std::sort(from, from + pairs);
    std::sort(to, to + pairs);
    return clash(from, to);
  }
  try {
    std::vector<int32_t> from(src, src + pairs), to(dst, dst + pairs);
    std::sort(from.begin(), from.end());
    std::sort(to.begin(), to.end());
    return clash(from.data(), to.data());
  } catch (const std::bad_alloc&) {
    return fail(EXL3_ENOMEM, "out of host memory");
  }
}

extern "C" int exl3_kv_copy_pages(const exl3_kv_cache* const* caches, int32_t count, const int32_t* src,
                                  const int32_t* dst, const int32_t* slots, int64_t pairs, void* stream) {
  if (int rc = check_copy(caches, count, src, dst, slots, pairs)) return rc;
  if (pairs == 0) return EXL3_OK;
  auto alike = [](const KvCacheView& a, const KvCacheView& b) {
    return a.format == b.format && a.kv_heads == b.kv_heads && a.head_dim == b.head_dim;
  };
  if (int rc = launch_gate("KV page copy")) return rc;
  CopyParams p;
  for (int first = 0; first < count; ++first) {
    // the caches of one shape together, where its first one stands
    const KvCacheView& c = caches[first]->view;
    bool seen = false;
    for (int i = 0; i < first && !seen; ++i) seen = alike(caches[i]->view, c);
    if (seen) continue;
    const bool coded = c.format == EXL3_KV_Q8 || c.format == EXL3_KV_Q4;
    p.page_shift = c.page_shift;
    p.kv_heads = c.kv_heads;
    p.row = c.format == EXL3_KV_Q4 ? c.head_dim / 2 : c.format == EXL3_KV_Q8 ? c.head_dim : 2 * c.head_dim;
    p.groups = coded ? c.head_dim / 32 : 0;
    for (int next = first; next < count;) {
      int n = 0;
      for (; next < count && n < kMostCaches; ++next) {
        const KvCacheView& v = caches[next]->view;
        if (!alike(v, c)) continue;
        p.keys[n] = v.k;
        p.values[n] = v.v;
        p.key_scales[n] = v.ks;
        p.value_scales[n++] = v.vs;
      }
      if (n == 0) break;
      for (int64_t at = 0; at < pairs;) {
        int m = 0, most = 0;
        for (; at < pairs && m < kMostPairs; ++at) {
          const int filled = slots ? slots[at] : 1 << c.page_shift;
          if (filled == 0) continue;
          p.src[m] = src[at];
          p.dst[m] = dst[at];
          p.slots[m++] = (uint16_t)filled;
          most = std::max(most, filled);
        }
        if (m == 0) continue;
        const int parts = (most * p.kv_heads * (p.row / 16) + kUnits - 1) / kUnits;
        const int more = (p.kv_heads * p.groups * ((most + 7) / 8) + kUnits - 1) / kUnits;
        hipLaunchKernelGGL(kv_copy_kernel, dim3((unsigned)(parts + more), (unsigned)m, 2u * (unsigned)n), dim3(256), 0,
                           (hipStream_t)stream, p, parts);
        if (int rc = check_launch("KV page copy")) return rc;
      }
    }
  }
  return EXL3_OK;
}

#endif  // __HIP_DEVICE_COMPILE__
