// Pages of the paged cache copied (layout: exl3_kv.hpp): forked sequences' last pages, pools
// that are compacted.
//
// One launch copies some 200 to 400 pairs of pages in up to 64 caches of one shape -- a model's
// layers -- named in the kernel's arguments, so that nothing is uploaded.  Where a pair copies its first
// n slots only, a head's n slots are one run of its page (its scales n of every group's run).
// Memory bounds it: every byte is read and written once, 16 at a time.  Measured, sources not in the
// caches: 230 pages of 131 KB in 4 caches, 121 MB, 47 us, 5.1 TB/s read and written (a large copy: 5.1);
// 48 partly filled 8-bit pages in 16 caches, 27 MB, 19 us (in the caches 11); one page's 9 slots in 32
// caches 3.7 us, a launch and one round trip.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <new>
#include <vector>

#include "../../include/exl3_hip.h"
#include "exl3_kv.hpp"
#include "exl3_kv_host.hpp"
#include "exl3_launch.hpp"

namespace exl3 {

constexpr int kWords = 504;      // of their pools and the pairs: 4 KB of arguments, as many as a launch takes
constexpr int kUnits = 1024;     // 16-byte units of a workgroup, four a thread

struct CopyParams {
  // the pools of every cache (keys, values and, where there are groups, the scales of both), the pages of
  // every pair (low half: copied, high half: copied to), the slots of every pair, four a word
  uint64_t words[kWords];
  int page_shift, kv_heads, row, groups;  // row: bytes of a cached head; groups: of scales, 0 without
  int caches, parts;                      // parts: workgroups of a page's codes
};

// Pools are named by numbers, so that their memory has to be called global (else the compiler's accesses
// wait for LDS too).
typedef __attribute__((address_space(1))) u32x4 Unit;
typedef __attribute__((address_space(1))) uint16_t Scale;
// STREAM: past the caches (copies that they do not hold).
template <bool STREAM>
__device__ __forceinline__ u32x4 read16(const Unit* p) {
  return STREAM ? __builtin_nontemporal_load(p) : *p;
}
template <bool STREAM>
__device__ __forceinline__ void write16(Unit* p, u32x4 v) {
  if constexpr (STREAM)
    __builtin_nontemporal_store(v, p);
  else
    *p = v;
}

// n / d for n below 2^22 and d up to 1024, by a multiplication: inv is 2^32 / d rounded up, off by less
// than 1, the quotient by less than n 2^-32 < 1 / d.  (2^32 / 1 is past 32 bits: d of 1 is no division.)
struct Divisor {
  uint32_t d, inv;
  __device__ __forceinline__ explicit Divisor(uint32_t v) : d(v), inv(0xffffffffu / v + 1) {}
  __device__ __forceinline__ uint32_t quotient(uint32_t n) const { return d == 1 ? n : __umulhi(n, inv); }
};

// grid (parts of a page, pairs, caches x sides): the parts of the codes, behind them those of the scales
// (in workgroups of their own: 48 forks in 16 8-bit caches 19 us, with the codes' ones 24).  A thread
// has four 16-byte units, all loaded before the first is stored.
template <bool STREAM>
__global__ __launch_bounds__(256) void kv_copy_kernel(CopyParams p) {
  const int pair = blockIdx.y, cache = blockIdx.z >> 1, side = blockIdx.z & 1;
  const int pools = p.groups ? 4 : 2, pages_at = p.caches * pools, slots_at = pages_at + gridDim.y;
  const uint32_t page = 1u << p.page_shift, slots = (uint32_t)(p.words[slots_at + pair / 4] >> (16 * (pair % 4))) & 0xffff;
  const uint64_t pages = p.words[pages_at + pair];
  const int64_t src = (uint32_t)pages, dst = pages >> 32;
  if ((int)blockIdx.x < p.parts) {
    // codes: the runs of all heads, `slots` slots each of 2^shift units, `page` slots apart
    const int shift = __builtin_ctz(p.row) - 4;
    const uint32_t units = (p.kv_heads * slots) << shift, first = blockIdx.x * kUnits + threadIdx.x;
    const int64_t whole = ((int64_t)p.kv_heads * page) << shift;
    Unit* pool = (Unit*)p.words[cache * pools + side];
    const Unit* from = pool + src * whole;
    Unit* to = pool + dst * whole;
    const Divisor by(slots);
    u32x4 v[4];
    uint32_t at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = first + i * 256;
      at[i] = u + ((by.quotient(u >> shift) * (page - slots)) << shift);
      if (u < units) v[i] = read16<STREAM>(from + at[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (first + i * 256 < units) write16<STREAM>(to + at[i], v[i]);
    return;
  }
  // scales: the runs of all groups, eight slots at a time, the last ones of a run one by one
  Scale* pool = (Scale*)p.words[cache * pools + 2 + side];
  const uint32_t runs = p.kv_heads * p.groups, pieces = (slots + 7) / 8;
  const Scale* from = pool + ((src * runs) << p.page_shift);
  Scale* to = pool + ((dst * runs) << p.page_shift);
  const Divisor by(pieces);
  for (int i = 0; i < 4; ++i) {
    const uint32_t u = (blockIdx.x - p.parts) * kUnits + i * 256 + threadIdx.x;
    if (u >= runs * pieces) return;
    const uint32_t run = by.quotient(u), slot = (u - run * pieces) * 8, at = (run << p.page_shift) + slot;
    if (slot + 8 <= slots) {
      write16<STREAM>((Unit*)(to + at), read16<STREAM>((const Unit*)(from + at)));
    } else {
      for (uint32_t e = 0; e < slots - slot; ++e) to[at + e] = from[at + e];
    }
  }
}
template __global__ void kv_copy_kernel<false>(CopyParams);
template __global__ void kv_copy_kernel<true>(CopyParams);

}  // namespace exl3

using namespace exl3;

#ifndef __HIP_DEVICE_COMPILE__

constexpr int kMostCaches = 64;  // of a launch: keys and values of each are a grid's z
constexpr double kCached = 64.0 * 1048576;  // bytes copied beyond which a copy goes past the caches

static_assert(sizeof(CopyParams) <= 4096, "a launch takes 4 KB of arguments");

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
  // Copies of more than 64 MB -- with their source half of what the caches hold -- go past them.  Cold, us, 16-bit pages of
  // four caches: 31 MB 14.3 past them, 18.5 through them; 63 MB 25.7, 30.8; 121 MB 47, 58.  But source and
  // copy are read again soon where a sequence is forked: 48 forks in 16 caches and the attention of all
  // layers after them 162 past them, 150 through them.
  double bytes = 0.0;
  for (int i = 0; i < count; ++i) {
    const KvCacheView& v = caches[i]->view;
    bytes += 2.0 * v.kv_heads * v.head_dim * (v.format == EXL3_KV_Q4 ? 0.5 : v.format == EXL3_KV_Q8 ? 1.0 : 2.0);
  }
  int64_t filled = 0;
  for (int64_t i = 0; i < pairs; ++i) filled += slots ? slots[i] : 1 << caches[0]->view.page_shift;
  const bool stream_past = bytes * filled > kCached;
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
        uint64_t* pools = p.words + (coded ? 4 : 2) * n++;
        pools[0] = (uintptr_t)v.k;
        pools[1] = (uintptr_t)v.v;
        if (coded) {
          pools[2] = (uintptr_t)v.ks;
          pools[3] = (uintptr_t)v.vs;
        }
      }
      if (n == 0) break;
      p.caches = n;
      uint64_t* words = p.words + (coded ? 4 : 2) * n;
      const int room = (int)(p.words + kWords - words) * 4 / 5;
      for (int64_t at = 0; at < pairs;) {
        uint16_t filled_slots[kWords];
        int m = 0, most = 0;
        for (; at < pairs && m < room; ++at) {
          const int used = slots ? slots[at] : 1 << c.page_shift;
          if (used == 0) continue;
          words[m] = (uint64_t)(uint32_t)src[at] | (uint64_t)(uint32_t)dst[at] << 32;
          filled_slots[m++] = (uint16_t)used;
          most = std::max(most, used);
        }
        if (m == 0) continue;
        for (int i = 0; i < m; ++i) {
          uint64_t& four = words[m + i / 4];
          four = (i % 4 ? four : 0) | (uint64_t)filled_slots[i] << (16 * (i % 4));
        }
        const int codes = most * p.kv_heads * (p.row / 16), scales = p.kv_heads * p.groups * ((most + 7) / 8);
        p.parts = (codes + kUnits - 1) / kUnits;
        const dim3 grid((unsigned)(p.parts + (scales + kUnits - 1) / kUnits), (unsigned)m, 2u * (unsigned)n);
        if (stream_past)
          hipLaunchKernelGGL(kv_copy_kernel<true>, grid, dim3(256), 0, (hipStream_t)stream, p);
        else
          hipLaunchKernelGGL(kv_copy_kernel<false>, grid, dim3(256), 0, (hipStream_t)stream, p);
        if (int rc = check_launch("KV page copy")) return rc;
      }
    }
  }
  return EXL3_OK;
}

#endif  // __HIP_DEVICE_COMPILE__
