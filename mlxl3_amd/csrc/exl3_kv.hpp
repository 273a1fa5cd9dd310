// The paged key/value cache as kernels see it, and what its kernels share:
// locating a token's page, moving eight values of a head, the codes of 8- and
// 4-bit caches.
//
// Layout (keys and values alike): pages of P tokens, P a power of two,
//   16-bit   [pages][kv_heads][P][D] of f16 or bf16
//   8-bit    [pages][kv_heads][P][D] bytes, code + 128
//   4-bit    [pages][kv_heads][P][D/2] bytes, code + 8 of channel 2i in the low half
//   scales   [pages][kv_heads][D/32][P] f16 (8- and 4-bit): value = code * scale
// A head's P tokens are contiguous, so a tile of 16 tokens is one run of 16 * D values.
// Scales lie token-fastest: the lanes of a matrix operand that hold successive tokens
// of one group of channels read their scales as one vector.
#pragma once

#include "exl3_device.hpp"

namespace exl3 {

enum : int { KV_Q4 = 4, KV_Q8 = 8, KV_F16 = DT_F16, KV_BF16 = DT_BF16 };

struct KvCacheView {
  uint8_t *k, *v;
  uint16_t *ks, *vs;  // null for 16-bit formats
  int64_t pages;
  int page_shift, kv_heads, head_dim, format;
};

struct KvBatchView {
  const int32_t* q_starts;  // [seqs + 1]
  const int32_t* kv_lens;   // [seqs]
  const int32_t* table;     // [seqs][table_pages]
  int seqs, table_pages;
};

// Bytes of n cached values.
__device__ __forceinline__ size_t kv_bytes(int format, size_t n) {
  return format == KV_Q8 ? n : format == KV_Q4 ? n >> 1 : n * 2;
}

// The page of position pos of sequence seq, or -1 where the table or the pool
// has none (the table is device data that the host does not read).
__device__ __forceinline__ int64_t kv_page(const KvCacheView& c, const KvBatchView& b, int seq,
                                           int64_t pos) {
  if (pos < 0 || (pos >> c.page_shift) >= b.table_pages) return -1;
  const int32_t page = b.table[(int64_t)seq * b.table_pages + (pos >> c.page_shift)];
  return page >= 0 && page < c.pages ? page : -1;
}

// The sequence that token row `token` belongs to (the last one that starts at or
// before it; empty sequences share their start with the next), or -1 behind the last.
__device__ __forceinline__ int kv_sequence(const KvBatchView& b, int64_t token) {
  if (token < b.q_starts[0] || token >= b.q_starts[b.seqs]) return -1;
  int lo = 0, hi = b.seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (b.q_starts[mid] <= token)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// Position of token row `token` of sequence seq: the new tokens are its last ones.
__device__ __forceinline__ int64_t kv_position(const KvBatchView& b, int seq, int64_t token) {
  return (int64_t)b.kv_lens[seq] - (int64_t)b.q_starts[seq + 1] + token;
}

// ---------------------------------------------------------------------------
// eight values
// ---------------------------------------------------------------------------
__device__ __forceinline__ float load1(const void* p, int dt, size_t i) {
  return dt == DT_F32 ? ((const float*)p)[i]
                      : dt == DT_F16 ? h2f(((const uint16_t*)p)[i]) : bf2f(((const uint16_t*)p)[i]);
}
__device__ __forceinline__ void store1(void* p, int dt, size_t i, float v) {
  if (dt == DT_F32)
    ((float*)p)[i] = v;
  else
    ((uint16_t*)p)[i] = dt == DT_F16 ? f2h(v) : f2bf(v);
}

// vec: the eight values are 16-byte aligned.
__device__ __forceinline__ void load8(const void* p, int dt, size_t i, bool vec, float (&x)[8]) {
  if (!vec) {
#pragma unroll
    for (int e = 0; e < 8; ++e) { x[e] = load1(p, dt, i + e); }
  } else if (dt == DT_F32) {
    const float4v a = *(const float4v*)((const float*)p + i);
    const float4v b = *(const float4v*)((const float*)p + i + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) { x[e] = a[e]; x[e + 4] = b[e]; }
  } else {
    const u32x4 w = *(const u32x4*)((const uint16_t*)p + i);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint16_t h = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
      x[e] = dt == DT_F16 ? h2f(h) : bf2f(h);
    }
  }
}
__device__ __forceinline__ void store8(void* p, int dt, size_t i, bool vec, const float (&x)[8]) {
  if (!vec) {
#pragma unroll
    for (int e = 0; e < 8; ++e) { store1(p, dt, i + e, x[e]); }
  } else if (dt == DT_F32) {
    float4v a, b;
#pragma unroll
    for (int e = 0; e < 4; ++e) { a[e] = x[e]; b[e] = x[e + 4]; }
    *(float4v*)((float*)p + i) = a;
    *(float4v*)((float*)p + i + 4) = b;
  } else {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint16_t lo = dt == DT_F16 ? f2h(x[2 * e]) : f2bf(x[2 * e]);
      const uint16_t hi = dt == DT_F16 ? f2h(x[2 * e + 1]) : f2bf(x[2 * e + 1]);
      w[e] = (uint32_t)lo | ((uint32_t)hi << 16);
    }
    *(u32x4*)((uint16_t*)p + i) = w;
  }
}

// Eight cached values as floats: `row` is the head's row of D values, d0 the first
// channel (a multiple of 8), `scale` its group's (8- and 4-bit formats).
__device__ __forceinline__ void kv_load8(const uint8_t* row, int format, int d0, float scale,
                                         float (&x)[8]) {
  if (format == KV_Q8) {
    const u32x2 w = *(const u32x2*)(row + d0);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = (float)((int)((w[e / 4] >> (8 * (e & 3))) & 255) - 128) * scale;
    }
  } else if (format == KV_Q4) {
    const uint32_t w = *(const uint32_t*)(row + d0 / 2);
#pragma unroll
    for (int e = 0; e < 8; ++e) { x[e] = (float)((int)((w >> (4 * e)) & 15) - 8) * scale; }
  } else {
    load8(row, format, (size_t)d0, true, x);
  }
}

}  // namespace exl3
