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

// Where token rows belong: a row's sequence (the first that ends behind it; -1 in front of
// the first or behind the last) and its position there, the new tokens being the sequence's
// last ones.
struct KvToken {
  int seq;
  int64_t pos;
};
// Of the `count` successive rows from `first` on, the lane's row `mine`.  The whole wave calls
// it, first and count the same in all lanes: the lanes look at 64 sequences at a time, for
// all rows that end there.
__device__ __forceinline__ KvToken kv_locate(const KvBatchView& b, int64_t first, int count, int mine) {
  const int lane = threadIdx.x & 63, start = b.q_starts[0];
  KvToken r{-1, 0};
  int i = 0;
  for (int s0 = 0; s0 < b.seqs && i < count; s0 += 64) {
    const int at = min(s0 + lane, b.seqs - 1);
    const int end = b.q_starts[at + 1], len = b.kv_lens[at];
    for (; i < count; ++i) {
      const int64_t token = first + i;
      const int n = __popcll(__ballot(s0 + lane < b.seqs && end <= token));
      if (n == 64 || s0 + n >= b.seqs) break;
      const int64_t pos = (int64_t)__builtin_amdgcn_readlane(len, n) - __builtin_amdgcn_readlane(end, n) + token;
      if (token >= start && mine == i) r = KvToken{s0 + n, pos};
    }
  }
  return r;
}

// ---------------------------------------------------------------------------
// values
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

// Eight values as they lie in memory, of 2 or 4 bytes each: loaded early, turned into
// floats where they are needed.
template <int BYTES>
struct Raw8 {
  u32x4 w[BYTES / 2];
  // vec: the values are 16-byte aligned.
  __device__ __forceinline__ void load(const void* p, size_t i, bool vec) {
    const uint8_t* from = (const uint8_t*)p + i * BYTES;
    if (vec) {
#pragma unroll
      for (int j = 0; j < BYTES / 2; ++j) w[j] = ((const u32x4*)from)[j];
    } else if constexpr (BYTES == 4) {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e / 4][e % 4] = ((const uint32_t*)from)[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[0][e] = (uint32_t)((const uint16_t*)from)[2 * e] | (uint32_t)((const uint16_t*)from)[2 * e + 1] << 16;
    }
  }
  __device__ __forceinline__ void get(int dt, float (&x)[8]) const {
    if constexpr (BYTES == 4) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t v = w[e / 4][e % 4];
        x[e] = __builtin_bit_cast(float, v);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint16_t h = (uint16_t)(w[0][e / 2] >> (16 * (e & 1)));
        x[e] = dt == DT_F16 ? h2f(h) : bf2f(h);
      }
    }
  }
};

// Two floats as 16-bit values of type dt, rounded to nearest even.
typedef float float2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf2v __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pack2(int dt, float a, float b) {
  const float2v v = {a, b};
  return dt == DT_F16 ? __builtin_bit_cast(uint32_t, __builtin_convertvector(v, half2v))
                      : __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf2v));
}

// Eight values to 16-byte aligned memory.
__device__ __forceinline__ void store8(void* p, int dt, size_t i, const float (&x)[8]) {
  if (dt == DT_F32) {
    float4v a, b;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      a[e] = x[e];
      b[e] = x[e + 4];
    }
    *(float4v*)((float*)p + i) = a;
    *(float4v*)((float*)p + i + 4) = b;
  } else {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = pack2(dt, x[2 * e], x[2 * e + 1]);
    *(u32x4*)((uint16_t*)p + i) = w;
  }
}

// ---------------------------------------------------------------------------
// codes
// ---------------------------------------------------------------------------
// Eight 8-bit codes (code + 128) as f16: byte b between 0x64 and itself is the f16 1024 + b,
// and 1024 + b - 1152 is exact.
__device__ __forceinline__ u32x4 codes8(uint32_t w0, uint32_t w1) {
  const half2v off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
  u32x4 r;
  r[0] = __builtin_amdgcn_perm(0x64646464u, w0, 0x04010400u);
  r[1] = __builtin_amdgcn_perm(0x64646464u, w0, 0x04030402u);
  r[2] = __builtin_amdgcn_perm(0x64646464u, w1, 0x04010400u);
  r[3] = __builtin_amdgcn_perm(0x64646464u, w1, 0x04030402u);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t x = r[i];
    r[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, x) + off);
  }
  return r;
}

// (a & m) | b in one instruction (the compiler makes two of it with literal operands).
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t m, uint32_t b) {
  uint32_t d;
  asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "s"(m), "v"(b));
  return d;
}

// Eight 4-bit codes (code + 8) as f16, in the order 0 4 1 5 2 6 3 7: a nibble in the lowest
// or second-lowest place of an f16's mantissa under the exponent of 1024 is 1024 + n or
// 1024 + 16 n.
__device__ __forceinline__ u32x4 codes4(uint32_t w) {
  const half2v off = {(_Float16)-1032.0f, (_Float16)-1032.0f};
  const half2v part = {(_Float16)0.0625f, (_Float16)0.0625f}, off16 = {(_Float16)-72.0f, (_Float16)-72.0f};
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t v = w >> (8 * i);
    const uint32_t lo = and_or(v, 0x000f000fu, 0x64006400u), hi = and_or(v, 0x00f000f0u, 0x64006400u);
    r[2 * i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, lo) + off);
    r[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(half2v, hi), part, off16));
  }
  return r;
}

// Eight f16 times one.
__device__ __forceinline__ u32x4 times(const u32x4& v, _Float16 s) {
  const half2v s2 = {s, s};
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t x = v[i];
    r[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, x) * s2);
  }
  return r;
}
__device__ __forceinline__ u32x4 decode8(uint32_t w0, uint32_t w1, _Float16 s) { return times(codes8(w0, w1), s); }

// Eight 4-bit codes times a scale in the channels' own order.
__device__ __forceinline__ u32x4 decode4(uint32_t w, _Float16 s) {
  const u32x4 d = times(codes4(w), s);
  const uint32_t a = d[0], b = d[1], c = d[2], e = d[3];
  return u32x4{__builtin_amdgcn_perm(b, a, 0x05040100u), __builtin_amdgcn_perm(e, c, 0x05040100u),
               __builtin_amdgcn_perm(b, a, 0x07060302u), __builtin_amdgcn_perm(e, c, 0x07060302u)};
}
}  // namespace exl3
