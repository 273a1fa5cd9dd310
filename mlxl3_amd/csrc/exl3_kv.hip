// Rotary positions, and writing and reading the paged key/value cache (layout:
// exl3_kv.hpp).
//
// Rotation: channel pairs (a, b) of a head turn by t = p * f_i,
//   (a, b) -> (a c - b s, a s + b c),  c = m cos t,  s = m sin t.
// t and its cosine and sine are formed in 64 bits and rounded to f32 once (at
// p = 100000 an f32 product alone is off by 0.004 rad); the products and their sum are
// f32.  A workgroup computes the cosines and sines of its tokens once, in LDS, for all
// heads.
//
// Quantisation: 32 neighbouring channels of a head share the f16 scale
//   s = f16(max|x| / 127)  (4 bits: / 7),  at most 65504,
// and store code = rint(x / s) (ties to even), clipped to +-127 (+-7); s = 0 stores
// zeros.  A group with a NaN or an infinity gets s = NaN, so that it reads back as
// NaN.  Everything is f32 with one rounding per operation, the quotient correctly
// rounded, so the codes do not depend on how the work is laid out.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <new>

#include "../../include/exl3_hip.h"
#include "exl3_kv_host.hpp"
#include "exl3_launch.hpp"

namespace exl3 {

// cos and sin of t for |t| < 2^40: quarter turns removed with pi/2 in two parts, then
// the Taylor series on [-pi/4, pi/4] (terms below 2^-56 left out).
__device__ __forceinline__ void sincos64(double t, double* s_out, double* c_out) {
  const double k = rint(t * 0.63661977236758134308);
  double r = fma(-k, 1.57079632679489661923, t);
  r = fma(-k, 6.123233995736766036e-17, r);
  const double z = r * r;
  double s = -1.0 / 1307674368000.0;  // 15!
  s = fma(s, z, 1.0 / 6227020800.0);
  s = fma(s, z, -1.0 / 39916800.0);
  s = fma(s, z, 1.0 / 362880.0);
  s = fma(s, z, -1.0 / 5040.0);
  s = fma(s, z, 1.0 / 120.0);
  s = fma(s, z, -1.0 / 6.0);
  s = fma(s * z, r, r);
  double c = 1.0 / 20922789888000.0;  // 16!
  c = fma(c, z, -1.0 / 87178291200.0);
  c = fma(c, z, 1.0 / 479001600.0);
  c = fma(c, z, -1.0 / 3628800.0);
  c = fma(c, z, 1.0 / 40320.0);
  c = fma(c, z, -1.0 / 720.0);
  c = fma(c, z, 1.0 / 24.0);
  c = fma(c, z, -0.5);
  c = fma(c, z, 1.0);
  const int q = (int)((int64_t)k & 3);
  const double a = q & 1 ? c : s, b = q & 1 ? s : c;
  *s_out = q & 2 ? -a : a;
  *c_out = (q + 1) & 2 ? -b : b;
}

struct RopeView {
  const float* freq;  // [pairs]; null: no rotation
  int pairs, interleaved;
  double scale;
};

// Cosine and sine of pair i at position pos, in f32.
__device__ __forceinline__ float2 rope_cs(const RopeView& r, int64_t pos, int i) {
  double s, c;
  sincos64((double)pos * (double)r.freq[i], &s, &c);
  return make_float2((float)(c * r.scale), (float)(s * r.scale));
}

constexpr int kMaxDim = 256;        // largest head
constexpr int kRopeTokens = 4;      // tokens per workgroup of the kernels below

struct RopeParams {
  const void* x;
  void* y;
  const int32_t* positions;  // null: positions of the batch
  KvBatchView batch;
  RopeView rope;
  int64_t tokens, x_stride, y_stride;
  int heads, head_dim, x_type, y_type;
};

// grid ceil(tokens / kRopeTokens).  VEC: a work item is eight pairs (two chunks of
// eight channels, or one chunk of neighbours) or a chunk behind the rotated
// channels; else one pair or one channel.  An item loads all it needs before it
// stores, so y may be x.
template <bool VEC>
__global__ __launch_bounds__(256) void rope_kernel(RopeParams p) {
  __shared__ float2 cs[kRopeTokens][kMaxDim / 2];
  __shared__ int live[kRopeTokens];
  const int64_t t0 = (int64_t)blockIdx.x * kRopeTokens;
  const int nt = (int)min((int64_t)kRopeTokens, p.tokens - t0);
  const int r = p.rope.pairs;
  for (int e = threadIdx.x; e < nt * r; e += 256) {
    const int t = e / r, i = e - t * r;
    int64_t pos = 0;
    bool on = true;
    if (p.positions) {
      pos = p.positions[t0 + t];
    } else {
      const int seq = kv_sequence(p.batch, t0 + t);
      on = seq >= 0;
      if (on) pos = kv_position(p.batch, seq, t0 + t);
    }
    cs[t][i] = rope_cs(p.rope, pos, i);
    if (i == 0) live[t] = on;
  }
  __syncthreads();
  const int W = VEC ? 8 : 1;
  // items of a head: rotated ones, then the channels behind them
  const int turned = p.rope.interleaved && VEC ? 2 * r / W : r / W;
  const int per_head = turned + (p.head_dim - 2 * r) / W;
  const int per_token = per_head * p.heads;
  for (int e = threadIdx.x; e < nt * per_token; e += 256) {
    const int t = e / per_token, i = e - t * per_token;
    const int h = i / per_head, c = i - h * per_head;
    if (!live[t]) continue;
    const size_t xr = (size_t)(t0 + t) * p.x_stride + (size_t)h * p.head_dim;
    const size_t yr = (size_t)(t0 + t) * p.y_stride + (size_t)h * p.head_dim;
    if (c >= turned) {
      const int d = 2 * r + (c - turned) * W;
      if (p.x == p.y) continue;
      if constexpr (VEC) {
        float v[8];
        load8(p.x, p.x_type, xr + d, true, v);
        store8(p.y, p.y_type, yr + d, true, v);
      } else {
        store1(p.y, p.y_type, yr + d, load1(p.x, p.x_type, xr + d));
      }
    } else if constexpr (VEC) {
      if (p.rope.interleaved) {
        float v[8];
        load8(p.x, p.x_type, xr + 8 * c, true, v);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const float2 f = cs[t][4 * c + n];
          const float a = v[2 * n], b = v[2 * n + 1];
          v[2 * n] = a * f.x - b * f.y;
          v[2 * n + 1] = a * f.y + b * f.x;
        }
        store8(p.y, p.y_type, yr + 8 * c, true, v);
      } else {
        float a[8], b[8];
        load8(p.x, p.x_type, xr + 8 * c, true, a);
        load8(p.x, p.x_type, xr + r + 8 * c, true, b);
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const float2 f = cs[t][8 * c + n];
          const float u = a[n], w = b[n];
          a[n] = u * f.x - w * f.y;
          b[n] = u * f.y + w * f.x;
        }
        store8(p.y, p.y_type, yr + 8 * c, true, a);
        store8(p.y, p.y_type, yr + r + 8 * c, true, b);
      }
    } else {
      const int da = p.rope.interleaved ? 2 * c : c, db = p.rope.interleaved ? 2 * c + 1 : c + r;
      const float a = load1(p.x, p.x_type, xr + da), b = load1(p.x, p.x_type, xr + db);
      const float2 f = cs[t][c];
      store1(p.y, p.y_type, yr + da, a * f.x - b * f.y);
      store1(p.y, p.y_type, yr + db, a * f.y + b * f.x);
    }
  }
}

// The host code below is left out of the device pass, which needs the instances spelled out.
template __global__ void rope_kernel<true>(RopeParams);
template __global__ void rope_kernel<false>(RopeParams);

// The scale of a group whose largest magnitude is `most` (NaN where it is not finite).
__device__ __forceinline__ uint16_t group_scale(float most, float levels) {
  if (!(most <= 3.402823466e38f)) return 0x7e00;
  return f2h(fminf(most / levels, 65504.0f));
}

// rint(x / s) clipped to +-levels: the quotient from the rounded reciprocal and one
// residual step, which rounds it correctly (s is an f16 value, so neither the reciprocal
// nor the residual under- or overflows where the clip does not decide).
__device__ __forceinline__ int group_code(float x, float s, float inv, float levels) {
  float q = x * inv;
  q = fmaf(fmaf(-q, s, x), inv, q);
  q = fabsf(q) <= levels ? q : copysignf(levels, x);
  return (int)rintf(q);
}

struct AppendParams {
  KvCacheView cache;
  KvBatchView batch;
  RopeView rope;
  const void *k, *v;
  int64_t tokens, k_stride, v_stride;
  int type, vec;  // vec: rows of k and v are 16-byte aligned
};

// grid ceil(tokens / kRopeTokens): a work item is eight channels of one head of one
// token's key or value; a quantised group is the items of four neighbouring lanes.
__global__ __launch_bounds__(256) void kv_append_kernel(AppendParams p) {
  __shared__ float2 cs[kRopeTokens][kMaxDim / 2];
  __shared__ int64_t page_of[kRopeTokens];
  __shared__ int64_t pos_of[kRopeTokens];
  const KvCacheView& c = p.cache;
  const int64_t t0 = (int64_t)blockIdx.x * kRopeTokens;
  const int nt = (int)min((int64_t)kRopeTokens, p.tokens - t0);
  if ((int)threadIdx.x < nt) {
    const int seq = kv_sequence(p.batch, t0 + threadIdx.x);
    const int64_t pos = seq < 0 ? -1 : kv_position(p.batch, seq, t0 + threadIdx.x);
    page_of[threadIdx.x] = seq < 0 ? -1 : kv_page(c, p.batch, seq, pos);
    pos_of[threadIdx.x] = pos;
  }
  __syncthreads();
  const int r = p.rope.freq ? p.rope.pairs : 0;
  for (int e = threadIdx.x; e < nt * r; e += 256) {
    const int t = e / r, i = e - t * r;
    cs[t][i] = rope_cs(p.rope, pos_of[t], i);
  }
  if (r) __syncthreads();
  const int D = c.head_dim, chunks = D / 8, per_side = chunks * c.kv_heads;
  const int pmask = (1 << c.page_shift) - 1;
  for (int e = threadIdx.x; e < nt * 2 * per_side; e += 256) {
    const int t = e / (2 * per_side), i = e - t * 2 * per_side;
    const bool value = i >= per_side;
    const int j = value ? i - per_side : i, h = j / chunks, d0 = (j - h * chunks) * 8;
    if (page_of[t] < 0) continue;  // the four lanes of a group leave together
    const void* src = value ? p.v : p.k;
    const size_t row =
        (size_t)(t0 + t) * (value ? p.v_stride : p.k_stride) + (size_t)h * D;
    float x[8];
    load8(src, p.type, row + d0, p.vec, x);
    if (!value && d0 < 2 * r) {
      if (p.rope.interleaved) {
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          if (d0 / 2 + n < r) {
            const float2 f = cs[t][d0 / 2 + n];
            const float a = x[2 * n], b = x[2 * n + 1];
            x[2 * n] = a * f.x - b * f.y;
            x[2 * n + 1] = a * f.y + b * f.x;
          }
        }
      } else if (r % 8 == 0) {
        const bool second = d0 >= r;
        const int i0 = second ? d0 - r : d0;
        float o[8];
        load8(src, p.type, row + (second ? d0 - r : d0 + r), p.vec, o);
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const float2 f = cs[t][i0 + n];
          x[n] = second ? o[n] * f.y + x[n] * f.x : x[n] * f.x - o[n] * f.y;
        }
      } else {
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const int d = d0 + n;
          if (d < 2 * r) {
            const bool second = d >= r;
            const float2 f = cs[t][second ? d - r : d];
            const float o = load1(src, p.type, row + (second ? d - r : d + r));
            x[n] = second ? o * f.y + x[n] * f.x : x[n] * f.x - o * f.y;
          }
        }
      }
    }
    const size_t head = (size_t)page_of[t] * c.kv_heads + h;
    const int slot = (int)(pos_of[t] & pmask);
    const size_t token = (head << c.page_shift) + slot;  // row of D values
    uint8_t* base = value ? c.v : c.k;
    if (c.format == KV_F16 || c.format == KV_BF16) {
      store8(base, c.format, token * D + d0, true, x);
      continue;
    }
    float most = 0.0f;
    bool whole = true;  // fmaxf drops a NaN
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      most = fmaxf(most, fabsf(x[n]));
      whole = whole && fabsf(x[n]) <= 3.402823466e38f;
    }
    if (!whole) most = __builtin_inff();
    most = fmaxf(most, xor_lanes<1>(most));
    most = fmaxf(most, xor_lanes<2>(most));
    const float levels = c.format == KV_Q8 ? 127.0f : 7.0f;
    const uint16_t sh = group_scale(most, levels);
    const float s = h2f(sh);
    const bool on = s > 0.0f;
    const float inv = on ? 1.0f / s : 0.0f;
    int code[8];
#pragma unroll
    for (int n = 0; n < 8; ++n) { code[n] = on ? group_code(x[n], s, inv, levels) : 0; }
    if (c.format == KV_Q8) {
      u32x2 w = {0, 0};
#pragma unroll
      for (int n = 0; n < 8; ++n) { w[n / 4] |= (uint32_t)(code[n] + 128) << (8 * (n & 3)); }
      *(u32x2*)(base + token * D + d0) = w;
    } else {
      uint32_t w = 0;
#pragma unroll
      for (int n = 0; n < 8; ++n) { w |= (uint32_t)(code[n] + 8) << (4 * n); }
      *(uint32_t*)(base + (token * D + d0) / 2) = w;
    }
    if ((d0 & 31) == 0) {
      uint16_t* sc = value ? c.vs : c.ks;
      sc[((head * (D / 32) + d0 / 32) << c.page_shift) + slot] = sh;
    }
  }
}

struct ReadParams {
  KvCacheView cache;
  KvBatchView batch;
  void *k, *v;
  int64_t tokens;
  int type;
};

// grid ceil(tokens / kRopeTokens): the items of kv_append_kernel, the other way.
__global__ __launch_bounds__(256) void kv_read_kernel(ReadParams p) {
  __shared__ int64_t page_of[kRopeTokens];
  __shared__ int slot_of[kRopeTokens];  // -1: behind the last sequence
  const KvCacheView& c = p.cache;
  const int64_t t0 = (int64_t)blockIdx.x * kRopeTokens;
  const int nt = (int)min((int64_t)kRopeTokens, p.tokens - t0);
  const int pmask = (1 << c.page_shift) - 1;
  if ((int)threadIdx.x < nt) {
    const int seq = kv_sequence(p.batch, t0 + threadIdx.x);
    const int64_t pos = seq < 0 ? 0 : kv_position(p.batch, seq, t0 + threadIdx.x);
    page_of[threadIdx.x] = seq < 0 ? -1 : kv_page(c, p.batch, seq, pos);
    slot_of[threadIdx.x] = seq < 0 ? -1 : (int)(pos & pmask);
  }
  __syncthreads();
  const int D = c.head_dim, chunks = D / 8, per_side = chunks * c.kv_heads;
  for (int e = threadIdx.x; e < nt * 2 * per_side; e += 256) {
    const int t = e / (2 * per_side), i = e - t * 2 * per_side;
    const bool value = i >= per_side;
    const int j = value ? i - per_side : i, h = j / chunks, d0 = (j - h * chunks) * 8;
    const int slot = slot_of[t];
    if (slot < 0) continue;
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};  // a token without a page reads as zeros
    if (page_of[t] >= 0) {
      const size_t head = (size_t)page_of[t] * c.kv_heads + h;
      const size_t token = (head << c.page_shift) + slot;
      float s = 1.0f;
      if (c.ks)
        s = h2f((value ? c.vs : c.ks)[((head * (D / 32) + d0 / 32) << c.page_shift) + slot]);
      kv_load8((value ? c.v : c.k) + kv_bytes(c.format, token * D), c.format, d0, s, x);
    }
    store8(value ? p.v : p.k, p.type, ((size_t)(t0 + t) * c.kv_heads + h) * D + d0, true, x);
  }
}

}  // namespace exl3

using namespace exl3;

#ifndef __HIP_DEVICE_COMPILE__

bool exl3::aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

static bool known_type(int t) { return t == EXL3_F16 || t == EXL3_BF16 || t == EXL3_F32; }
static size_t type_bytes(int t) { return t == EXL3_F32 ? 4 : 2; }
static bool rows_aligned(const void* p, int64_t stride, int type) {
  return aligned16(p) && (size_t)stride * type_bytes(type) % 16 == 0;
}

extern "C" int exl3_kv_cache_create(void* k, void* v, uint16_t* k_scales, uint16_t* v_scales,
                                    int32_t format, int64_t pages, int32_t page_tokens,
                                    int32_t kv_heads, int32_t head_dim, exl3_kv_cache** out_handle) {
  if (!out_handle) return fail(EXL3_EINVAL, "null out_handle");
  *out_handle = nullptr;
  if (format != EXL3_KV_F16 && format != EXL3_KV_BF16 && format != EXL3_KV_Q8 &&
      format != EXL3_KV_Q4)
    return fail(EXL3_EINVAL, "unknown KV cache format %d", format);
  if (page_tokens < 16 || page_tokens > 1024 || (page_tokens & (page_tokens - 1)))
    return fail(EXL3_EINVAL, "KV pages hold a power of two of 16 to 1024 tokens, got %d",
                page_tokens);
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return fail(EXL3_EUNSUPPORTED, "KV heads of 64, 128 or 256 channels are supported, got %d",
                head_dim);
  if (kv_heads < 1 || kv_heads > 1024)
    return fail(EXL3_EINVAL, "invalid KV head count %d", kv_heads);
  if (pages < 1 || pages > INT32_MAX)
    return fail(EXL3_EINVAL, "invalid KV page count %lld", (long long)pages);
  const bool coded = format == EXL3_KV_Q8 || format == EXL3_KV_Q4;
  if (!k || !v || (coded && (!k_scales || !v_scales)))
    return fail(EXL3_EINVAL, "null KV cache buffer");
  if (!coded && (k_scales || v_scales))
    return fail(EXL3_EINVAL, "16-bit KV caches have no scales");
  if (!aligned16(k) || !aligned16(v) || !aligned16(k_scales) || !aligned16(v_scales))
    return fail(EXL3_EINVAL, "KV cache buffers must be 16-byte aligned");
  exl3_kv_cache* h = new (std::nothrow) exl3_kv_cache;
  if (!h) return fail(EXL3_ENOMEM, "out of host memory");
  h->view.k = (uint8_t*)k;
  h->view.v = (uint8_t*)v;
  h->view.ks = k_scales;
  h->view.vs = v_scales;
  h->view.pages = pages;
  h->view.page_shift = __builtin_ctz((unsigned)page_tokens);
  h->view.kv_heads = kv_heads;
  h->view.head_dim = head_dim;
  h->view.format = format;
  *out_handle = h;
  return EXL3_OK;
}

extern "C" void exl3_kv_cache_destroy(exl3_kv_cache* handle) { delete handle; }

int exl3::check_batch(const exl3_kv_cache* cache, const exl3_kv_batch* batch, int64_t tokens,
                      KvBatchView* view) {
  if (!batch) return fail(EXL3_EINVAL, "null KV batch");
  if (tokens < 0) return fail(EXL3_EINVAL, "negative token count");
  if (batch->seqs < 1) return fail(EXL3_EINVAL, "a KV batch has at least one sequence");
  if (!batch->q_starts || !batch->kv_lens) return fail(EXL3_EINVAL, "null KV batch lengths");
  if (cache && (!batch->block_table || batch->table_pages < 1))
    return fail(EXL3_EINVAL, "a KV batch needs a block table");
  view->q_starts = batch->q_starts;
  view->kv_lens = batch->kv_lens;
  view->table = batch->block_table;
  view->seqs = batch->seqs;
  view->table_pages = batch->table_pages;
  return EXL3_OK;
}

static int check_rope(const exl3_rope_spec* rope, int head_dim, RopeView* view) {
  if (!rope->inv_freq) return fail(EXL3_EINVAL, "null rotary frequencies");
  if (rope->rotary_dim < 2 || rope->rotary_dim % 2 || rope->rotary_dim > head_dim)
    return fail(EXL3_EINVAL, "rotary dimension %d of heads of %d channels", rope->rotary_dim,
                head_dim);
  if (!std::isfinite(rope->scale)) return fail(EXL3_EINVAL, "rotary scale must be finite");
  view->freq = rope->inv_freq;
  view->pairs = rope->rotary_dim / 2;
  view->interleaved = rope->interleaved != 0;
  view->scale = rope->scale;
  return EXL3_OK;
}

static int token_blocks(int64_t tokens, unsigned* blocks) {
  const int64_t n = (tokens + kRopeTokens - 1) / kRopeTokens;
  if (n > INT32_MAX) return fail(EXL3_EINVAL, "too many tokens: %lld", (long long)tokens);
  *blocks = (unsigned)n;
  return EXL3_OK;
}

extern "C" int exl3_rope(const exl3_rope_spec* rope, const void* x, int32_t x_type, int64_t tokens,
                         int32_t heads, int32_t head_dim, int64_t x_stride,
                         const int32_t* positions, const exl3_kv_batch* batch, void* y,
                         int32_t y_type, int64_t y_stride, void* stream) {
  if (!rope) return fail(EXL3_EINVAL, "null rotary spec");
  if (tokens < 0) return fail(EXL3_EINVAL, "negative token count");
  if (!known_type(x_type) || !known_type(y_type))
    return fail(EXL3_EINVAL, "unsupported rotary dtypes %d and %d", x_type, y_type);
  if (heads < 1 || heads > 65536 || head_dim < 2 || head_dim > kMaxDim)
    return fail(EXL3_EINVAL, "invalid rotary heads: %d of %d channels", heads, head_dim);
  const int64_t width = (int64_t)heads * head_dim;
  if (tokens > 1 && (x_stride < width || y_stride < width))
    return fail(EXL3_EINVAL, "token strides are at least heads * head_dim");
  if (!positions == !batch)
    return fail(EXL3_EINVAL, "rotary positions come from an array or from a KV batch");
  RopeParams p{};
  if (int rc = check_rope(rope, head_dim, &p.rope)) return rc;
  if (batch)
    if (int rc = check_batch(nullptr, batch, tokens, &p.batch)) return rc;
  if (tokens == 0) return EXL3_OK;
  if (!x || !y) return fail(EXL3_EINVAL, "null rotary input or output");
  if (x == y && (x_type != y_type || (tokens > 1 && x_stride != y_stride)))
    return fail(EXL3_EINVAL, "rotation in place keeps the type and the stride");
  unsigned blocks;
  if (int rc = token_blocks(tokens, &blocks)) return rc;
  p.x = x;
  p.y = y;
  p.positions = positions;
  p.tokens = tokens;
  p.x_stride = x_stride;
  p.y_stride = y_stride;
  p.heads = heads;
  p.head_dim = head_dim;
  p.x_type = x_type;
  p.y_type = y_type;
  // eight channels at a time where every chunk starts 16-byte aligned and no chunk
  // holds a border of the rotated channels
  const bool vec = head_dim % 8 == 0 && p.rope.pairs % (p.rope.interleaved ? 4 : 8) == 0 &&
                   rows_aligned(x, tokens > 1 ? x_stride : 0, x_type) &&
                   rows_aligned(y, tokens > 1 ? y_stride : 0, y_type);
  if (int rc = launch_gate("rotary launch")) return rc;
  if (vec)
    hipLaunchKernelGGL(rope_kernel<true>, dim3(blocks), dim3(256), 0, (hipStream_t)stream, p);
  else
    hipLaunchKernelGGL(rope_kernel<false>, dim3(blocks), dim3(256), 0, (hipStream_t)stream, p);
  return check_launch("rotary launch");
}

extern "C" int exl3_kv_append(const exl3_kv_cache* cache, const exl3_kv_batch* batch,
                              const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                              int32_t type, int64_t tokens, const exl3_rope_spec* rope,
                              void* stream) {
  if (!cache) return fail(EXL3_EINVAL, "null KV cache");
  AppendParams p{};
  p.cache = cache->view;
  if (int rc = check_batch(cache, batch, tokens, &p.batch)) return rc;
  if (!known_type(type)) return fail(EXL3_EINVAL, "unsupported KV input dtype %d", type);
  const int64_t width = (int64_t)p.cache.kv_heads * p.cache.head_dim;
  if (tokens > 1 && (k_stride < width || v_stride < width))
    return fail(EXL3_EINVAL, "token strides are at least kv_heads * head_dim");
  if (rope)
    if (int rc = check_rope(rope, p.cache.head_dim, &p.rope)) return rc;
  if (tokens == 0) return EXL3_OK;
  if (!k || !v) return fail(EXL3_EINVAL, "null KV input");
  unsigned blocks;
  if (int rc = token_blocks(tokens, &blocks)) return rc;
  p.k = k;
  p.v = v;
  p.tokens = tokens;
  p.k_stride = k_stride;
  p.v_stride = v_stride;
  p.type = type;
  p.vec = rows_aligned(k, tokens > 1 ? k_stride : 0, type) &&
          rows_aligned(v, tokens > 1 ? v_stride : 0, type);
  if (int rc = launch_gate("KV append")) return rc;
  hipLaunchKernelGGL(kv_append_kernel, dim3(blocks), dim3(256), 0, (hipStream_t)stream, p);
  return check_launch("KV append");
}

extern "C" int exl3_kv_read(const exl3_kv_cache* cache, const exl3_kv_batch* batch, void* k,
                            void* v, int32_t type, int64_t tokens, void* stream) {
  if (!cache) return fail(EXL3_EINVAL, "null KV cache");
  ReadParams p{};
  p.cache = cache->view;
  if (int rc = check_batch(cache, batch, tokens, &p.batch)) return rc;
  if (!known_type(type)) return fail(EXL3_EINVAL, "unsupported KV output dtype %d", type);
  if (tokens == 0) return EXL3_OK;
  if (!k || !v) return fail(EXL3_EINVAL, "null KV output");
  if (!aligned16(k) || !aligned16(v))
    return fail(EXL3_EINVAL, "KV outputs must be 16-byte aligned");
  unsigned blocks;
  if (int rc = token_blocks(tokens, &blocks)) return rc;
  p.k = k;
  p.v = v;
  p.tokens = tokens;
  p.type = type;
  if (int rc = launch_gate("KV read")) return rc;
  hipLaunchKernelGGL(kv_read_kernel, dim3(blocks), dim3(256), 0, (hipStream_t)stream, p);
  return check_launch("KV read");
}

#endif  // __HIP_DEVICE_COMPILE__
