// Attention of new tokens over the paged cache (layout: exl3_kv.hpp).
//
//   y_row = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q_row . k_t - m),
//
// over the tokens t that the row sees: t < kv_len, causal t <= its position, window
// t > its position - window.  m is the largest score so far: one pass over the cache
// with a running maximum and sum, both f32.  A row that sees nothing gives zeros.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/exl3_hip.h"
#include "exl3_kv_host.hpp"
#include "exl3_launch.hpp"

namespace exl3 {

struct AttnParams {
  KvCacheView cache;
  KvBatchView batch;
  const void* q;
  void* y;
  int64_t tokens, q_stride, y_stride;
  int heads, group, q_type, causal, window;
  float scale2;  // scale * log2(e): scores in units of a factor of two
};

__device__ __forceinline__ float wave_sum(float v) {
  v += xor_lanes<1>(v);
  v += xor_lanes<2>(v);
  v += xor_lanes<4>(v);
  v += xor_lanes<8>(v);
  v += xor_lanes<16>(v);
  v += xor_lanes<32>(v);
  return v;
}

// One wave per (token row, query head), the head's channels spread over its lanes.
template <int E>
__global__ __launch_bounds__(64) void attn_row_kernel(AttnParams p) {
  const int64_t token = blockIdx.x;
  const int head = blockIdx.y, lane = threadIdx.x;
  const int seq = kv_sequence(p.batch, token);
  if (seq < 0) return;
  const KvCacheView& c = p.cache;
  const int D = 64 * E;
  const int64_t pos = kv_position(p.batch, seq, token);
  const int64_t room = (int64_t)p.batch.table_pages << c.page_shift;
  int64_t hi = min((int64_t)p.batch.kv_lens[seq], room), lo = 0;
  if (p.causal) hi = min(hi, pos + 1);
  if (p.window > 0) lo = max(lo, pos - p.window + 1);
  float q[E], acc[E], m = -__builtin_inff(), l = 0.0f;
  for (int e = 0; e < E; ++e) {
    q[e] = load1(p.q, p.q_type, (size_t)token * p.q_stride + (size_t)head * D + E * lane + e);
    acc[e] = 0.0f;
  }
  const int kvh = head / p.group;
  for (int64_t t = lo; t < hi; ++t) {
    const int64_t page = kv_page(c, p.batch, seq, t);
    if (page < 0) continue;
    const size_t h = (size_t)page * c.kv_heads + kvh;
    const int slot = (int)(t & ((1 << c.page_shift) - 1));
    const size_t row = kv_bytes(c.format, ((h << c.page_shift) + slot) * D);
    float s = 0.0f, v[E], ks = 1.0f, vs = 1.0f;
    if (c.ks) {
      const size_t g = ((h * (D / 32) + E * lane / 32) << c.page_shift) + slot;
      ks = h2f(c.ks[g]);
      vs = h2f(c.vs[g]);
    }
    for (int e = 0; e < E; ++e) {
      const int d = E * lane + e;
      float k;
      if (c.format == KV_Q8) {
        k = (float)((int)c.k[row + d] - 128) * ks;
        v[e] = (float)((int)c.v[row + d] - 128) * vs;
      } else if (c.format == KV_Q4) {
        k = (float)(((int)c.k[row + d / 2] >> (4 * (d & 1)) & 15) - 8) * ks;
        v[e] = (float)(((int)c.v[row + d / 2] >> (4 * (d & 1)) & 15) - 8) * vs;
      } else {
        k = load1(c.k + row, c.format, d);
        v[e] = load1(c.v + row, c.format, d);
      }
      s += q[e] * k;
    }
    s = wave_sum(s) * p.scale2;
    const float n = fmaxf(m, s);
    const float base = n == -__builtin_inff() ? 0.0f : n;
    const float f = exp2f(m - base), w = exp2f(s - base);
    l = l * f + w;
    for (int e = 0; e < E; ++e) acc[e] = acc[e] * f + w * v[e];
    m = n;
  }
  for (int e = 0; e < E; ++e)
    store1(p.y, p.q_type, (size_t)token * p.y_stride + (size_t)head * D + E * lane + e,
           l > 0.0f || l != l ? acc[e] / l : 0.0f);
}

template __global__ void attn_row_kernel<1>(AttnParams);
template __global__ void attn_row_kernel<2>(AttnParams);
template __global__ void attn_row_kernel<4>(AttnParams);

}  // namespace exl3

using namespace exl3;

#ifndef __HIP_DEVICE_COMPILE__

extern "C" size_t exl3_attention_workspace_bytes(const exl3_kv_cache* cache,
                                                 const exl3_kv_batch* batch, int64_t tokens,
                                                 int32_t heads) {
  if (!cache || !batch || tokens <= 0 || heads <= 0) return 0;
  return 0;
}

extern "C" int exl3_attention(const exl3_kv_cache* cache, const exl3_kv_batch* batch,
                              const void* q, int32_t q_type, int64_t tokens, int32_t heads,
                              int64_t q_stride, float scale, int32_t causal, int32_t window,
                              void* y, int64_t y_stride, void* workspace, size_t workspace_bytes,
                              void* stream) {
  if (!cache) return fail(EXL3_EINVAL, "null KV cache");
  AttnParams p{};
  p.cache = cache->view;
  if (int rc = check_batch(cache, batch, tokens, &p.batch)) return rc;
  if (q_type != EXL3_F16 && q_type != EXL3_BF16)
    return fail(EXL3_EINVAL, "attention takes f16 or bf16 queries, got dtype %d", q_type);
  const bool coded = p.cache.format == EXL3_KV_Q8 || p.cache.format == EXL3_KV_Q4;
  if (!coded && p.cache.format != q_type)
    return fail(EXL3_EINVAL, "queries of a 16-bit KV cache have its type");
  if (heads < 1 || heads > 65535 || heads % p.cache.kv_heads)
    return fail(EXL3_EINVAL, "%d query heads over %d KV heads", heads, p.cache.kv_heads);
  if (!(scale > 0.0f) || !std::isfinite(scale))
    return fail(EXL3_EINVAL, "attention scale must be positive and finite");
  if (window < 0) return fail(EXL3_EINVAL, "negative attention window %d", window);
  if (batch->max_q < 1) return fail(EXL3_EINVAL, "max_q must be positive");
  const int64_t width = (int64_t)heads * p.cache.head_dim;
  if (tokens > 1 && (q_stride < width || y_stride < width))
    return fail(EXL3_EINVAL, "token strides are at least heads * head_dim");
  if (tokens == 0) return EXL3_OK;
  if (!q || !y) return fail(EXL3_EINVAL, "null attention input or output");
  if (tokens > INT32_MAX) return fail(EXL3_EINVAL, "too many tokens: %lld", (long long)tokens);
  const size_t need = exl3_attention_workspace_bytes(cache, batch, tokens, heads);
  if (need && (!workspace || workspace_bytes < need))
    return fail(EXL3_EINVAL, "workspace too small: need %zu bytes, got %zu", need, workspace_bytes);
  p.q = q;
  p.y = y;
  p.tokens = tokens;
  p.q_stride = q_stride;
  p.y_stride = y_stride;
  p.heads = heads;
  p.group = heads / p.cache.kv_heads;
  p.q_type = q_type;
  p.causal = causal != 0;
  p.window = window;
  p.scale2 = scale * 1.4426950408889634f;
  if (int rc = launch_gate("attention")) return rc;
  const dim3 grid((unsigned)tokens, (unsigned)heads);
  hipStream_t s = (hipStream_t)stream;
  if (p.cache.head_dim == 64)
    hipLaunchKernelGGL(attn_row_kernel<1>, grid, dim3(64), 0, s, p);
  else if (p.cache.head_dim == 128)
    hipLaunchKernelGGL(attn_row_kernel<2>, grid, dim3(64), 0, s, p);
  else
    hipLaunchKernelGGL(attn_row_kernel<4>, grid, dim3(64), 0, s, p);
  return check_launch("attention");
}

#endif  // __HIP_DEVICE_COMPILE__
