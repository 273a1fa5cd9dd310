// Attention of new tokens over the paged cache (layout: exl3_kv.hpp).
//
//   y_row = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q_row . k_t - m),
//
// over the tokens t that the row sees: t < kv_len, causal t <= its position, window
// t > its position - window; with a prefix t < prefix too, whatever its position.  Shaped scores
// are capped and biased first (exl3_attn.hpp).  m lies near the largest score so far (kSlack, kRoom): one pass
// over the cache with a running maximum and sum, both f32.  A row that sees nothing gives zeros.
//
// The rows of a launch are (token, query head of a group) pairs: all heads that read one
// cache head share its bytes.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/exl3_hip.h"
#include "exl3_attn_launch.hpp"
#include "exl3_kv_host.hpp"
#include "exl3_launch.hpp"

namespace exl3 {

// The splits or ranges of a row joined: grid (rows / rows per workgroup, kv heads, tiles or
// sequences).  D / 4 lanes hold a row's sums, four channels each; 2^shift such groups share
// the splits of one row, so that a row's loads are in flight together, and meet in LDS in a
// fixed order.
// A split that saw nothing has a maximum of -inf and a sum of 0, and its sums, which are
// not written, are not used.  Its latency bounds it: 5 us for 32 splits of 32 rows (a launch
// alone takes 2 to 3), 53 before the loads went out together.
template <int D, int S>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnParams p, int rows, int shift) {
  constexpr int L = D / 4, kGroups = 256 / L, kBatch = 8;
  __shared__ float4v sums[kGroups][L];
  __shared__ float totals[kGroups];
  const int group = threadIdx.x / L, lane = threadIdx.x % L;
  const int per = 1 << shift, part = group & (per - 1);  // groups of a row, which of them
  const int in_tile = blockIdx.x * (kGroups >> shift) + (group >> shift);
  const int kvh = blockIdx.y, tile = blockIdx.z;
  int row0;
  const Work w = tile_work<S>(p, tile, rows, row0);
  const int row = row0 + in_tile;
  const bool live = in_tile < rows && row < w.rows;
  int count = p.splits;
  const size_t step = (size_t)p.cache.kv_heads * rows;
  size_t first = (size_t)tile * p.splits;
  if (p.budget) {  // this sequence's ranges lie behind those of the ones before
    const int size = range_tokens<S>(p);
    count = range_count(size, seen_tokens<S>(p, w));
    if (count < 2) return;
    float before = 0.0f;
    for (int seq = threadIdx.x & 63; seq < tile; seq += 64)
      before += (float)range_count(size, seen_tokens<S>(p, sequence_work<S>(p, seq)));
    first = (size_t)wave_sum(before);
  }
  const size_t slot = first * step + (size_t)kvh * rows + in_tile;
  float4v acc = {0, 0, 0, 0};
  float total = 0.0f;
  if (live) {
    float most = -__builtin_inff();
    for (int s0 = 0; s0 < count; s0 += kBatch) {
      float m[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int s = min(s0 + i, count - 1);
        m[i] = p.stats[(slot + s * step) * 2];
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) most = fmaxf(most, m[i]);
    }
    const float base = most == -__builtin_inff() ? 0.0f : most;
    for (int s0 = part; s0 < count; s0 += per * kBatch) {
      float f[kBatch], l[kBatch];
      bool saw[kBatch];
      float4v v[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int s = s0 + i * per;
        const size_t at = slot + min(s, count - 1) * step;
        const float m = p.stats[at * 2];
        l[i] = p.stats[at * 2 + 1];
        const bool on = s < count && !(m == -__builtin_inff() && l[i] == 0.0f);
        saw[i] = on;
        f[i] = on ? __builtin_amdgcn_exp2f(m - base) : 0.0f;
        l[i] = on ? l[i] : 0.0f;
        v[i] = *(const float4v*)(p.part + at * D + 4 * lane);  // may be unwritten: see below
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        total += l[i] * f[i];
        const float4v sum = acc + v[i] * f[i];
        acc = saw[i] ? sum : acc;
      }
    }
  }
  sums[group][lane] = acc;
  if (lane == 0) totals[group] = total;
  __syncthreads();
  if (!live || part) return;
  for (int g = 1; g < per; ++g) {
    acc += sums[group + g][lane];
    total += totals[group + g];
  }
  const size_t yi = (size_t)(w.start + row / p.group) * p.y_stride +
                    (size_t)(kvh * p.group + row % p.group) * D + 4 * lane;
#pragma unroll
  for (int e = 0; e < 4; ++e) store1(p.y, p.q_type, yi + e, total != 0.0f ? acc[e] / total : 0.0f);
}
#define EXL3_JOIN_INST(D) \
  template __global__ void attn_join_kernel<D, kPlain>(AttnParams, int, int); \
  template __global__ void attn_join_kernel<D, kEarly>(AttnParams, int, int);
EXL3_JOIN_INST(64) EXL3_JOIN_INST(128) EXL3_JOIN_INST(256)

EXL3_FEW(EXL3_FEW_INST, kPlain)
EXL3_MANY(EXL3_MANY_INST, kPlain)

}  // namespace exl3

using namespace exl3;

#ifndef __HIP_DEVICE_COMPILE__

namespace {

size_t align256(size_t v) { return (v + 255) / 256 * 256; }

// Few rows (decode, drafts) go to attn_few_kernel, up to 16 or 32 of them -- 32 of 256 channels
// do not fit its registers -- others to attn_many_kernel.  Rows 17 to 32, us: 20 rows over
// 6001 4-bit tokens 24.5 (many 26.5), 32 rows of 8 sequences over 4096 16-bit ones 36.3 (34.5):
// the border could lie between the two for 16 bits, by 5 %.
//
// Where the tiles leave the chip idle their tokens are split, evenly or by the batch's sum, into
// as many workgroups as run at once: three a CU with 16 rows, two with 32 or 128, one of 256
// channels.  (Half as many: 32 8-bit decodes 122 us instead of 95, 512 rows over 8192 107 for
// 103, but a sequence of 4000 with fifteen of 200 17.7 for 21.3 and 64 rows over 8192 30.4 for
// 35.8; twice as many: drafts 33 for 24, 512 rows 127.)  No more than 32 of a sequence, which
// one launch has to join (16: one token over 131071 120 us for 105; 64: 110, of 64 channels 24
// for 21, of 256 40 for 45), and none shorter than 128 tokens for few rows (256: one token over
// 1000 12.2 us for 11.2) or 512 for many (256: 256 rows over 8192 36 us for 30).
//
// Ranges by the sum cost every workgroup a look at all lengths, some 3 us a call (drafts 28.0
// for 24.5), and save the wait for the longest sequence (8192 + 31 x 200 tokens 39 us to 24, 32
// decodes of 1000 to 8192 99 to 95): from 1024 tokens a split on.
AttnShape choose(const KvCacheView& c, const exl3_kv_batch& b, int64_t tokens, int heads, int window) {
  const int group = heads / c.kv_heads;
  const int64_t rows = (int64_t)b.max_q * group;
  AttnShape s;
  s.few = rows <= (c.head_dim == 256 ? 16 : 32);
  s.rows = s.few ? rows > 16 ? 32 : 16 : kManyRows;
  s.one_tile = rows <= s.rows;
  s.tiles = s.one_tile ? b.seqs
                       : std::min((rows + s.rows - 1) / s.rows * b.seqs, tokens * group / s.rows + b.seqs);
  const int64_t room = (int64_t)b.table_pages << c.page_shift;
  int64_t most = b.max_kv > 0 ? std::min<int64_t>(b.max_kv, room) : room;  // tokens a row sees
  if (window > 0) most = std::min<int64_t>(most, (int64_t)window + b.max_q);
  const int64_t resident = c.head_dim == 256 ? 256 : s.rows == 16 ? 768 : 512;
  const int64_t groups = s.tiles * c.kv_heads, want = (resident + groups - 1) / groups;
  const int64_t least = s.few ? 128 : 512;
  s.splits = (int)std::max<int64_t>(1, std::min(std::min<int64_t>(want, kMostRanges), (most + least / 2) / least));
  s.slots = s.splits > 1 ? groups * s.splits : 0;
  s.budget = 0;
  if (s.few && b.seqs > 1 && s.splits > 1 && most / s.splits >= 1024) {
    s.budget = (int)(resident / c.kv_heads - b.seqs / 2);  // seqs * kv_heads < resident: at least 1
    s.slots = std::max(s.slots, (s.budget + b.seqs + 1) * (int64_t)c.kv_heads);  // a window may ask for either
  }
  return s;
}

}  // namespace

extern "C" size_t exl3_attention_workspace_bytes(const exl3_kv_cache* cache,
                                                 const exl3_kv_batch* batch, int64_t tokens,
                                                 int32_t heads) {
  if (!cache || !batch || tokens <= 0 || heads <= 0 || batch->seqs <= 0 || batch->max_q <= 0 ||
      batch->table_pages <= 0 || heads % cache->view.kv_heads)
    return 0;
  const AttnShape sh = choose(cache->view, *batch, tokens, heads, 0);
  const size_t rows = (size_t)sh.slots * sh.rows;
  return align256(rows * cache->view.head_dim * 4) + align256(rows * 8);
}

// exl3_attention; without `run` its checks alone.
static int attention_call(const exl3_kv_cache* cache, const exl3_kv_batch* batch, const void* q,
                          int32_t q_type, int64_t tokens, int32_t heads, int64_t q_stride,
                          float scale, int32_t causal, int32_t window, const exl3_attn_scores* scores,
                          void* y, int64_t y_stride, void* workspace, size_t workspace_bytes,
                          void* stream, bool run) {
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
  const float scale2 = scale * 1.4426950408889634f;
  if (!(scale > 0.0f) || !std::isfinite(scale2))
    return fail(EXL3_EINVAL, "attention scale must be positive and finite");
  if (window < 0) return fail(EXL3_EINVAL, "negative attention window %d", window);
  int shaped = kPlain;
  if (scores) {
    const float cap = scores->softcap;
    if (cap != 0.0f && !(cap >= 0x1p-64f && cap <= 0x1p64f))
      return fail(EXL3_EINVAL, "attention softcap must be 0 or 2^-64 to 2^64, got %g", cap);
    p.cap2 = cap * kLog2e;
    p.slopes = scores->slopes;
    p.prefix = causal ? scores->prefix : nullptr;
    // the factors of kCapped and kEarly far inside f32's range, else one step after the other
    const float rate = cap != 0.0f ? 2.0f * kLog2e / p.cap2 * scale2 : 0.0f;
    const bool near = scale2 >= 0x1p-20f && scale2 <= 0x1p20f;
    if (cap != 0.0f)
      shaped = p.cap2 > kLargeCap || !(rate >= 0x1p-100f && rate <= 0x1p100f) ? kLate : p.slopes ? kBoth : kCapped;
    else if (p.slopes)
      shaped = near ? kEarly : kLate;
    else if (p.prefix)
      shaped = near ? kSeen : kLate;
  }
  if (batch->max_q < 1) return fail(EXL3_EINVAL, "max_q must be positive");
  if (batch->seqs > 65535)
    return fail(EXL3_EUNSUPPORTED, "attention takes up to 65535 sequences, got %d", batch->seqs);
  const int64_t width = (int64_t)heads * p.cache.head_dim;
  if (tokens > 1 && (q_stride < width || y_stride < width))
    return fail(EXL3_EINVAL, "token strides are at least heads * head_dim");
  if (tokens == 0) return EXL3_OK;
  if (!q || !y) return fail(EXL3_EINVAL, "null attention input or output");
  if (q == y && tokens > 1 && q_stride != y_stride)
    return fail(EXL3_EINVAL, "attention in place keeps the stride");
  if (tokens * (heads / p.cache.kv_heads) > INT32_MAX)
    return fail(EXL3_EUNSUPPORTED, "too many tokens: %lld", (long long)tokens);
  const size_t need = exl3_attention_workspace_bytes(cache, batch, tokens, heads);
  if (need && (!workspace || workspace_bytes < need))
    return fail(EXL3_EINVAL, "workspace too small: need %zu bytes, got %zu", need, workspace_bytes);
  if (need && !aligned16(workspace))
    return fail(EXL3_EINVAL, "attention workspace must be 16-byte aligned");
  // (a prefix makes no row see more: a row's position is at most max_q tokens from its sequence's end, so
  // that it sees up to window + max_q: 8 new tokens of 30008 under a window of 64 and a prefix of 30000
  // 11 us, without the window 31)
  const AttnShape sh = choose(p.cache, *batch, tokens, heads, window);
  if (sh.tiles * sh.splits * p.cache.kv_heads > kMostBlocks)
    return fail(EXL3_EUNSUPPORTED, "attention of %lld tokens needs too many workgroups", (long long)tokens);
  if (!run) return EXL3_OK;
  p.q = q;
  p.y = y;
  p.q_stride = q_stride;
  p.y_stride = y_stride;
  p.tokens = (int)tokens;
  p.group = heads / p.cache.kv_heads;
  p.q_type = q_type;
  p.causal = causal != 0;
  p.window = window;
  p.max_q = batch->max_q;
  p.splits = sh.splits;
  p.budget = sh.budget;
  p.one_tile = sh.one_tile;
  p.q_vec = aligned16(q) && (tokens == 1 || q_stride % 8 == 0);
  p.y_vec = ((uintptr_t)y & 7) == 0 && (tokens == 1 || y_stride % 4 == 0);
  p.scale2 = scale2;
  p.part = (float*)workspace;
  p.stats = (float*)((uint8_t*)workspace + align256((size_t)sh.slots * sh.rows * p.cache.head_dim * 4));
  const int D = p.cache.head_dim;
  hipStream_t s = (hipStream_t)stream;
  if (int rc = launch_gate("attention")) return rc;
  switch (shaped) {
    case kPlain: launch_attention<kPlain>(p, sh, s); break;
    case kSeen: case kEarly: launch_attention_early(p, sh, shaped == kSeen, s); break;
    case kCapped: case kBoth: launch_attention_capped(p, sh, shaped == kBoth, s); break;
    default: launch_attention_late(p, sh, s);
  }
  if (int rc = check_launch("attention")) return rc;
  if (!sh.slots) return EXL3_OK;
  if (int rc = launch_gate("attention join")) return rc;
  const int rows_most = (int)std::min<int64_t>(sh.rows, (int64_t)batch->max_q * p.group);
  // as many groups of lanes per row as there are splits to share
  const int groups = 1024 / D, most = sh.budget ? kMostRanges : sh.splits;
  int shift = 0;
  while ((2 << shift) <= groups && (1 << shift) < most) ++shift;
  const int per_block = groups >> shift;
  const dim3 grid((unsigned)((rows_most + per_block - 1) / per_block), (unsigned)p.cache.kv_heads,
                  (unsigned)sh.tiles);
  auto join = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, p, sh.rows, shift); };
  if (shaped)
    D == 64 ? join(attn_join_kernel<64, kEarly>) : D == 128 ? join(attn_join_kernel<128, kEarly>)
                                                          : join(attn_join_kernel<256, kEarly>);
  else
    D == 64 ? join(attn_join_kernel<64, kPlain>) : D == 128 ? join(attn_join_kernel<128, kPlain>)
                                                           : join(attn_join_kernel<256, kPlain>);
  return check_launch("attention join");
}

extern "C" int exl3_attention(const exl3_kv_cache* cache, const exl3_kv_batch* batch,
                              const void* q, int32_t q_type, int64_t tokens, int32_t heads,
                              int64_t q_stride, float scale, int32_t causal, int32_t window,
                              void* y, int64_t y_stride, void* workspace, size_t workspace_bytes,
                              void* stream) {
  return attention_call(cache, batch, q, q_type, tokens, heads, q_stride, scale, causal, window, nullptr, y, y_stride,
                        workspace, workspace_bytes, stream, true);
}

extern "C" int exl3_attention_scores(const exl3_kv_cache* cache, const exl3_kv_batch* batch,
                                     const void* q, int32_t q_type, int64_t tokens, int32_t heads,
                                     int64_t q_stride, float scale, int32_t causal, int32_t window,
                                     const exl3_attn_scores* scores, void* y, int64_t y_stride,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  return attention_call(cache, batch, q, q_type, tokens, heads, q_stride, scale, causal, window, scores, y, y_stride,
                        workspace, workspace_bytes, stream, true);
}

namespace {

// Workspace of an attention block: the projections' (its counters first), then q, k, v as
// projected, q as attention takes it where that is another type, attention's own.
struct Block {
  int heads, types[3];      // output types of q, k and v
  size_t linear, part[3], rounded, attention, total;
};

int plan_block(const exl3_linear* q, const exl3_linear* k, const exl3_linear* v, const exl3_linear* o,
               const exl3_kv_cache* cache, const exl3_kv_batch* batch, int32_t x_type, int64_t rows,
               Block* b) {
  if (!q || !k || !v || !o) return fail(EXL3_EINVAL, "null EXL3 linear handle");
  if (!cache) return fail(EXL3_EINVAL, "null KV cache");
  KvBatchView view;
  if (int rc = check_batch(cache, batch, rows, &view)) return rc;
  if (rows < 1) return fail(EXL3_EINVAL, "empty attention block input");
  if (x_type != EXL3_F16 && x_type != EXL3_BF16)
    return fail(EXL3_EINVAL, "attention blocks take f16 or bf16 activations, got dtype %d", x_type);
  const int D = cache->view.head_dim;
  const exl3_linear* parts[3] = {q, k, v};
  const int32_t wide = exl3_linear_out_features(q), narrow = cache->view.kv_heads * D;
  if (wide % D || (wide / D) % cache->view.kv_heads || exl3_linear_out_features(k) != narrow ||
      exl3_linear_out_features(v) != narrow || exl3_linear_in_features(o) != wide)
    return fail(EXL3_EINVAL, "attention block widths differ from the cache's heads");
  b->heads = wide / D;
  const size_t group = exl3_group_workspace_bytes(parts, 3, rows);
  if (!group) return fail(EXL3_EINVAL, "incompatible grouped projections");
  b->linear = align256(std::max(group, exl3_linear_workspace_bytes(o, rows)));
  size_t at = b->linear;
  for (int i = 0; i < 3; ++i) {
    b->types[i] = exl3_linear_output_dtype(parts[i], x_type);
    b->part[i] = at;
    at += align256((size_t)rows * (i ? narrow : wide) * (b->types[i] == EXL3_F32 ? 4 : 2));
  }
  b->rounded = at;
  if (b->types[0] != x_type) at += align256((size_t)rows * wide * 2);
  b->attention = at;
  b->total = at + exl3_attention_workspace_bytes(cache, batch, rows, b->heads);
  return EXL3_OK;
}

}  // namespace

extern "C" size_t exl3_attn_block_workspace_bytes(const exl3_linear* q, const exl3_linear* k,
                                                  const exl3_linear* v, const exl3_linear* o,
                                                  const exl3_kv_cache* cache,
                                                  const exl3_kv_batch* batch, int32_t x_type,
                                                  int64_t rows) {
  Block b;
  return plan_block(q, k, v, o, cache, batch, x_type, rows, &b) ? 0 : b.total;
}

extern "C" int exl3_attn_block_forward_scores(const exl3_linear* q, const exl3_linear* k,
                                              const exl3_linear* v, const exl3_linear* o,
                                              const exl3_kv_cache* cache, const exl3_kv_batch* batch,
                                              const exl3_rope_spec* rope, float scale, int32_t window,
                                              const exl3_attn_scores* scores, const void* x,
                                              int32_t x_type, int64_t rows, void* y, void* workspace,
                                              size_t workspace_bytes, void* stream) {
  Block b;
  if (int rc = plan_block(q, k, v, o, cache, batch, x_type, rows, &b)) return rc;
  if (!x || !y) return fail(EXL3_EINVAL, "null attention block input or output");
  if (!workspace || workspace_bytes < b.total)
    return fail(EXL3_EINVAL, "workspace too small: need %zu bytes, got %zu", b.total, workspace_bytes);
  if (!aligned16(workspace)) return fail(EXL3_EINVAL, "attention workspace must be 16-byte aligned");
  if (b.types[1] != b.types[2])
    return fail(EXL3_EUNSUPPORTED, "keys and values of an attention block have one type: both biased or neither");
  if (!rope && b.types[0] != x_type)
    return fail(EXL3_EUNSUPPORTED, "biased bf16 queries need a rotation, which rounds them");
  uint8_t* ws = (uint8_t*)workspace;
  const exl3_linear* parts[3] = {q, k, v};
  void* qkv[3] = {ws + b.part[0], ws + b.part[1], ws + b.part[2]};
  void* query = b.types[0] == x_type ? qkv[0] : ws + b.rounded;
  const int D = cache->view.head_dim;
  const int64_t wide = (int64_t)b.heads * D, narrow = (int64_t)cache->view.kv_heads * D;
  auto turn = [&](bool run) {
    return rope ? rope_call(rope, qkv[0], b.types[0], rows, b.heads, D, wide, nullptr, batch, query, x_type, wide,
                            stream, run)
                : (int)EXL3_OK;
  };
  auto append = [&](bool run) {
    return append_call(cache, batch, qkv[1], narrow, qkv[2], narrow, b.types[1], rows, rope, stream, run);
  };
  auto attend = [&](bool run) {
    return attention_call(cache, batch, query, x_type, rows, b.heads, wide, scale, 1, window, scores, query, wide,
                          ws + b.attention, b.total - b.attention, stream, run);
  };
  // what a later part would refuse is refused before the first one's launch (the group's own
  // checks come before that)
  if (int rc = turn(false)) return rc;
  if (int rc = append(false)) return rc;
  if (int rc = attend(false)) return rc;
  if (int rc = check_linear_rows(o, rows)) return rc;
  if (int rc = exl3_group_forward(parts, 3, x, x_type, rows, qkv, ws, b.linear, stream)) return rc;
  if (int rc = turn(true)) return rc;
  if (int rc = append(true)) return rc;
  if (int rc = attend(true)) return rc;
  return exl3_linear_forward(o, query, x_type, rows, y, exl3_linear_output_dtype(o, x_type), ws, b.linear,
                             stream);
}

extern "C" int exl3_attn_block_forward(const exl3_linear* q, const exl3_linear* k,
                                       const exl3_linear* v, const exl3_linear* o,
                                       const exl3_kv_cache* cache, const exl3_kv_batch* batch,
                                       const exl3_rope_spec* rope, float scale, int32_t window,
                                       const void* x, int32_t x_type, int64_t rows, void* y,
                                       void* workspace, size_t workspace_bytes, void* stream) {
  return exl3_attn_block_forward_scores(q, k, v, o, cache, batch, rope, scale, window, nullptr, x, x_type, rows, y,
                                        workspace, workspace_bytes, stream);
}

#endif  // __HIP_DEVICE_COMPILE__
