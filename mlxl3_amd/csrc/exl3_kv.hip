// Rotary positions, and writing and reading the paged key/value cache (layout:
// exl3_kv.hpp).
//
// Rotation: channel pairs (a, b) of a head turn by t = p * f_i,
//   (a, b) -> (a c - b s, a s + b c),  c = m cos t,  s = m sin t.
// t and its cosine and sine are formed in 64 bits and rounded to f32 once (at
// p = 100000 an f32 product alone is off by 0.004 rad); the products and their sum are
// f32.  A workgroup computes the cosines and sines of its tokens once, in LDS, for its
// heads.  Memory bounds it: 4096 tokens of 40 bf16 heads of 128, 64 channels rotated, take
// 16.5 us, 5.1 TB/s read and written (a copy of as many bytes 18.5).  One token of 32 heads
// takes 4, most of it the launch.
//
// Quantisation: 32 neighbouring channels of a head share the f16 scale
//   s = f16(max|x| / 127)  (4 bits: / 7),  at most 65504,
// and store code = rint(x / s) (ties to even), clipped to +-127 (+-7); s = 0 stores
// zeros.  A group with a NaN or an infinity gets s = NaN, so that it reads back as
// NaN.  Everything is f32 with one rounding per operation, the quotient correctly
// rounded, so the codes do not depend on how the work is laid out.
//
// Writing 4096 tokens of 8 heads of 128, keys rotated, takes 11 us (values in the caches) to
// 12.5: to 16 bits 3.1 TB/s, to 8 bits 2.3.  What bounds it is one short-lived workgroup's
// chain of dependent steps -- where its tokens belong, their turns, their page, the scale --
// which four workgroups a CU do not hide, and a thousand vector instructions a wave beside it.
// Written and read back, 4096 tokens take 19.3 us, 64 sequences' tokens 7.7, one token 6.3:
// two launches with that chain each.
// Reading 60059 tokens of two sequences back from 4 bits as f16 takes 56 us, 5.6 TB/s; the
// writes alone (246 MB) take 37 in a plain fill.  Stores that bypass the caches take
// 5 us off it and put as many on whoever reads the values next: not used.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <new>
#include <type_traits>

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
  const int q = (int)(k - 4.0 * floor(0.25 * k));
  const double a = q & 1 ? c : s, b = q & 1 ? s : c;
  *s_out = q & 2 ? -a : a;
  *c_out = (q + 1) & 2 ? -b : b;
}

struct RopeView {
  const float* freq;  // [pairs]; null: no rotation
  int pairs, interleaved;
  double scale;
};

// Cosines and sines of a workgroup's tokens, [tokens][stride] in LDS.  A thread has one pair:
// its frequency is loaded once, early, beside the workgroup's other first loads.
struct RopeTable {
  int pair, token, step;  // the thread's pair and first token, tokens at a time
  float freq;
  __device__ __forceinline__ RopeTable(const RopeView& r, int pairs) {
    step = 256 / max(pairs, 1);
    token = threadIdx.x / max(pairs, 1);
    pair = threadIdx.x - token * pairs;
    freq = pairs && token < step ? r.freq[pair] : 0.0f;
  }
  __device__ __forceinline__ void fill(const RopeView& r, const int64_t* positions, int tokens, float2* cs,
                                       int stride) const {
    if (token >= step) return;
    for (int t = token; t < tokens; t += step) {
      double s, c;
      sincos64((double)positions[t] * (double)freq, &s, &c);
      cs[t * stride + pair] = make_float2((float)(c * r.scale), (float)(s * r.scale));
    }
  }
};

constexpr int kBatch = 4;     // heads whose loads a thread has in flight

struct RopeParams {
  const void* x;
  void* y;
  const int32_t* positions;  // null: positions of the batch
  KvBatchView batch;
  RopeView rope;
  int64_t tokens, x_stride, y_stride;
  int heads, head_dim, x_type, y_type;
  int lanes;  // per token: a thread's channels (below) are the same in all heads
  int per;    // heads of a workgroup
};

// grid (tokens / (256 / lanes), heads / per).  A thread has, of one token's heads in turn,
// VEC: eight pairs (two chunks of eight channels, or one chunk of neighbours) or a chunk
// behind the rotated channels; else one pair or one channel.  Its cosines and sines stay in
// registers.  It loads all it needs of a head before it stores, so y may be x.  BYTES: of a
// value of x (VEC).
template <bool VEC, int BYTES>
__global__ __launch_bounds__(256) void rope_kernel(RopeParams p) {
  __shared__ float2 cs[2048];        // [tokens][pairs]: at most 8 pairs a lane
  __shared__ int64_t position[256];
  constexpr int W = VEC ? 8 : 1;
  const int L = p.lanes, most = 256 / L, r = p.rope.pairs;
  const int64_t t0 = (int64_t)blockIdx.x * most;
  const int nt = (int)min((int64_t)most, p.tokens - t0);
  const int t = threadIdx.x / L, c = threadIdx.x - t * L;
  const bool two = !p.rope.interleaved;  // the pair's second half lies r channels further
  const int turned = VEC && !two ? 2 * r / W : r / W;
  const bool tail = c >= turned;
  const RopeTable turns(p.rope, r);
  bool on = t < nt;
  int64_t pos = 0;
  if (p.positions) {
    if (on) pos = p.positions[t0 + t];
  } else {
    const int first = __builtin_amdgcn_readfirstlane(t), last = min(__builtin_amdgcn_readlane(t, 63), nt - 1);
    const KvToken at = kv_locate(p.batch, t0 + first, last - first + 1, t - first);
    pos = at.pos;
    on = on && at.seq >= 0;
  }
  const int h0 = blockIdx.y * p.per, h1 = min(h0 + p.per, p.heads);
  const int da = tail ? 2 * r + (c - turned) * W : !two ? c * (VEC ? 8 : 2) : c * W;
  const int db = two ? da + r : da + 1;  // db: not with neighbours of a chunk
  const size_t xr = (size_t)(t0 + t) * p.x_stride, yr = (size_t)(t0 + t) * p.y_stride;
  Raw8<BYTES> a[VEC ? kBatch : 1], b[VEC ? kBatch : 1];
  float fa[VEC ? 1 : kBatch], fb[VEC ? 1 : kBatch];
  auto load = [&](int h) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (!on || h + u >= h1) continue;
      const size_t row = xr + (size_t)(h + u) * p.head_dim;
      if constexpr (VEC) {
        a[u].load(p.x, row + da, true);
        if (two && !tail) b[u].load(p.x, row + db, true);
      } else {
        fa[u] = load1(p.x, p.x_type, row + da);
        if (!tail) fb[u] = load1(p.x, p.x_type, row + db);
      }
    }
  };
  load(h0);
  if (c == 0 && t < nt) position[t] = pos;
  __syncthreads();
  turns.fill(p.rope, position, nt, cs, r);
  __syncthreads();
  if (!on || (tail && p.x == p.y)) return;
  constexpr int N = VEC ? 8 : 1;
  float2 f[N];
#pragma unroll
  for (int n = 0; n < N; ++n) f[n] = cs[tail ? 0 : min(t * r + (two ? c * W : c * (VEC ? 4 : 1)) + n, 2047)];
  for (int h = h0; h < h1; h += kBatch) {
    if (h > h0) load(h);
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (h + u >= h1) continue;
      const size_t row = yr + (size_t)(h + u) * p.head_dim;
      if constexpr (VEC) {
        float x[8], z[8];
        a[u].get(p.x_type, x);
        if (!tail && two) {
          b[u].get(p.x_type, z);
#pragma unroll
          for (int n = 0; n < 8; ++n) {
            const float v = x[n], w = z[n];
            x[n] = v * f[n].x - w * f[n].y;
            z[n] = v * f[n].y + w * f[n].x;
          }
          store8(p.y, p.y_type, row + db, z);
        } else if (!tail) {
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const float v = x[2 * n], w = x[2 * n + 1];
            x[2 * n] = v * f[n].x - w * f[n].y;
            x[2 * n + 1] = v * f[n].y + w * f[n].x;
          }
        }
        store8(p.y, p.y_type, row + da, x);
      } else if (tail) {
        store1(p.y, p.y_type, row + da, fa[u]);
      } else {
        store1(p.y, p.y_type, row + da, fa[u] * f[0].x - fb[u] * f[0].y);
        store1(p.y, p.y_type, row + db, fa[u] * f[0].y + fb[u] * f[0].x);
      }
    }
  }
}

// The host code below is left out of the device pass, which needs the instances spelled out.
template __global__ void rope_kernel<true, 2>(RopeParams);
template __global__ void rope_kernel<true, 4>(RopeParams);
template __global__ void rope_kernel<false, 2>(RopeParams);

// The scale of a group whose largest magnitude is `most` (NaN where it is not finite).
__device__ __forceinline__ uint16_t group_scale(float most, float levels) {
  if (!(most <= 3.402823466e38f)) return 0x7e00;
  return f2h(fminf(most / levels, 65504.0f));
}

// rint(x / s) clipped to +-levels, plus levels + 1, in the low byte: the quotient from the
// rounded reciprocal and one residual step, which rounds it correctly (s is an f16 value, so
// neither the reciprocal nor the residual under- or overflows where the clip does not
// decide); a sum of that size rounds to whole numbers, ties to even.
__device__ __forceinline__ uint32_t group_code(float x, float s, float inv, float levels) {
  float q = x * inv;
  q = fmaf(fmaf(-q, s, x), inv, q);
  q = __builtin_amdgcn_fmed3f(q, -levels, levels) + (12582912.0f + levels + 1.0f);
  return __builtin_bit_cast(uint32_t, q);
}
// Four low bytes as one word.
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x0c0c0400u), hi = __builtin_amdgcn_perm(d, c, 0x04000c0cu);
  return lo | hi;
}

struct AppendParams {
  KvCacheView cache;
  KvBatchView batch;
  RopeView rope;
  const void *k, *v;
  int64_t tokens, k_stride, v_stride;
  int type, vec;     // vec: rows of k and v are 16-byte aligned
  int heads, parts;  // heads of a workgroup, and workgroups for all heads of a side
};

// The workgroups of an append or a read: 256 / (D / 8) tokens each (a thread has eight
// channels of one token), blockIdx.y the keys' or values' side and a few heads.
template <int D>
struct Tile {
  static constexpr int kLanes = D / 8, kTokens = 256 / kLanes;
  int token, d0;     // the thread's token in the workgroup and its first channel
  bool value;
  int h0, h1;
  __device__ __forceinline__ Tile(int heads, int parts, int kv_heads) {
    token = threadIdx.x / kLanes;
    d0 = (threadIdx.x % kLanes) * 8;
    value = (int)blockIdx.y >= parts;
    h0 = ((int)blockIdx.y - (value ? parts : 0)) * heads;
    h1 = min(h0 + heads, kv_heads);
  }
  // The thread's token, or seq = -1 behind the last.
  __device__ __forceinline__ KvToken locate(const KvBatchView& b, int64_t t0, int64_t tokens) const {
    constexpr int n = 64 / kLanes;  // tokens of a wave
    const int first = __builtin_amdgcn_readfirstlane(token);
    return kv_locate(b, t0 + first, (int)min((int64_t)n, tokens - t0 - first), token - first);
  }
};

// grid (tokens, sides x parts): a quantised group is the channels of four neighbouring
// lanes.  A token's values are read where they lie, its rotation's other half a second time
// (from the caches), and all loads of a workgroup start before it looks for its tokens.
template <int FMT, int D, int BYTES>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendParams p) {
  typedef Tile<D> W;
  __shared__ float2 cs[W::kTokens][D / 2];
  __shared__ int64_t positions[W::kTokens];
  const KvCacheView& c = p.cache;
  const W w(p.heads, p.parts, c.kv_heads);
  const int64_t t0 = (int64_t)blockIdx.x * W::kTokens;
  const int nt = (int)min((int64_t)W::kTokens, p.tokens - t0);
  const int r = p.rope.freq && !w.value ? p.rope.pairs : 0;
  const bool half = !p.rope.interleaved && r % 8 == 0 && w.d0 < 2 * r, second = w.d0 >= r;
  const void* src = w.value ? p.v : p.k;
  const size_t row = (size_t)(t0 + w.token) * (w.value ? p.v_stride : p.k_stride) + w.d0;
  Raw8<BYTES> x[kBatch], other[kBatch];
  auto load = [&](int h0) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (h0 + u >= w.h1 || w.token >= nt) continue;
      const size_t at = row + (size_t)(h0 + u) * D;
      x[u].load(src, at, p.vec);
      if (half) other[u].load(src, second ? at - r : at + r, p.vec);
    }
  };
  const RopeTable turns(p.rope, r);
  load(w.h0);
  const KvToken at = w.locate(p.batch, t0, p.tokens);
  if (r) {
    if (w.d0 == 0) positions[w.token] = at.pos;
    __syncthreads();
    turns.fill(p.rope, positions, nt, cs[0], D / 2);
    __syncthreads();
  }
  const int64_t page = at.seq < 0 ? -1 : kv_page(c, p.batch, at.seq, at.pos);
  if (page < 0) return;  // all lanes of a token leave together
  const int slot = (int)(at.pos & ((1 << c.page_shift) - 1));
  const float2* f = cs[w.token];
  for (int h0 = w.h0; h0 < w.h1; h0 += kBatch) {
    if (h0 > w.h0) load(h0);
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (h0 + u >= w.h1) continue;
      float v[8];
      x[u].get(p.type, v);
      if (w.d0 < 2 * r) {
        if (p.rope.interleaved) {
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            if (w.d0 / 2 + n < r) {
              const float2 g = f[w.d0 / 2 + n];
              const float a = v[2 * n], b = v[2 * n + 1];
              v[2 * n] = a * g.x - b * g.y;
              v[2 * n + 1] = a * g.y + b * g.x;
            }
          }
        } else if (half) {
          float o[8];
          other[u].get(p.type, o);
#pragma unroll
          for (int n = 0; n < 8; ++n) {
            const float2 g = f[second ? w.d0 - r + n : w.d0 + n];
            v[n] = second ? o[n] * g.y + v[n] * g.x : v[n] * g.x - o[n] * g.y;
          }
        } else {
#pragma unroll 1
          for (int n = 0; n < 8; ++n) {
            const int d = w.d0 + n;
            if (d >= 2 * r) break;
            const bool back = d >= r;
            const float2 g = f[back ? d - r : d];
            const size_t i = row - w.d0 + (size_t)(h0 + u) * D;
            const float a = load1(src, p.type, i + d), o = load1(src, p.type, i + (back ? d - r : d + r));
            const float turned = back ? o * g.y + a * g.x : a * g.x - o * g.y;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = e == n ? turned : v[e];
          }
        }
      }
      const size_t head = (size_t)page * c.kv_heads + h0 + u;
      const size_t token = (head << c.page_shift) + slot;  // row of D values
      uint8_t* base = w.value ? c.v : c.k;
      if constexpr (FMT >= 9) {
        store8(base, FMT, token * D + w.d0, v);
      } else {
        float most = 0.0f;
        bool whole = true;  // fmaxf drops a NaN
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          most = fmaxf(most, fabsf(v[n]));
          whole = whole && fabsf(v[n]) <= 3.402823466e38f;
        }
        if (!whole) most = __builtin_inff();
        most = fmaxf(most, xor_lanes<1>(most));
        most = fmaxf(most, xor_lanes<2>(most));
        constexpr float levels = FMT == KV_Q8 ? 127.0f : 7.0f;
        const uint16_t sh = group_scale(most, levels);
        const float s = h2f(sh);
        const bool on = s > 0.0f;
        const float inv = on ? 1.0f / s : 0.0f;
        uint32_t code[8];
#pragma unroll
        for (int n = 0; n < 8; ++n) code[n] = group_code(v[n], s, inv, levels);
        if constexpr (FMT == KV_Q8) {
          const uint32_t zero = 0x80808080u;
          const u32x2 o = {on ? low_bytes(code[0], code[1], code[2], code[3]) : zero,
                           on ? low_bytes(code[4], code[5], code[6], code[7]) : zero};
          *(u32x2*)(base + token * D + w.d0) = o;
        } else {
          // a byte each: the even channel's nibble, and the odd one's above it
          const uint32_t even = low_bytes(code[0], code[2], code[4], code[6]) & 0x0f0f0f0fu;
          const uint32_t odd = low_bytes(code[1], code[3], code[5], code[7]) & 0x0f0f0f0fu;
          *(uint32_t*)(base + (token * D + w.d0) / 2) = on ? even | odd << 4 : 0x88888888u;
        }
        if ((w.d0 & 31) == 0) {
          uint16_t* sc = w.value ? c.vs : c.ks;
          sc[((head * (D / 32) + w.d0 / 32) << c.page_shift) + slot] = sh;
        }
      }
    }
  }
}

struct ReadParams {
  KvCacheView cache;
  KvBatchView batch;
  void *k, *v;
  int64_t tokens;
  int type, heads, parts;
};

// The workgroups of kv_append_kernel, the other way.
template <int FMT, int D>
__global__ __launch_bounds__(256) void kv_read_kernel(ReadParams p) {
  typedef Tile<D> W;
  constexpr int kWords = FMT >= 9 ? 4 : FMT == KV_Q8 ? 2 : 1;
  const KvCacheView& c = p.cache;
  const W w(p.heads, p.parts, c.kv_heads);
  const int64_t t0 = (int64_t)blockIdx.x * W::kTokens;
  const KvToken at = w.locate(p.batch, t0, p.tokens);
  if (at.seq < 0) return;
  const int64_t page = kv_page(c, p.batch, at.seq, at.pos);  // a token without one reads as zeros
  const int slot = (int)(at.pos & ((1 << c.page_shift) - 1));
  const uint8_t* base = w.value ? c.v : c.k;
  const uint16_t* scales = w.value ? c.vs : c.ks;
  for (int h0 = w.h0; h0 < w.h1; h0 += kBatch) {
    uint32_t x[kBatch][kWords];
    uint16_t scale[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const size_t head = (size_t)max(page, (int64_t)0) * c.kv_heads + min(h0 + u, w.h1 - 1);
      const size_t token = (head << c.page_shift) + slot;
      const uint8_t* from = base + (token * D + w.d0) * kWords / 2;
      if constexpr (kWords == 4) {
        const u32x4 q = *(const u32x4*)from;
#pragma unroll
        for (int n = 0; n < 4; ++n) x[u][n] = q[n];
      } else if constexpr (kWords == 2) {
        const u32x2 q = *(const u32x2*)from;
        x[u][0] = q[0];
        x[u][1] = q[1];
      } else {
        x[u][0] = *(const uint32_t*)from;
      }
      if constexpr (FMT < 9) scale[u] = scales[((head * (D / 32) + w.d0 / 32) << c.page_shift) + slot];
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (h0 + u >= w.h1) continue;
      void* out = w.value ? p.v : p.k;
      const size_t at = ((size_t)(t0 + w.token) * c.kv_heads + h0 + u) * D + w.d0;
      if (p.type == DT_F16) {
        // code * scale is rounded once either way: in f16 arithmetic, two at a time
        u32x4 o;
        if constexpr (FMT == KV_F16) {
          o = u32x4{x[u][0], x[u][1], x[u][2], x[u][3]};
        } else if constexpr (FMT == KV_BF16) {
#pragma unroll
          for (int n = 0; n < 4; ++n) o[n] = pack2(DT_F16, bf2f((uint16_t)x[u][n]), bf2f((uint16_t)(x[u][n] >> 16)));
        } else {
          const _Float16 s = __builtin_bit_cast(_Float16, scale[u]);
          if constexpr (FMT == KV_Q8)
            o = decode8(x[u][0], x[u][1], s);
          else
            o = decode4(x[u][0], s);
        }
        if (page < 0) o = u32x4{0, 0, 0, 0};
        *(u32x4*)((uint16_t*)out + at) = o;
        continue;
      }
      float y[8];
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        if constexpr (FMT == KV_Q8) {
          y[n] = (float)((int)((x[u][n / 4] >> (8 * (n & 3))) & 255) - 128) * h2f(scale[u]);
        } else if constexpr (FMT == KV_Q4) {
          y[n] = (float)((int)((x[u][0] >> (4 * n)) & 15) - 8) * h2f(scale[u]);
        } else {
          const uint16_t v = (uint16_t)(x[u][n / 2] >> (16 * (n & 1)));
          y[n] = FMT == KV_F16 ? h2f(v) : bf2f(v);
        }
        y[n] = page >= 0 ? y[n] : 0.0f;
      }
      store8(out, p.type, at, y);
    }
  }
}

#define EXL3_KV_D(M, FMT) M(FMT, 64) M(FMT, 128) M(FMT, 256)
#define EXL3_KV(M) EXL3_KV_D(M, KV_F16) EXL3_KV_D(M, KV_BF16) EXL3_KV_D(M, KV_Q8) EXL3_KV_D(M, KV_Q4)
#define EXL3_KV_INST(FMT, D)                                        \
  template __global__ void kv_append_kernel<FMT, D, 2>(AppendParams); \
  template __global__ void kv_append_kernel<FMT, D, 4>(AppendParams); \
  template __global__ void kv_read_kernel<FMT, D>(ReadParams);
EXL3_KV(EXL3_KV_INST)

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

// Heads per workgroup of an append or a read: a batch of loads each while that leaves
// four workgroups per CU.  4096 tokens of 8 heads, 8 bits, written and read back: 4 heads each
// 20.2 us; 2 heads 22.8 and 1 head 30.1 (the turns are computed for each), 8 heads 22.2.
static int head_parts(int64_t tokens, const KvCacheView& c, dim3* grid, int* heads, int* parts) {
  const int64_t n = (tokens + 2048 / c.head_dim - 1) / (2048 / c.head_dim);
  if (n > kMostBlocks) return fail(EXL3_EUNSUPPORTED, "too many tokens: %lld", (long long)tokens);
  int per = kBatch;
  while (per > 1 && n * 2 * ((c.kv_heads + per - 1) / per) < 1024) per /= 2;
  *heads = per;
  *parts = (c.kv_heads + per - 1) / per;
  *grid = dim3((unsigned)n, 2u * (unsigned)*parts);
  return EXL3_OK;
}

// f(format, head width) as template arguments of f.
template <typename F>
static void by_format(const KvCacheView& c, F&& f) {
  auto width = [&](auto fmt) {
    if (c.head_dim == 64)
      f(fmt, std::integral_constant<int, 64>{});
    else if (c.head_dim == 128)
      f(fmt, std::integral_constant<int, 128>{});
    else
      f(fmt, std::integral_constant<int, 256>{});
  };
  switch (c.format) {
    case EXL3_KV_F16: width(std::integral_constant<int, KV_F16>{}); break;
    case EXL3_KV_BF16: width(std::integral_constant<int, KV_BF16>{}); break;
    case EXL3_KV_Q8: width(std::integral_constant<int, KV_Q8>{}); break;
    default: width(std::integral_constant<int, KV_Q4>{});
  }
}

int exl3::rope_call(const exl3_rope_spec* rope, const void* x, int32_t x_type, int64_t tokens,
                    int32_t heads, int32_t head_dim, int64_t x_stride, const int32_t* positions,
                    const exl3_kv_batch* batch, void* y, int32_t y_type, int64_t y_stride,
                    void* stream, bool launch) {
  if (!rope) return fail(EXL3_EINVAL, "null rotary spec");
  if (tokens < 0) return fail(EXL3_EINVAL, "negative token count");
  if (!known_type(x_type) || !known_type(y_type))
    return fail(EXL3_EINVAL, "unsupported rotary dtypes %d and %d", x_type, y_type);
  if (heads < 1 || heads > 65536 || head_dim < 2 || head_dim > 256)
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
  const int pairs = p.rope.pairs, chunk = vec ? 8 : 1;
  p.lanes = (p.rope.interleaved && vec ? 2 * pairs : pairs) / chunk + (head_dim - 2 * pairs) / chunk;
  const int64_t blocks = (tokens + 256 / p.lanes - 1) / (256 / p.lanes);
  if (blocks > kMostBlocks) return fail(EXL3_EUNSUPPORTED, "too many tokens: %lld", (long long)tokens);
  // two batches of loads a thread while that leaves two workgroups per CU.  40 heads of 128,
  // us: 4096 tokens 16.5 (one batch 17.0, four 16.5); 1000 tokens 7.2 (four workgroups a CU
  // 8.1, eight 10.6: the turns are computed for each); 64 tokens 4.2 (3.9, 4.0)
  p.per = 2 * kBatch;
  while (p.per > 1 && blocks * ((heads + p.per - 1) / p.per) < 512) p.per /= 2;
  const dim3 grid((unsigned)blocks, (unsigned)((heads + p.per - 1) / p.per));
  if (!launch) return EXL3_OK;
  if (int rc = launch_gate("rotary launch")) return rc;
  hipStream_t s = (hipStream_t)stream;
  if (vec && x_type == EXL3_F32)
    hipLaunchKernelGGL((rope_kernel<true, 4>), grid, dim3(256), 0, s, p);
  else if (vec)
    hipLaunchKernelGGL((rope_kernel<true, 2>), grid, dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL((rope_kernel<false, 2>), grid, dim3(256), 0, s, p);
  return check_launch("rotary launch");
}

extern "C" int exl3_rope(const exl3_rope_spec* rope, const void* x, int32_t x_type, int64_t tokens,
                         int32_t heads, int32_t head_dim, int64_t x_stride,
                         const int32_t* positions, const exl3_kv_batch* batch, void* y,
                         int32_t y_type, int64_t y_stride, void* stream) {
  return rope_call(rope, x, x_type, tokens, heads, head_dim, x_stride, positions, batch, y, y_type, y_stride,
                   stream, true);
}

int exl3::append_call(const exl3_kv_cache* cache, const exl3_kv_batch* batch, const void* k,
                      int64_t k_stride, const void* v, int64_t v_stride, int32_t type,
                      int64_t tokens, const exl3_rope_spec* rope, void* stream, bool launch) {
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
  dim3 grid;
  if (int rc = head_parts(tokens, p.cache, &grid, &p.heads, &p.parts)) return rc;
  p.k = k;
  p.v = v;
  p.tokens = tokens;
  p.k_stride = k_stride;
  p.v_stride = v_stride;
  p.type = type;
  p.vec = rows_aligned(k, tokens > 1 ? k_stride : 0, type) &&
          rows_aligned(v, tokens > 1 ? v_stride : 0, type);
  if (!launch) return EXL3_OK;
  if (int rc = launch_gate("KV append")) return rc;
  by_format(p.cache, [&](auto fmt, auto dim) {
    if (type == EXL3_F32)
      hipLaunchKernelGGL((kv_append_kernel<fmt(), dim(), 4>), grid, dim3(256), 0, (hipStream_t)stream, p);
    else
      hipLaunchKernelGGL((kv_append_kernel<fmt(), dim(), 2>), grid, dim3(256), 0, (hipStream_t)stream, p);
  });
  return check_launch("KV append");
}

extern "C" int exl3_kv_append(const exl3_kv_cache* cache, const exl3_kv_batch* batch,
                              const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                              int32_t type, int64_t tokens, const exl3_rope_spec* rope,
                              void* stream) {
  return append_call(cache, batch, k, k_stride, v, v_stride, type, tokens, rope, stream, true);
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
  dim3 grid;
  if (int rc = head_parts(tokens, p.cache, &grid, &p.heads, &p.parts)) return rc;
  p.k = k;
  p.v = v;
  p.tokens = tokens;
  p.type = type;
  if (int rc = launch_gate("KV read")) return rc;
  by_format(p.cache, [&](auto fmt, auto dim) {
    hipLaunchKernelGGL((kv_read_kernel<fmt(), dim()>), grid, dim3(256), 0, (hipStream_t)stream, p);
  });
  return check_launch("KV read");
}

#endif  // __HIP_DEVICE_COMPILE__
