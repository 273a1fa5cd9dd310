// Root-mean-square norm of rows, with the residual's addition:
//
//   s = x + r   (without a residual x)      total = s, rounded to r's type
//   y = s * rsqrt(sum s^2 / width + eps) * w
//
// s is f32 and not rounded on the way to y, the sum of squares is f32: up to 8 V squares in
// a lane, then a tree.  Memory bounds it (every value is read and written once), so a row stays in
// registers between its sum and its outputs: T threads hold 8 V values each, as few as do.  Rows of more
// than 32768 values are read again instead (from the caches).
//
// Measured in a graph, inputs not in the caches: 4096 rows of 4096 bf16 values with an f32 residual 36 us,
// 5.6 TB/s (a large copy: 5.1; a call from Python among others 39.9, of which the kernel 33.7), of 8192 with half the rows 39, of 2048 with twice as many 35, of 1024 35; with a
// bf16 residual 26; 20000 tokens' 32 heads of 128 f16 values, without one, 65 us, 5.0 TB/s, 2001 tokens'
// 9.5.  One row of 4096 takes 3.4, a launch and one round trip to memory.
//
// A sum that overflows is formed again from values 2^-100 times smaller: bf16 and f32 rows
// beyond 1e18 are right.  A row that holds an infinity gives NaN in its place and zeros
// elsewhere, a NaN makes the row NaN.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/exl3_hip.h"
#include "exl3_kv.hpp"
#include "exl3_kv_host.hpp"
#include "exl3_launch.hpp"

namespace exl3 {

struct NormParams {
  const void *x, *w, *r;  // w, r: null where there is none
  void *y, *total;        // total: null where nobody wants it
  int64_t rows, x_stride, r_stride, y_stride, total_stride;  // of tokens, in elements
  int heads, width;       // row = token * heads + head, heads contiguous
  int x_type, w_type, r_type, y_type;
  float eps;
};

// The sum of v over the T threads of a row, the same in all of them.
template <int T>
__device__ __forceinline__ float row_sum(float v, float* parts) {
  v += xor_lanes<1>(v);
  v += xor_lanes<2>(v);
  v += xor_lanes<4>(v);
  if constexpr (T >= 16) v += xor_lanes<8>(v);
  if constexpr (T >= 32) v += xor_lanes<16>(v);
  if constexpr (T >= 64) v += xor_lanes<32>(v);
  if constexpr (T > 64) {
    if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < T / 64; ++i) v += parts[i];
    __syncthreads();
  }
  return v;
}

// Eight neighbouring values of a row, from value `at` of `width`.  WHOLE: the row's chunks are whole and
// 16-byte aligned; else they lie as they lie, in memory instructions as wide, and the last one is
// loaded and stored value by value (3276 rows of 5121 bf16 values with an f32 residual 40 us, all of
// it value by value 131; rows of 5120, whole: 37).
template <int BYTES, bool WHOLE>
struct Chunk : Raw8<BYTES> {
  __device__ __forceinline__ void load(const void* p, size_t row, int at, int width) {
    const uint8_t* from = (const uint8_t*)p + (row + at) * BYTES;
    if (WHOLE || at + 8 <= width) {
#pragma unroll
      for (int j = 0; j < BYTES / 2; ++j) {
        if constexpr (WHOLE)
          this->w[j] = ((const u32x4*)from)[j];
        else
          __builtin_memcpy(&this->w[j], from + 16 * j, 16);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        uint32_t v = 0;
        if (at + e < width) v = BYTES == 4 ? ((const uint32_t*)from)[e] : ((const uint16_t*)from)[e];
        if constexpr (BYTES == 4)
          this->w[e / 4][e % 4] = v;
        else if (e % 2 == 0)
          this->w[0][e / 2] = v;
        else
          this->w[0][e / 2] |= v << 16;
      }
    }
  }
};
template <bool WHOLE>
__device__ __forceinline__ void store_chunk(void* p, int type, size_t row, int at, int width, const float (&x)[8]) {
  if constexpr (WHOLE) {
    store8(p, type, row + at, x);
  } else if (at + 8 <= width) {
    if (type == DT_F32) {
      __builtin_memcpy((float*)p + row + at, x, 32);
    } else {
      u32x4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = pack2(type, x[2 * e], x[2 * e + 1]);
      __builtin_memcpy((uint16_t*)p + row + at, &w, 16);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (at + e < width) store1(p, type, row + at + e, x[e]);
  }
}

// XB, RB: bytes of x and of the residual (0: none).  LOOP: rows that registers do not hold, V chunks
// a thread at a time.
template <bool WHOLE, int XB, int RB, int T, int V, bool LOOP>
__global__ __launch_bounds__(T < 256 ? 256 : T) void rms_norm_kernel(NormParams p) {
  __shared__ float parts[T > 64 ? T / 64 : 1];
  const int t = threadIdx.x % T;
  const int64_t row = (int64_t)blockIdx.x * (T < 256 ? 256 / T : 1) + threadIdx.x / T;
  const bool on = T >= 256 || row < p.rows;
  const int64_t token = p.heads == 1 ? row : row / p.heads;
  const size_t in_token = p.heads == 1 ? 0 : (size_t)(row - token * p.heads) * p.width;
  const size_t xr = (size_t)token * p.x_stride + in_token, rr = (size_t)token * p.r_stride + in_token;
  const size_t yr = (size_t)token * p.y_stride + in_token, tr = (size_t)token * p.total_stride + in_token;
  float s[V][8];
  // chunk c of the thread, the lanes' chunks side by side; outside the row: none
  auto place = [&](int from, int c) { return from + (c * T + t) * 8; };
  auto load = [&](int from) __attribute__((always_inline)) {
    Chunk<XB, WHOLE> x[V];
    Chunk<RB ? RB : 2, WHOLE> r[V];
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const int at = place(from, c);
      if (!on || at >= p.width) continue;
      x[c].load(p.x, xr, at, p.width);
      if (RB) r[c].load(p.r, rr, at, p.width);
    }
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const bool in = on && place(from, c) < p.width;
      float b[8];
      x[c].get(p.x_type, s[c]);
      if (RB) r[c].get(p.r_type, b);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[c][e] = in ? RB ? s[c][e] + b[e] : s[c][e] : 0.0f;
    }
  };
  auto square_sum = [&](float f) __attribute__((always_inline)) {
    float sum = 0.0f;
    for (int from = 0; from < (LOOP ? p.width : 1); from += 8 * T * V) {
      if constexpr (LOOP) load(from);
      float part = 0.0f;
#pragma unroll
      for (int c = 0; c < V; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float v = s[c][e] * f;
          part = fmaf(v, v, part);
        }
      sum += part;
    }
    return row_sum<T>(sum, parts);
  };
  if constexpr (!LOOP) load(0);
  const float sum = square_sum(1.0f);
  float inv = __builtin_amdgcn_rsqf(sum / (float)p.width + p.eps), unit = 1.0f;  // y = s unit inv w
  bool over = !(sum <= 3.402823466e38f);
  if constexpr (T < 64) over = __any(over);
  if (over) {
    const float small = square_sum(7.888609052e-31f);  // 2^-100
    if (!(sum <= 3.402823466e38f) && small <= 3.402823466e38f) {
      inv = (float)(1.0 / sqrt((double)small / p.width + (double)p.eps * 0x1p-200));
      unit = 7.888609052e-31f;
    }
  }
  for (int from = 0; from < (LOOP ? p.width : 1); from += 8 * T * V) {
    if constexpr (LOOP) load(from);
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const int at = place(from, c);
      if (!on || at >= p.width) continue;
      if (RB && p.total) store_chunk<WHOLE>(p.total, p.r_type, tr, at, p.width, s[c]);
      float w[8];
      if (p.w) {
        if (p.w_type == DT_F32) {
          Chunk<4, WHOLE> raw;
          raw.load(p.w, 0, at, p.width);
          raw.get(p.w_type, w);
        } else {
          Chunk<2, WHOLE> raw;
          raw.load(p.w, 0, at, p.width);
          raw.get(p.w_type, w);
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s[c][e] *= unit;
        s[c][e] *= inv;
        if (p.w) s[c][e] *= w[e];
      }
      store_chunk<WHOLE>(p.y, p.y_type, yr, at, p.width, s[c]);
    }
  }
}

#define EXL3_NORM_T(M, WHOLE, XB, RB)                                                                \
  M(WHOLE, XB, RB, 8, 1, false) M(WHOLE, XB, RB, 16, 1, false) M(WHOLE, XB, RB, 32, 1, false)        \
  M(WHOLE, XB, RB, 64, 1, false) M(WHOLE, XB, RB, 256, 1, false)                                     \
  M(WHOLE, XB, RB, 256, 2, false) M(WHOLE, XB, RB, 256, 4, false) M(WHOLE, XB, RB, 1024, 2, false)   \
  M(WHOLE, XB, RB, 1024, 4, false) M(WHOLE, XB, RB, 1024, 4, true)
#define EXL3_NORM_B(M, WHOLE)                                                                        \
  EXL3_NORM_T(M, WHOLE, 2, 0) EXL3_NORM_T(M, WHOLE, 2, 2) EXL3_NORM_T(M, WHOLE, 2, 4)                \
  EXL3_NORM_T(M, WHOLE, 4, 0) EXL3_NORM_T(M, WHOLE, 4, 2) EXL3_NORM_T(M, WHOLE, 4, 4)
#define EXL3_NORM_INST(WHOLE, XB, RB, T, V, LOOP) \
  template __global__ void rms_norm_kernel<WHOLE, XB, RB, T, V, LOOP>(NormParams);
EXL3_NORM_B(EXL3_NORM_INST, true)
EXL3_NORM_B(EXL3_NORM_INST, false)

}  // namespace exl3

using namespace exl3;

#ifndef __HIP_DEVICE_COMPILE__

namespace {

template <bool WHOLE, int XB, int RB, int T, int V, bool LOOP = false>
void launch(const NormParams& p, hipStream_t s) {
  constexpr int kRows = T < 256 ? 256 / T : 1;
  const dim3 grid((unsigned)((p.rows + kRows - 1) / kRows));
  hipLaunchKernelGGL((rms_norm_kernel<WHOLE, XB, RB, T, V, LOOP>), grid, dim3(T < 256 ? 256 : T), 0, s, p);
}

template <bool WHOLE, int XB, int RB>
void launch(const NormParams& p, hipStream_t s) {
  const int w = p.width;
  w <= 64      ? launch<WHOLE, XB, RB, 8, 1>(p, s)
  : w <= 128   ? launch<WHOLE, XB, RB, 16, 1>(p, s)
  : w <= 256   ? launch<WHOLE, XB, RB, 32, 1>(p, s)
  : w <= 512   ? launch<WHOLE, XB, RB, 64, 1>(p, s)
  : w <= 2048  ? launch<WHOLE, XB, RB, 256, 1>(p, s)
  : w <= 4096  ? launch<WHOLE, XB, RB, 256, 2>(p, s)
  : w <= 8192  ? launch<WHOLE, XB, RB, 256, 4>(p, s)
  : w <= 16384 ? launch<WHOLE, XB, RB, 1024, 2>(p, s)
  : w <= 32768 ? launch<WHOLE, XB, RB, 1024, 4>(p, s)
               : launch<WHOLE, XB, RB, 1024, 4, true>(p, s);
}

template <bool WHOLE>
void launch(const NormParams& p, hipStream_t s) {
  const int rb = !p.r ? 0 : p.r_type == DT_F32 ? 4 : 2;
  if (p.x_type == DT_F32)
    rb == 0 ? launch<WHOLE, 4, 0>(p, s) : rb == 2 ? launch<WHOLE, 4, 2>(p, s) : launch<WHOLE, 4, 4>(p, s);
  else
    rb == 0 ? launch<WHOLE, 2, 0>(p, s) : rb == 2 ? launch<WHOLE, 2, 2>(p, s) : launch<WHOLE, 2, 4>(p, s);
}

constexpr int kMostWidth = 1 << 17;

bool float_type(int t) { return t == EXL3_F16 || t == EXL3_BF16 || t == EXL3_F32; }
bool rows_aligned(const void* p, int64_t stride, int type) {
  return aligned16(p) && (size_t)stride * (type == EXL3_F32 ? 4 : 2) % 16 == 0;
}

}  // namespace

extern "C" int exl3_rms_norm(const void* x, int32_t x_type, int64_t tokens, int32_t heads, int32_t width,
                             int64_t x_stride, const void* weight, int32_t weight_type, float eps,
                             const void* residual, int32_t residual_type, int64_t residual_stride,
                             void* total, int64_t total_stride, void* y, int32_t y_type,
                             int64_t y_stride, void* stream) {
  if (tokens < 0) return fail(EXL3_EINVAL, "negative token count");
  if (!float_type(x_type) || !float_type(y_type))
    return fail(EXL3_EINVAL, "unsupported norm dtypes %d and %d", x_type, y_type);
  if (weight && !float_type(weight_type)) return fail(EXL3_EINVAL, "unsupported norm weight dtype %d", weight_type);
  if (residual && !float_type(residual_type)) return fail(EXL3_EINVAL, "unsupported residual dtype %d", residual_type);
  if (heads < 1 || heads > 65536) return fail(EXL3_EINVAL, "invalid norm heads: %d", heads);
  if (width < 1 || width > kMostWidth)
    return fail(EXL3_EUNSUPPORTED, "norms take rows of 1 to %d values, got %d", kMostWidth, width);
  if (!(eps >= 1.17549435e-38f) || !std::isfinite(eps))
    return fail(EXL3_EINVAL, "norm eps must be a positive normal number");
  if (total && !residual) return fail(EXL3_EINVAL, "a sum needs a residual");
  const int64_t need = (int64_t)heads * width;
  if (tokens > 1 && (x_stride < need || y_stride < need || (residual && residual_stride < need) ||
                     (total && total_stride < need)))
    return fail(EXL3_EINVAL, "token strides are at least heads * width");
  if (tokens == 0) return EXL3_OK;
  if (!x || !y) return fail(EXL3_EINVAL, "null norm input or output");
  if (total == y) return fail(EXL3_EINVAL, "the sum and the norm are two outputs");
  const int64_t xs = tokens > 1 ? x_stride : 0, ys = tokens > 1 ? y_stride : 0;
  const int64_t rs = tokens > 1 ? residual_stride : 0, ts = tokens > 1 ? total_stride : 0;
  // an output in place of an input: every thread reads what it writes over
  auto in_place = [&](const void* out, int type, int64_t stride, const void* in, int in_type, int64_t in_stride) {
    return out != in || (type == in_type && stride == in_stride);
  };
  if (!in_place(y, y_type, ys, x, x_type, xs) || (residual && !in_place(y, y_type, ys, residual, residual_type, rs)) ||
      (total && (!in_place(total, residual_type, ts, x, x_type, xs) ||
                 !in_place(total, residual_type, ts, residual, residual_type, rs))))
    return fail(EXL3_EINVAL, "a norm in place keeps the type and the stride");
  const int64_t per = width <= 64 ? 32 : width <= 128 ? 16 : width <= 256 ? 8 : width <= 512 ? 4 : 1;
  const int64_t most = width > 8192 ? kMostBlocks / 4 : kMostBlocks;
  if (tokens > INT64_MAX / need || tokens * heads > most * per)
    return fail(EXL3_EUNSUPPORTED, "too many tokens: %lld", (long long)tokens);
  NormParams p{};
  p.x = x;
  p.w = weight;
  p.r = residual;
  p.y = y;
  p.total = total;
  p.rows = tokens * heads;
  p.x_stride = xs;
  p.r_stride = rs;
  p.y_stride = ys;
  p.total_stride = ts;
  p.heads = heads;
  p.width = width;
  p.x_type = x_type;
  p.w_type = weight_type;
  p.r_type = residual_type;
  p.y_type = y_type;
  p.eps = eps;
  const bool whole = width % 8 == 0 && rows_aligned(x, xs, x_type) && rows_aligned(y, ys, y_type) &&
                     (!residual || rows_aligned(residual, rs, residual_type)) &&
                     (!total || rows_aligned(total, ts, residual_type)) && (!weight || aligned16(weight));
  if (int rc = launch_gate("RMS norm")) return rc;
  whole ? launch<true>(p, (hipStream_t)stream) : launch<false>(p, (hipStream_t)stream);
  return check_launch("RMS norm");
}

#endif  // __HIP_DEVICE_COMPILE__
