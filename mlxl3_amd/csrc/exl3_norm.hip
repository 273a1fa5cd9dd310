// Root-mean-square norm of rows, with the residual's addition:
//
//   s = x + r   (without a residual x)      total = s, rounded to r's type
//   y = s * rsqrt(sum s^2 / width + eps) * w
//
// s is f32 and not rounded on the way to y, the sum of squares is f32: up to 8 V squares in
// a lane, then a tree.  Memory bounds it (every value is read and written once), so a row stays in
// registers between its sum and its outputs: T threads hold 8 V values each.  Rows of more
// than 32768 values are read again instead (from the caches).
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
  v += xor_lanes<8>(v);
  if constexpr (T >= 64) {
    v += xor_lanes<16>(v);
    v += xor_lanes<32>(v);
  }
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

// Chunk c of a thread's values: VEC: eight neighbours, 16-byte aligned; else every T-th, so that
// the lanes of a load are neighbours.
template <bool VEC, int T>
__device__ __forceinline__ int value_at(int c, int e, int t) {
  return VEC ? (c * T + t) * 8 + e : (c * 8 + e) * T + t;
}

template <int BYTES>
__device__ __forceinline__ void load_values(const void* p, int type, size_t row, int at, float (&v)[8]) {
  Raw8<BYTES> raw;
  raw.load(p, row + at, true);
  raw.get(type, v);
}

// XB, RB: bytes of x and of the residual (0: none), with VEC.  LOOP: rows that registers do not
// hold, V chunks at a time.
template <bool VEC, int XB, int RB, int T, int V, bool LOOP>
__global__ __launch_bounds__(T < 256 ? 256 : T) void rms_norm_kernel(NormParams p) {
  __shared__ float parts[T > 64 ? T / 64 : 1];
  const int t = threadIdx.x % T;
  const int64_t row = (int64_t)blockIdx.x * (T < 256 ? 256 / T : 1) + threadIdx.x / T;
  const bool on = T >= 256 || row < p.rows;
  const int64_t token = p.heads == 1 ? row : row / p.heads;
  const size_t in_token = p.heads == 1 ? 0 : (size_t)(row - token * p.heads) * p.width;
  const size_t xr = (size_t)token * p.x_stride + in_token, rr = (size_t)token * p.r_stride + in_token;
  const size_t yr = (size_t)token * p.y_stride + in_token, tr = (size_t)token * p.total_stride + in_token;
  constexpr int kSpan = 8 * T * V;
  float s[V][8];
  auto load = [&](int from) __attribute__((always_inline)) {
    if constexpr (VEC) {
      Raw8<XB> x[V];
      Raw8<RB ? RB : 2> r[V];
#pragma unroll
      for (int c = 0; c < V; ++c) {
        const int at = from + value_at<true, T>(c, 0, t);
        if (!on || at >= p.width) continue;
        x[c].load(p.x, xr + at, true);
        if (RB) r[c].load(p.r, rr + at, true);
      }
#pragma unroll
      for (int c = 0; c < V; ++c) {
        const bool in = on && from + value_at<true, T>(c, 0, t) < p.width;
        float b[8];
        x[c].get(p.x_type, s[c]);
        if (RB) r[c].get(p.r_type, b);
#pragma unroll
        for (int e = 0; e < 8; ++e) s[c][e] = in ? RB ? s[c][e] + b[e] : s[c][e] : 0.0f;
      }
    } else {
#pragma unroll
      for (int c = 0; c < V; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int at = from + value_at<false, T>(c, e, t);
          s[c][e] = 0.0f;
          if (!on || at >= p.width) continue;
          s[c][e] = load1(p.x, p.x_type, xr + at);
          if (p.r) s[c][e] += load1(p.r, p.r_type, rr + at);
        }
    }
  };
  auto squares = [&](float f) __attribute__((always_inline)) {
    float sum = 0.0f;
#pragma unroll
    for (int c = 0; c < V; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = s[c][e] * f;
        sum = fmaf(v, v, sum);
      }
    return sum;
  };
  auto square_sum = [&](float f) __attribute__((always_inline)) {
    float sum = 0.0f;
    if constexpr (LOOP) {
      for (int from = 0; from < p.width; from += kSpan) {
        load(from);
        sum += squares(f);
      }
    } else {
      sum = squares(f);
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
  auto store = [&](int from) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < V; ++c) {
      if constexpr (VEC) {
        const int at = from + value_at<true, T>(c, 0, t);
        if (!on || at >= p.width) continue;
        if (RB && p.total) store8(p.total, p.r_type, tr + at, s[c]);
        float w[8];
        if (p.w) {
          if (p.w_type == DT_F32)
            load_values<4>(p.w, p.w_type, 0, at, w);
          else
            load_values<2>(p.w, p.w_type, 0, at, w);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          s[c][e] *= unit;
          s[c][e] *= inv;
          if (p.w) s[c][e] *= w[e];
        }
        store8(p.y, p.y_type, yr + at, s[c]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int at = from + value_at<false, T>(c, e, t);
          if (!on || at >= p.width) continue;
          if (p.r && p.total) store1(p.total, p.r_type, tr + at, s[c][e]);
          const float v = s[c][e] * unit * inv;
          store1(p.y, p.y_type, yr + at, p.w ? v * load1(p.w, p.w_type, at) : v);
        }
      }
    }
  };
  if constexpr (LOOP) {
    for (int from = 0; from < p.width; from += kSpan) {
      load(from);
      store(from);
    }
  } else {
    store(0);
  }
}

#define EXL3_NORM_T(M, VEC, XB, RB) \
  M(VEC, XB, RB, 16, 1, false) M(VEC, XB, RB, 64, 1, false) M(VEC, XB, RB, 256, 1, false) \
  M(VEC, XB, RB, 256, 2, false) M(VEC, XB, RB, 256, 4, false) M(VEC, XB, RB, 1024, 2, false) \
  M(VEC, XB, RB, 1024, 4, false) M(VEC, XB, RB, 1024, 4, true)
#define EXL3_NORM(M) \
  EXL3_NORM_T(M, true, 2, 0) EXL3_NORM_T(M, true, 2, 2) EXL3_NORM_T(M, true, 2, 4) EXL3_NORM_T(M, true, 4, 0) \
  EXL3_NORM_T(M, true, 4, 2) EXL3_NORM_T(M, true, 4, 4) EXL3_NORM_T(M, false, 0, 0)
#define EXL3_NORM_INST(VEC, XB, RB, T, V, LOOP) \
  template __global__ void rms_norm_kernel<VEC, XB, RB, T, V, LOOP>(NormParams);
EXL3_NORM(EXL3_NORM_INST)

}  // namespace exl3

using namespace exl3;

#ifndef __HIP_DEVICE_COMPILE__

namespace {

template <bool VEC, int XB, int RB, int T, int V, bool LOOP = false>
void launch(const NormParams& p, hipStream_t s) {
  constexpr int kRows = T < 256 ? 256 / T : 1;
  const dim3 grid((unsigned)((p.rows + kRows - 1) / kRows));
  hipLaunchKernelGGL((rms_norm_kernel<VEC, XB, RB, T, V, LOOP>), grid, dim3(T < 256 ? 256 : T), 0, s, p);
}

template <bool VEC, int XB, int RB>
void launch(const NormParams& p, hipStream_t s) {
  const int w = p.width;
  w <= 128     ? launch<VEC, XB, RB, 16, 1>(p, s)
  : w <= 512   ? launch<VEC, XB, RB, 64, 1>(p, s)
  : w <= 2048  ? launch<VEC, XB, RB, 256, 1>(p, s)
  : w <= 4096  ? launch<VEC, XB, RB, 256, 2>(p, s)
  : w <= 8192  ? launch<VEC, XB, RB, 256, 4>(p, s)
  : w <= 16384 ? launch<VEC, XB, RB, 1024, 2>(p, s)
  : w <= 32768 ? launch<VEC, XB, RB, 1024, 4>(p, s)
               : launch<VEC, XB, RB, 1024, 4, true>(p, s);
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
  const int64_t per = width <= 128 ? 16 : width <= 512 ? 4 : 1, most = width > 8192 ? kMostBlocks / 4 : kMostBlocks;
  if (tokens > INT64_MAX / need || (tokens * heads + per - 1) / per > most)
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
  // eight values at a time where every chunk of eight is 16-byte aligned and whole
  const bool vec = width % 8 == 0 && rows_aligned(x, xs, x_type) && rows_aligned(y, ys, y_type) &&
                   (!residual || rows_aligned(residual, rs, residual_type)) &&
                   (!total || rows_aligned(total, ts, residual_type)) && (!weight || aligned16(weight));
  if (int rc = launch_gate("RMS norm")) return rc;
  hipStream_t s = (hipStream_t)stream;
  const int xb = x_type == EXL3_F32 ? 4 : 2, rb = !residual ? 0 : residual_type == EXL3_F32 ? 4 : 2;
  if (!vec)
    launch<false, 0, 0>(p, s);
  else if (xb == 2)
    rb == 0 ? launch<true, 2, 0>(p, s) : rb == 2 ? launch<true, 2, 2>(p, s) : launch<true, 2, 4>(p, s);
  else
    rb == 0 ? launch<true, 4, 0>(p, s) : rb == 2 ? launch<true, 4, 2>(p, s) : launch<true, 4, 4>(p, s);
  return check_launch("RMS norm");
}

#endif  // __HIP_DEVICE_COMPILE__
