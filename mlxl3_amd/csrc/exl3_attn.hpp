// Device code shared by the attention kernels: element types, fragments of the paged
// cache, the running softmax.
#pragma once

#include "exl3_kv.hpp"

namespace exl3 {

// What becomes of scores (the kernels' S; below).  For few rows, which memory bounds, kEarly does for
// kSeen and kCapped for kBoth.
enum : int { kPlain = 0, kEarly = 1, kCapped = 2, kLate = 3, kSeen = 4, kBoth = 5 };

struct AttnParams {
  KvCacheView cache;
  KvBatchView batch;
  const void* q;
  void* y;
  float* part;    // weighted sums [slots][rows][D]; slots: [tiles][splits or ranges][kv heads]
  float* stats;   // [slots][rows][2] their maximum and sum of weights
  int64_t q_stride, y_stride;
  int tokens;     // rows of q and y
  int group, q_type, causal, window;
  int max_q;
  int splits;     // even ranges of the tokens that a tile sees
  int budget;     // else ranges by the batch's sum (few rows), about; 0: even ones
  int one_tile;   // every sequence's rows fit one workgroup: tile = sequence
  int q_vec, y_vec;  // rows of q are 16-byte, rows of y 8-byte aligned
  float scale2;   // scale * log2(e): scores in units of a factor of two
  // of calls with shaped scores: cap2 = cap * log2(e), 0 without a cap
  float cap2;
  const float* slopes;    // of every head, or null
  const int32_t* prefix;  // of every sequence, or null
};

typedef float float16v __attribute__((ext_vector_type(16)));

// Matrix operands of eight 16-bit values, and what an attention kernel does with them.
struct F16 {
  typedef half8 V8;
  typedef _Float16 E;
  static constexpr float kRoom = 7.0f;  // below
  static __device__ __forceinline__ float4v mfma16(V8 a, V8 b, float4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float16v mfma32(V8 a, V8 b, float16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
struct BF16 {
  typedef bf8 V8;
  typedef __bf16 E;
  static constexpr float kRoom = 0.0f;
  static __device__ __forceinline__ float4v mfma16(V8 a, V8 b, float4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float16v mfma32(V8 a, V8 b, float16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};

typedef short short4v __attribute__((ext_vector_type(4)));

// Four rows of 16 16-bit values in LDS, transposed on the way to registers: of each 16
// lanes, lane 4j + c names values 4c .. 4c + 3 of row j, and lane i gets value i of rows
// 0 .. 3.
__device__ __forceinline__ u32x2 lds_transpose4(const uint8_t* p) {
  typedef __attribute__((address_space(3))) short4v* LdsPtr;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(size_t)lds_offset(p)));
}

// The compiler moves no instruction across this.
__device__ __forceinline__ void pin() { __builtin_amdgcn_sched_barrier(0); }

// Whether any of eight 16-bit values is a NaN or an infinity.
template <typename T>
__device__ __forceinline__ bool not_finite(const u32x4& v) {
  constexpr uint32_t mask = __is_same(T, BF16) ? 0x7f807f80u : 0x7c007c00u;
  constexpr uint32_t lo = mask & 0xffffu, hi = mask & 0xffff0000u;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = v[i];
    bad = bad || (w & lo) == lo || (w & hi) == hi;
  }
  return bad;
}

// Whether a coded group may hold a value that is no finite f16: its scale's magnitude against the
// least one that a code takes past 65504 -- 512 = 65536 / 128 for 8 bits, 8192 = 65536 / 8 for
// 4 -- NaN and infinity lie above both.
template <int FMT>
__device__ __forceinline__ bool past_f16(uint32_t scale) {
  return (scale & 0x7fff) >= (FMT == KV_Q8 ? 0x6000u : 0x7000u);
}

// Where channel e of eight lies in codes4's order, and which channel lies at place e.
__device__ __forceinline__ constexpr int place4(int e) { return e < 4 ? 2 * e : 2 * e - 7; }
__device__ __forceinline__ constexpr int channel4(int e) { return (e >> 1) | ((e & 1) << 2); }

// code * scale needs up to 18 bits, an f16 has 11.  Rounded to those it is off by half as much
// as an f16 query or output is, and a large score by many times that: with f16 queries a
// value is two f16 -- the scale's leading bits times the code, exact, and the rest (8 bits:
// to 2^-15) -- each with its own product.  With bf16 queries one rounded f16 is enough: the
// outputs are 8 times coarser than its 2^-11, and so were the queries when they were rounded to
// bf16, so that a key's part in a score's error (2^-11 of the sum of magnitudes at most) is an
// eighth of what the query's is already.  Same box, us: 32 decodes over 8192 8-bit tokens, f16, one
// part 86.4 (2-norm error 8.3e-4, 2.1e-4 of it the output's own rounding), two 94.5 (2.9e-4);
// four drafts of 5 over 6001 4-bit tokens, bf16, 24.3 (1.8e-3 against 1.6e-3) and 27.6 (1.6e-3);
// 2048 f16 rows over 8192 8-bit tokens 307 (6.7e-4) and 520 (2.9e-4).
template <int FMT, int PARTS>
__device__ __forceinline__ void scale_parts(uint32_t scale, _Float16& hi, _Float16& lo) {
  const _Float16 s = __builtin_bit_cast(_Float16, (uint16_t)scale);
  hi = PARTS == 1 ? s : __builtin_bit_cast(_Float16, (uint16_t)(scale & (FMT == KV_Q8 ? 0xff80u : 0xfff8u)));
  lo = s - hi;
}

// Eight query channels from element i on, as they lie.
__device__ __forceinline__ u32x4 load_q8(const AttnParams& p, size_t i) {
  const uint16_t* q = (const uint16_t*)p.q + i;
  if (p.q_vec) return *(const u32x4*)q;
  u32x4 r;
#pragma unroll
  for (int e = 0; e < 4; ++e) r[e] = (uint32_t)q[2 * e] | (uint32_t)q[2 * e + 1] << 16;
  return r;
}

// The products of coded caches are f16.  A bf16 has fewer bits than that and a wider range, so
// bf16 queries are multiplied by the power of two that takes a row's largest magnitude to
// 2^15 .. 2^16: exact but for channels below 2^-29 of it, which are off by up to 2^-40 of it.
// Their scores are multiplied by its inverse, with the scale.  (From 2^-111 down the factor stays
// 2^126, so that the inverse is a normal f32.)
__device__ __forceinline__ float largest_bf16(const u32x4& w, float most) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t v = w[e];
    most = fmaxf(most, fmaxf(fabsf(bf2f((uint16_t)v)), fabsf(bf2f((uint16_t)(v >> 16)))));
  }
  return most;
}
// Where the products' sums start from a bias (kEarly): from 2^-10 down, so that the bias over the scale
// stays inside f32's range; queries are off by 2^-50 or so then.
template <int S>
__device__ __forceinline__ uint32_t fit_exponent(float most) {
  return max(__builtin_bit_cast(uint32_t, most) >> 23, S == kEarly ? 117u : 16u);
}
__device__ __forceinline__ float fit_factor(uint32_t e) { return __builtin_bit_cast(float, (269 - e) << 23); }
// The scale times the inverse, a normal f32 too: a masked score, -inf, times zero would be NaN,
// as would a score of zero times infinity (at the lower border all scores round to weights of 1).
__device__ __forceinline__ float fit_scale(float scale2, uint32_t e) {
  const float inverse = __builtin_bit_cast(float, (e - 15) << 23);
  return fminf(fmaxf(scale2 * inverse, 1.17549435e-38f), 3.402823466e38f);
}

// Eight query channels as T: T is the queries' own type for 16-bit caches, f16 for coded ones
// (bf16 queries times `factor`; 4 bits: in codes4's order).
template <int FMT, typename T, bool SCALED>
__device__ __forceinline__ typename T::V8 query_operand(const u32x4& w, float factor) {
  uint16_t h[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) h[e] = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
  if constexpr (SCALED) {
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = f2h(bf2f(h[e]) * factor);
  }
  u32x4 r;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int a = FMT == KV_Q4 ? channel4(2 * e) : 2 * e, b = FMT == KV_Q4 ? channel4(2 * e + 1) : 2 * e + 1;
    r[e] = (uint32_t)h[a] | ((uint32_t)h[b] << 16);
  }
  return __builtin_bit_cast(typename T::V8, r);
}

// What a workgroup works on: sequence, its first row of the call's tensors, rows
// (tokens x heads of the group), first new position, length cut to the table's room.  Rows
// that q does not have are not touched, whatever q_starts says.
struct Work {
  int seq, start, rows, first, len;
  int prefix;            // tokens that all rows see (0 of a plain call)
  const int32_t* table;  // the sequence's row of the block table
};
template <int S>
__device__ __forceinline__ Work sequence_work(const AttnParams& p, int seq) {
  Work w;
  w.seq = seq;
  w.start = p.batch.q_starts[seq];
  const int64_t n = (int64_t)p.batch.q_starts[seq + 1] - w.start;
  const int64_t have = w.start < 0 ? 0 : (int64_t)p.tokens - w.start;
  w.rows = (int)max((int64_t)0, min(min(n, have), (int64_t)p.max_q)) * p.group;
  const int kv = p.batch.kv_lens[seq];
  const int64_t room = (int64_t)p.batch.table_pages << p.cache.page_shift;
  w.len = (int)max((int64_t)0, min(min((int64_t)kv, room), (int64_t)INT32_MAX - 4095));
  w.first = (int)max((int64_t)INT32_MIN, (int64_t)kv - n);
  w.prefix = S && p.prefix ? p.prefix[seq] : 0;
  w.table = p.batch.table + (int64_t)seq * p.batch.table_pages;
  return w;
}

// The tokens that row `row` (token row / group of the sequence) may see: [lo, hi).
struct Seen {
  int lo, hi;
};
template <int S>
__device__ __forceinline__ Seen row_sees(const AttnParams& p, const Work& w, int row) {
  const int64_t pos = (int64_t)w.first + row / p.group, len = w.len;
  Seen s{0, w.len};
  if (p.causal) s.hi = (int)max((int64_t)0, min(len, S ? max(pos + 1, (int64_t)w.prefix) : pos + 1));
  if (p.window > 0) s.lo = (int)min(len, max((int64_t)0, pos - p.window + 1));
  return s;
}

__device__ __forceinline__ float wave_sum(float v) {
  v += xor_lanes<1>(v);
  v += xor_lanes<2>(v);
  v += xor_lanes<4>(v);
  v += xor_lanes<8>(v);
  v += xor_lanes<16>(v);
  v += xor_lanes<32>(v);
  return v;
}

// The sequence that item `i` belongs to, `items` telling how many each has; i becomes its
// number there.  Behind the last item: no rows.  Every lane of a wave calls it with one i.
template <int S, typename F>
__device__ __forceinline__ Work work_of(const AttnParams& p, int& i, F&& items) {
  const int lane = threadIdx.x & 63;
  for (int s0 = 0; s0 < p.batch.seqs; s0 += 64) {
    const int seq = s0 + lane;
    const Work x = seq < p.batch.seqs ? sequence_work<S>(p, seq) : Work{};
    const int mine = seq < p.batch.seqs ? items(x) : 0;
    int upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int other = __shfl_up(upto, d);
      if (lane >= d) upto += other;
    }
    const uint64_t past = __ballot(upto > i);
    if (past) {
      const int at = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)past) - 1);
      i -= __builtin_amdgcn_readlane(upto - mine, at);
      auto of = [&](int v) { return __builtin_amdgcn_readlane(v, at); };
      return Work{s0 + at, of(x.start), of(x.rows), of(x.first), of(x.len), S ? of(x.prefix) : 0,
                  p.batch.table + (int64_t)(s0 + at) * p.batch.table_pages};
    }
    i -= __builtin_amdgcn_readlane(upto, 63);
  }
  return Work{};
}

// Sequence and first row of tile `tile`, sequences cut into tiles of `rows` rows; a tile
// behind the last has no rows.
template <int S>
__device__ __forceinline__ Work tile_work(const AttnParams& p, int tile, int rows, int& row0) {
  row0 = 0;
  if (p.one_tile) return sequence_work<S>(p, tile);
  const Work w = work_of<S>(p, tile, [&](const Work& x) { return (x.rows + rows - 1) / rows; });
  row0 = tile * rows;
  return w;
}

// The table's entry for the 16 tokens from t (a multiple of 16) on, hi > 0 the end of the
// tokens in use.  Wave-uniform: a scalar load (no kernel writes the table), not waited for
// here; page_ok says later whether it names a page.
__device__ __forceinline__ int table_entry(const AttnParams& p, const Work& w, int t, int hi) {
  typedef const __attribute__((address_space(4))) int32_t* ScalarPtr;
  return ((ScalarPtr)(size_t)w.table)[(uint32_t)min(t, hi - 1) >> p.cache.page_shift];
}
__device__ __forceinline__ int page_ok(const AttnParams& p, int entry, int t, int hi) {
  return t < hi && (uint32_t)entry < (uint32_t)p.cache.pages ? entry : -1;  // pages < 2^31
}

// A tile's tokens split evenly: the length of each of p.splits ranges of `n` tokens, a multiple
// of 128.  It goes by the sequence's own length, not by what the host was told.
__device__ __forceinline__ int split_tokens(const AttnParams& p, int n) {
  return (int)max(((uint32_t)(n + p.splits - 1) / p.splits + 127) & ~127u, 128u);
}
// The tokens that a sequence's rows see, from a multiple of 16 on; a sequence with rows has one.
template <int S>
__device__ __forceinline__ int seen_tokens(const AttnParams& p, const Work& w) {
  if (w.rows == 0) return 0;
  const int lo = row_sees<S>(p, w, 0).lo & ~15;
  return max(row_sees<S>(p, w, w.rows - 1).hi - lo, 1);
}

// A batch of few rows split by its sum: ranges of equally many tokens for all sequences, longer
// sequences in more of them, so that a ragged batch's workgroups take equally long.  Every
// workgroup forms the sum of the tokens seen for itself and cuts them into about `budget`
// ranges, at most budget + seqs (a sequence's last one may be short).
constexpr int kMostRanges = 32;  // of a sequence: a row's ranges are joined by few lanes
// The tokens of a range, by the batch (a wave calls it) and by the sequence's own.
template <int S>
__device__ __forceinline__ int range_tokens(const AttnParams& p) {
  float total = 0.0f;
  for (int s0 = 0; s0 < p.batch.seqs; s0 += 64) {
    const int seq = s0 + (threadIdx.x & 63);
    if (seq < p.batch.seqs) total += (float)seen_tokens<S>(p, sequence_work<S>(p, seq));
  }
  total = wave_sum(total);
  return __builtin_amdgcn_readfirstlane(((int)fminf(total / p.budget, 2147483392.0f) + 128) & ~127);
}
__device__ __forceinline__ int range_tokens(int each, int n) {
  constexpr int unit = kMostRanges * 128;
  return max(each, (n + unit - 1) / unit * 128);
}
__device__ __forceinline__ int range_count(int each, int n) {
  const uint32_t size = range_tokens(each, n);
  return (int)(((uint32_t)n + size - 1) / size);
}

// Weights are taken against m, at first the largest score less T::kRoom (in factors of two).  A
// score above it by no more than T::kRoom and this does not move m: so most steps rescale
// nothing and exchange nothing between lanes.  The largest weight is then one of 2^kRoom to
// 2^(kRoom + kSlack): 256 for bf16, 2^15 for f16, and their sums stay far inside f32's range.
// f16 needs the room below: what it cannot hold, weights under 2^-25, is 2^-32 of the largest
// then and was 2^-25 of it without, so that thousands of tokens 15 to 17 nats below one whose
// values are small lost 6 to 100 % of their part.
constexpr float kSlack = 8.0f;

// They are exp2(fma(score, scale2, -m)), m from the rounded product for some score: the others'
// unrounded ones pass that by up to half a step of it, nothing until m is large, and at 2^27 a
// factor of 2^8, at 2^34 of 2^512.  Once a maximum of a wave is beyond this, products are
// rounded before m is taken off, exactly: none passes the largest.  (Then every step goes the
// way of a moving maximum, so that others have no further branch.)
constexpr float kFar = 65536.0f;
// m of a row that has seen nothing yet: finite, so that neither m less m nor a masked score
// (-inf) less m is NaN.  Kept as -inf outside the loops.
constexpr float kNothing = -3.402823466e38f;
__device__ __forceinline__ float seen_max(float m) { return m == kNothing ? -__builtin_inff() : m; }
// The slack of a wave whose lanes' maxima are now m: kept as it is or, far, below every difference.
__device__ __forceinline__ float slack_at(float m, float slack) {
  const float s = __any(fabsf(m) > kFar && m != kNothing) ? kNothing : slack;
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, s)));
}

// Shaped scores: x is a score in factors of two, s scale log2(e).
//
// Capped it is cap2 tanh(u), u = x / cap2: a score z becomes cap tanh(z / cap).  tanh(u) = 1 - 2 / (1 +
// e^2u), and of all scores of a row softmax takes off what it likes: less cap2 a capped score is
//   2 cap2 c,  c = -1 / (1 + 2^(rate x)),  rate = 2 log2(e) / cap2.
// So a call with a cap (kCapped, with a bias kBoth) puts c where the product was, in four instructions,
// and goes on as a plain one whose scale is 2 cap2.  c is off by 2^-23 or so, the score by cap2 times
// that, 1e-5 under a cap of 50.  (tanh's polynomials in u^2 up to |u| = 1, in tiles where no score is beyond, are
// as many instructions or more and a maximum: 2048 rows over 8192 bf16 tokens 335 us for 304, plain 256.)
//
// The bias by distance takes slope2 = slope log2(e) times it off the score.  Without a cap the sums of the
// products start from it, divided by what scores are multiplied by (kEarly), and all else is as for
// plain scores; under a cap it is added to c, divided by 2 cap2.
//
// Caps above 256, where the error above is too much for small scores (|u| < 1/4 takes tanh's series there,
// and nothing is taken off), and factors whose quotients may leave f32's range go one step
// after the other (kLate): times the scale, capped, biased.  That is no fast way for many rows -- a cap
// above 256 forms both c and the series, and divides by the cap, for every score: 2048 rows over 8192 bf16
// tokens under a cap of 1000 585 us for 288 to 302 under 50 (heads of 64 525 for 208 to 222, over 8 bits with
// f16 queries 802 to 831 for 554 to 578), a bias under a scale of 1e-8 281 to 292 for 248 to 260 -- and
// costs few rows little: one token over 8192 15.7 for 15.1.
//
// A prefix only moves the end of what a row sees (kSeen: without a cap and a bias).
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLargeCap = 256.0f * kLog2e;
__device__ __forceinline__ float squashed(float x, float rate) {
  return __builtin_amdgcn_rcpf(-1.0f - __builtin_amdgcn_exp2f(x * rate));
}
// What c's exponent is of a product, that of a score (both finite and positive).
__device__ __forceinline__ float cap_rate(const AttnParams& p, float scale2) {
  return fminf(2.0f * kLog2e / p.cap2 * scale2, 3.402823466e38f);
}
// A score capped, where there is a cap.
__device__ __forceinline__ float capped(const AttnParams& p, float x) {
  if (p.cap2 == 0.0f) return x;
  const float c = 2.0f * p.cap2 * squashed(x, cap_rate(p, 1.0f));
  if (p.cap2 <= kLargeCap) return c;
  const float u = x / p.cap2, v = u * u;
  const float series =
      fmaf(v, fmaf(v, fmaf(v, fmaf(v, 0.021869489f, -0.053968254f), 0.13333333f), -0.33333333f), 1.0f);
  return fabsf(u) < 0.25f ? x * series : p.cap2 + c;
}
__device__ __forceinline__ float biased(float x, float slope2, float away) { return fmaf(-slope2, fabsf(away), x); }
__device__ __forceinline__ float slope_of(const AttnParams& p, int head) {
  return p.slopes ? __builtin_amdgcn_fmed3f(p.slopes[head], -4294967296.0f, 4294967296.0f) * kLog2e : 0.0f;
}

// One row over the tokens [lo, hi) by one wave, its channels spread over the lanes (lane
// l holds channels E l ..): running maximum m, sum l and weighted values acc.  Touches
// only tokens that the row sees.
template <int E, int S>
__device__ __forceinline__ void row_pass(const AttnParams& p, const Work& w, int kvh, int row, int lo, int hi,
                                         int lane, float& m, float& l, float (&acc)[E]) {
  const KvCacheView& c = p.cache;
  constexpr int D = 64 * E;
  const size_t qi = (size_t)(w.start + row / p.group) * p.q_stride +
                    (size_t)(kvh * p.group + row % p.group) * D + E * lane;
  float q[E];
  m = -__builtin_inff();
  l = 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = load1(p.q, p.q_type, qi + e);
    acc[e] = 0.0f;
  }
  for (int t = lo; t < hi; ++t) {
    const int64_t page = kv_page(c, p.batch, w.seq, t);
    if (page < 0) continue;
    const size_t h = (size_t)page * c.kv_heads + kvh;
    const int slot = t & ((1 << c.page_shift) - 1);
    const size_t row0 = kv_bytes(c.format, ((h << c.page_shift) + slot) * D);
    float s = 0.0f, v[E], ks = 1.0f, vs = 1.0f;
    if (c.ks) {
      const size_t g = ((h * (D / 32) + E * lane / 32) << c.page_shift) + slot;
      ks = h2f(c.ks[g]);
      vs = h2f(c.vs[g]);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int d = E * lane + e;
      float k;
      if (c.format == KV_Q8) {
        k = (float)((int)c.k[row0 + d] - 128) * ks;
        v[e] = (float)((int)c.v[row0 + d] - 128) * vs;
      } else if (c.format == KV_Q4) {
        k = (float)(((int)c.k[row0 + d / 2] >> (4 * (d & 1)) & 15) - 8) * ks;
        v[e] = (float)(((int)c.v[row0 + d / 2] >> (4 * (d & 1)) & 15) - 8) * vs;
      } else {
        k = load1(c.k + row0, c.format, d);
        v[e] = load1(c.v + row0, c.format, d);
      }
      s += q[e] * k;
    }
    s = wave_sum(s) * p.scale2;
    if constexpr (S) {
      s = capped(p, s);
      if (p.slopes) s = biased(s, slope_of(p, kvh * p.group + row % p.group), (float)(w.first + row / p.group - t));
    }
    const float n = fmaxf(m, s);
    const float base = n == -__builtin_inff() ? 0.0f : n;
    const float f = exp2f(m - base), x = exp2f(s - base);
    l = l * f + x;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = acc[e] * f + x * v[e];
    m = n;
  }
}

}  // namespace exl3
