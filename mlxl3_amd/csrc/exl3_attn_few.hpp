// Attention of few rows (tokens x heads of a group, at most 16 RT) over the cache:
// decode and short drafts.  The cache's bytes bound it, so every byte is read once, by
// one wave, straight into registers.
//
// A workgroup (4 waves) takes a range of one sequence's tokens for one cache head; wave w
// takes steps of 32 tokens w, w + 4, ...  A step:
//   S^T = K Q^T   16x16x32 MFMAs, K rows (tokens) as the A operand as they lie in the
//                 cache, the group's queries as the B operand.  Lane l then holds, of
//                 query l % 16, tokens 4 (l / 16) + i of both 16-token blocks;
//   P   = exp2(S - m), rounded to 16 bits: already the B operand of the next product,
//                 eight tokens a lane, so no lane exchange;
//   O^T += V^T P^T  with V^T read from LDS transposed (four tokens of a channel a read),
//                 in the token order that P has.  V goes through the wave's own LDS, so
//                 there is no barrier in the loop.
// m moves only when some score passes it by kSlack and the type's room (P and its sums stay
// inside 16 bits' and f32's range), so a step usually has no exchange between lanes
// at all; the sum l is kept per lane and reduced once at the end.
// The waves' results meet in LDS; with more than one range per sequence they are joined
// by attn_join_kernel.  Shaped scores (S, exl3_attn.hpp) take their instructions from S, before the
// mask, or start the products' sums: mostly within 5 % of plain ones (one token over 1000: 11.3 us for
// 10.8; 32 8-bit decodes 92 to 98 either way).
//
// P rounded to 16 bits is the product's operand type; its sum l is of the unrounded ones.
// The loop's only waits are for its own loads: the next step's keys and values are on the
// way while this one's are used.
//
// Measured, heads of 128 channels, 4 query heads a cache head, the join included: one bf16
// token over 131071 16-bit tokens 105 us, 5.1 TB/s; 32 f16 tokens (5 heads) over 32 sequences
// of up to 8192 8-bit tokens 95 us, 4.0 TB/s (equally long ones 4.75, 16 bits 5.5: there
// decoding and its two parts are 1.7e7 vector instructions, a third of the time, with no unit
// at its limit -- 12 waves a CU and 41 % of their time waiting), over 4 bits 75, with bf16 queries
// 61; drafts of 5, 4, 3 and 2 tokens over 6001 to 2988 4-bit tokens 23.5 us; one token over 1000
// 11 us, two launches and a few dependent loads.
#pragma once

#include "exl3_attn.hpp"

namespace exl3 {

template <int FMT, typename T, int D, int RT, int PARTS>
struct Few {
  static constexpr bool kRaw = FMT >= 9;
  static constexpr int kSteps = D / 32;                                 // MFMAs over the channels
  static constexpr int kRow = kRaw ? 2 * D : FMT == KV_Q8 ? D : D / 2;  // bytes of a cached head
  // keys: channels of a lane's vector load, and loads per 16 tokens
  static constexpr int kVec = kRaw ? 8 : FMT == KV_Q8 || D == 64 ? 16 : 32;
  static constexpr int kKeyLoads = D / 4 / kVec;
  static constexpr int kKeyWords = kVec * kRow / D / 4;
  static constexpr int kParts = PARTS;  // f16 that a coded value is made of (below)
  static constexpr bool kScaled = !kRaw && PARTS == 1;  // bf16 queries, to fit f16
  // Values go through LDS kSpan channels at a time: with two parts half a head, so that
  // three workgroups still fit a CU (32 rows: the results at the end need as much).  Of their
  // 16-byte loads: lanes per row, rows per load, loads.
  static constexpr int kSpans = PARTS == 1 || D == 64 || RT == 2 ? 1 : 2, kSpan = D / kSpans;
  static constexpr int kLanes = kRow / kSpans / 16, kRows = 64 / kLanes, kSpanLoads = 32 / kRows;
  static constexpr int kValueLoads = kSpans * kSpanLoads;
  static constexpr int kPart = 32 * kSpan * 2;
  static constexpr int kWaveLds = kParts * kPart > 16 * RT * D * 4 ? kParts * kPart : 16 * RT * D * 4;

  // First channel of lane group g's operand in MFMA step s.
  static __device__ __forceinline__ int channel(int s, int g) {
    constexpr int n = kVec / 8;
    return (s / n) * 4 * kVec + g * kVec + (s % n) * 8;
  }
  // Byte of 16-byte chunk c of row t of the values in LDS.  The transposing read takes 32
  // bytes (a pair of chunks) of each of 8 rows at a time: pairs change places so that
  // those fall into different banks.  A write of decoded codes takes every 2nd or 4th
  // chunk of one to eight rows: the two of a pair change places too so that those do.
  static __device__ __forceinline__ int place(int t, int c) {
    const int r = kSpan == 64 ? t >> 1 : t;  // rows that start in the same bank
    const int odd = kRaw ? 0 : kSpan == 256 ? c >> 4 : FMT == KV_Q8 ? r : r >> 1;
    const int swz = kSpan == 64 ? (r & 3) << 1 : (r & 7) << 1;
    return t * kSpan * 2 + ((c ^ swz ^ (odd & 1)) << 4);
  }

  struct Keys {
    uint32_t w[2][kKeyLoads][kKeyWords];
    uint32_t s[2][kRaw ? 1 : kKeyLoads];  // (16-bit elements would go through scratch)
  };
  struct Values {
    u32x4 w[kValueLoads];
    uint32_t s[kRaw ? 1 : kValueLoads];
  };

  static __device__ __forceinline__ void load_keys(const AttnParams& p, const int (&page)[2], int kvh, int t0,
                                                   int lane, Keys& k) {
    const KvCacheView& c = p.cache;
    const int r = lane & 15, g = lane >> 4;
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      const size_t h = (size_t)max(page[a], 0) * c.kv_heads + kvh;
      const int slot = (t0 + 16 * a) & ((1 << c.page_shift) - 1);
      const uint8_t* b = c.k + ((h << c.page_shift) + slot) * kRow;
      const uint16_t* sc = kRaw ? nullptr : c.ks + ((h * (D / 32)) << c.page_shift) + slot;
#pragma unroll
      for (int u = 0; u < kKeyLoads; ++u) {
        const int ch = u * 4 * kVec + g * kVec;
        const uint8_t* from = b + r * kRow + ch * kRow / D;
        if constexpr (kKeyWords == 4) {
          const u32x4 v = *(const u32x4*)from;
#pragma unroll
          for (int i = 0; i < 4; ++i) k.w[a][u][i] = v[i];
        } else {
          const u32x2 v = *(const u32x2*)from;
          k.w[a][u][0] = v[0];
          k.w[a][u][1] = v[1];
        }
        if constexpr (!kRaw) k.s[a][u] = sc[((ch / 32) << c.page_shift) + r];
      }
    }
  }
  // The operand of step s for block a, in kParts parts.
  static __device__ __forceinline__ void key(const Keys& k, int a, int s, typename T::V8 (&part)[kParts]) {
    constexpr int n = kVec / 8;
    const int u = s / n, i = s % n;
    if constexpr (kRaw) {
      u32x4 r;
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] = k.w[a][u][e];
      part[0] = __builtin_bit_cast(typename T::V8, r);
    } else {
      _Float16 hi, lo;
      scale_parts<FMT, PARTS>(k.s[a][u], hi, lo);
      u32x4 c;
      if constexpr (FMT == KV_Q8)
        c = codes8(k.w[a][u][2 * i], k.w[a][u][2 * i + 1]);
      else
        c = codes4(k.w[a][u][i]);
      part[0] = __builtin_bit_cast(typename T::V8, times(c, hi));
      if constexpr (kParts == 2) part[1] = __builtin_bit_cast(typename T::V8, times(c, lo));
    }
  }

  static __device__ __forceinline__ void load_values(const AttnParams& p, const int (&page)[2], int kvh, int t0,
                                                     int lane, Values& v) {
    const KvCacheView& c = p.cache;
    const uint8_t* b[2];
    const uint16_t* sc[2];
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      const size_t h = (size_t)max(page[a], 0) * c.kv_heads + kvh;
      const int slot = (t0 + 16 * a) & ((1 << c.page_shift) - 1);
      b[a] = c.v + ((h << c.page_shift) + slot) * kRow;
      sc[a] = kRaw ? nullptr : c.vs + ((h * (D / 32)) << c.page_shift) + slot;
    }
    const int r = lane / kLanes, ch = lane % kLanes;
#pragma unroll
    for (int u = 0; u < kValueLoads; ++u) {
      const int span = u / kSpanLoads, from = (span * kLanes + ch) * 16;  // byte of the head's row
      const int t = (u % kSpanLoads) * kRows + r;
      const bool second = kRows > 16 ? t >= 16 : (u % kSpanLoads) * kRows >= 16;
      v.w[u] = *(const u32x4*)((second ? b[1] : b[0]) + (t & 15) * kRow + from);
      if constexpr (!kRaw) {
        const int group = from * D / kRow / 32;
        v.s[u] = (second ? sc[1] : sc[0])[(group << c.page_shift) + (t & 15)];
      }
    }
  }
  // A span's values to LDS as 16-bit rows (4 bits: channels in codes4's order); rows outside
  // [live_lo, live_hi) or of a block without a page become zeros.  Returns whether an
  // edge's other rows may hold a value that is not finite.
  template <bool EDGE>
  static __device__ __forceinline__ bool put_values(const Values& v, int span, uint8_t* lds, int lane, int live_lo,
                                                    int live_hi, bool on0, bool on1) {
    const int r = lane / kLanes, ch = lane % kLanes;
    bool bad = false;
#pragma unroll
    for (int u0 = 0; u0 < kSpanLoads; ++u0) {
      const int u = span * kSpanLoads + u0, t = u0 * kRows + r;
      const bool live = !EDGE || (t >= live_lo && t < live_hi && (t < 16 ? on0 : on1));
      if (EDGE && live) bad = bad || (kRaw ? not_finite<T>(v.w[u]) : past_f16<FMT>(v.s[kRaw ? 0 : u]));
      constexpr int n = kRaw ? 1 : FMT == KV_Q8 ? 2 : 4;  // 16-byte chunks of the decoded row
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const int at = place(t, ch * n + i);
        if constexpr (kRaw) {
          *(u32x4*)(lds + at) = live ? v.w[u] : u32x4{0, 0, 0, 0};
        } else {
          _Float16 hi, lo;
          scale_parts<FMT, PARTS>(v.s[u], hi, lo);
          u32x4 c;
          if constexpr (FMT == KV_Q8) {
            const uint32_t w0 = v.w[u][2 * i], w1 = v.w[u][2 * i + 1];
            c = codes8(w0, w1);
          } else {
            const uint32_t w0 = v.w[u][i];
            c = codes4(w0);
          }
          *(u32x4*)(lds + at) = live ? times(c, hi) : u32x4{0, 0, 0, 0};
          if constexpr (kParts == 2) *(u32x4*)(lds + kPart + at) = live ? times(c, lo) : u32x4{0, 0, 0, 0};
        }
      }
    }
    return bad;
  }
  static __device__ __forceinline__ typename T::V8 value(const uint8_t* lds, int dt, int lane) {
    const int g = lane >> 4, j = (lane >> 2) & 3, c = lane & 3;
    const int t = 4 * g + j, chunk = dt * 2 + (c >> 1), half = (c & 1) * 8;
    const u32x2 lo = lds_transpose4(lds + place(t, chunk) + half);
    const u32x2 hi = lds_transpose4(lds + place(t + 16, chunk) + half);
    const u32x4 r = {lo[0], lo[1], hi[0], hi[1]};
    return __builtin_bit_cast(typename T::V8, r);
  }
};

// grid (kv heads, splits, sequences) or (kv heads, ranges by the batch's sum): ranges that there
// are come before those left over, which would take the place of others on a CU
template <int FMT, typename T, int D, int RT, int PARTS, int S>
__global__ __launch_bounds__(256, D == 256 ? 1 : RT == 1 ? 3 : 2) void attn_few_kernel(AttnParams p) {
  typedef Few<FMT, T, D, RT, PARTS> F;
  typedef typename T::V8 V8;
  extern __shared__ __align__(16) uint8_t lds[];  // 4 kWaveLds
  __shared__ float wave_m[4][16 * RT], wave_l[4][16 * RT];
  __shared__ int retry;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kvh = blockIdx.x;
  int part = blockIdx.y, size = INT32_MAX & ~127;
  Work w;
  if (p.budget) {
    size = range_tokens<S>(p);
    w = work_of<S>(p, part, [&](const Work& x) { return range_count(size, seen_tokens<S>(p, x)); });
  } else {
    w = sequence_work<S>(p, blockIdx.z);
  }
  if (w.rows == 0) return;
  const Seen top = row_sees<S>(p, w, 0), end = row_sees<S>(p, w, w.rows - 1);
  // rows see later tokens the later they are: the union is [top.lo, end.hi), what all see
  // [end.lo, top.hi)
  const int seen = seen_tokens<S>(p, w);
  size = p.budget ? range_tokens(size, seen) : p.splits > 1 ? split_tokens(p, seen) : size;
  const bool whole = p.budget ? seen <= size : p.splits == 1;  // the result is final
  const size_t slot0 = ((size_t)(blockIdx.z * gridDim.y + blockIdx.y) * p.cache.kv_heads + kvh) * (16 * RT);
  if ((int64_t)part * size >= seen) {  // a split that a short sequence has no tokens for
    for (int e = threadIdx.x; e < 2 * w.rows; e += 256)
      p.stats[slot0 * 2 + e] = e & 1 ? 0.0f : -__builtin_inff();
    return;
  }
  const int t0 = (top.lo & ~15) + part * size;
  const int t1 = (int)min((int64_t)t0 + size, (int64_t)end.hi);
  if (threadIdx.x == 0) retry = 0;
  __syncthreads();

  const int n = lane & 15, g = lane >> 4;
  uint8_t* my = lds + wave * F::kWaveLds;
  V8 q[RT][F::kSteps];
  float scale2[RT], rate[RT];  // the call's, of rows that were scaled times the inverse; of capped scores
  Seen see[RT];
  float slope2[RT];  // of shaped scores: the row's bias,
  int at[RT];        // its position less this lane's first token of a step
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int row = rt * 16 + n;
    const int r = row < w.rows ? row : 0;  // rows past the last repeat the first; nobody reads them
    see[rt] = row_sees<S>(p, w, r);
    const size_t qi =
        (size_t)(w.start + r / p.group) * p.q_stride + (size_t)(kvh * p.group + r % p.group) * D;
    if constexpr (S) {
      slope2[rt] = slope_of(p, kvh * p.group + r % p.group);
      at[rt] = w.first + r / p.group - 4 * g;
    }
    u32x4 raw[F::kSteps];
    float factor = 1.0f, most = 0.0f;
    scale2[rt] = p.scale2;
#pragma unroll
    for (int s = 0; s < F::kSteps; ++s) raw[s] = load_q8(p, qi + F::channel(s, g));
    if constexpr (F::kScaled) {
#pragma unroll
      for (int s = 0; s < F::kSteps; ++s) most = largest_bf16(raw[s], most);
      most = fmaxf(most, xor_lanes<16>(most));
      most = fmaxf(most, xor_lanes<32>(most));
      const uint32_t e = fit_exponent<S>(most);
      factor = fit_factor(e);
      scale2[rt] = fit_scale(p.scale2, e);
    }
#pragma unroll
    for (int s = 0; s < F::kSteps; ++s) q[rt][s] = query_operand<FMT, T, F::kScaled>(raw[s], factor);
  }
  float4v o[RT][D / 16];
  float m[RT], l[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = kNothing;
    l[rt] = 0.0f;
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) o[rt][dt] = float4v{0, 0, 0, 0};
  }
  bool again = false;
  // of the wave, and what scores are multiplied by as weights; far (kFar): less than 0 and 1
  float slack = kSlack + T::kRoom, unit[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    if constexpr (S == kEarly) slope2[rt] /= scale2[rt];
    if constexpr (S == kCapped) {
      rate[rt] = cap_rate(p, scale2[rt]);
      scale2[rt] = 2.0f * p.cap2;
      slope2[rt] /= scale2[rt];
    }
    unit[rt] = S == kLate ? 1.0f : scale2[rt];
  }

  typename F::Keys k;
  typename F::Values v;
  int page[2], next[2];  // of the step loaded; the table's entries for the one behind it
  auto find = [&](int t) __attribute__((always_inline)) {
#pragma unroll
    for (int a = 0; a < 2; ++a) next[a] = table_entry(p, w, t + 16 * a, max(t1, 1));
  };
  auto check = [&](int t) __attribute__((always_inline)) {
#pragma unroll
    for (int a = 0; a < 2; ++a) page[a] = page_ok(p, next[a], t + 16 * a, t1);
  };
  int t = t0 + 32 * wave;
  if (w.len > 0) {
    find(t);
    check(t);
    F::load_keys(p, page, kvh, t, lane, k);
    F::load_values(p, page, kvh, t, lane, v);
    find(t + 128);
  }
  for (; t < t1; t += 128) {
    const bool edge = t < end.lo || t + 32 > min(top.hi, t1) || page[0] < 0 || page[1] < 0;
    float4v s[RT][2];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        s[rt][a] = float4v{0, 0, 0, 0};
        if (S == kEarly) {
          const float away = (float)(at[rt] - t);
#pragma unroll
          for (int i = 0; i < 4; ++i) s[rt][a][i] = -slope2[rt] * fabsf(away - (float)(16 * a + i));
        }
      }
#pragma unroll
    for (int st = 0; st < F::kSteps; ++st)
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        V8 key[F::kParts];
        F::key(k, a, st, key);
#pragma unroll
        for (int part = 0; part < F::kParts; ++part)
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) s[rt][a] = T::mfma16(key[part], q[rt][st], s[rt][a]);
      }
    // values that some rows see and others do not must be finite for the product below (a
    // zero weight times an infinity is no zero); where they are not, the rows are done one
    // by one at the end
    const bool on0 = page[0] >= 0, on1 = page[1] >= 0;
    auto put = [&](int span) __attribute__((always_inline)) {
      if (edge) {
        const bool bad =
            F::template put_values<true>(v, span, my, lane, top.lo - t, min(end.hi, t1) - t, on0, on1);
        again = again || (bad && (top.lo < end.lo || top.hi < end.hi));
      } else {
        F::template put_values<false>(v, span, my, lane, 0, 32, true, true);
      }
    };
    put(0);
    // the next step's loads, always, so that a wait for them never has to count both ways
    // (behind the end they read the pool's first page, and nobody uses that)
    check(t + 128);
    F::load_keys(p, page, kvh, t + 128, lane, k);
    if (F::kSpans == 1) F::load_values(p, page, kvh, t + 128, lane, v);
    V8 w8[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float x[8], most = -__builtin_inff();
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = s[rt][i >> 2][i & 3];
      if constexpr (S == kCapped) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = squashed(x[i], rate[rt]);
        if (p.slopes) {
          const float away = (float)(at[rt] - t);
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = biased(x[i], slope2[rt], away - (float)((i >> 2) * 16 + (i & 3)));
        }
      }
      if constexpr (S == kLate) {
        const float away = (float)(at[rt] - t);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          x[i] = biased(capped(p, x[i] * scale2[rt]), slope2[rt], away - (float)((i >> 2) * 16 + (i & 3)));
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (edge) {
          const int token = t + (i >> 2) * 16 + 4 * g + (i & 3);
          const bool live = token >= see[rt].lo && token < min(see[rt].hi, t1) && ((i >> 2) ? on1 : on0);
          x[i] = live ? x[i] : -__builtin_inff();
        }
        most = fmaxf(most, x[i]);
      }
      if constexpr (S != kLate) most *= scale2[rt];
      if (__any(most - m[rt] > slack)) {
        most = fmaxf(most, xor_lanes<16>(most));
        most = fmaxf(most, xor_lanes<32>(most));
        const float up = fmaxf(m[rt], most - T::kRoom);
        const float f = __builtin_amdgcn_exp2f(m[rt] - up);
        m[rt] = up;
        l[rt] *= f;
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) o[rt][dt] *= f;
        if constexpr (S != kLate) slack = slack_at(up, slack);
        if (S != kLate && slack < 0.0f) {
          unit[rt] = 1.0f;
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] *= scale2[rt];
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = __builtin_amdgcn_exp2f(fmaf(x[i], unit[rt], -m[rt]));
        l[rt] += x[i];
        w8[rt][i] = (typename T::E)x[i];
      }
    }
#pragma unroll
    for (int span = 0; span < F::kSpans; ++span) {
      if (span) {
        put(span);
        if (span == F::kSpans - 1) F::load_values(p, page, kvh, t + 128, lane, v);
      }
#pragma unroll
      for (int i = 0; i < F::kSpan / 16; ++i)
#pragma unroll
        for (int part = 0; part < F::kParts; ++part) {
          const V8 val = F::value(my + part * F::kPart, i, lane);
          const int dt = span * (F::kSpan / 16) + i;
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) o[rt][dt] = T::mfma16(val, w8[rt], o[rt][dt]);
        }
    }
    // here, where no LDS read is waited for before the next step's keys are (a wait for one
    // waits for scalar loads as well)
    find(t + 256);
  }

  // the waves' results: maxima and sums, then weighted sums [row][channel] in LDS
  if (again) retry = 1;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    l[rt] += xor_lanes<16>(l[rt]);
    l[rt] += xor_lanes<32>(l[rt]);
    if (g == 0) {
      wave_m[wave][rt * 16 + n] = seen_max(m[rt]);
      wave_l[wave][rt * 16 + n] = l[rt];
    }
    float* out = (float*)my + (rt * 16 + n) * D;
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) *(float4v*)(out + dt * 16 + 4 * g) = o[rt][dt];
  }
  __syncthreads();
  if (retry) {
    // one row at a time, by the wave that then stands for all four
    __syncthreads();
    constexpr int E = D / 64;
    for (int row = wave; row < 16 * RT; row += 4) {
      float rm = -__builtin_inff(), rl = 0.0f, acc[E] = {};
      if (row < w.rows) {
        const Seen s = row_sees<S>(p, w, row);
        row_pass<E, S>(p, w, kvh, row, max(s.lo, t0), min(s.hi, t1), lane, rm, rl, acc);
      }
      for (int o4 = 0; o4 < 4; ++o4) {
        if (lane == 0) {
          wave_m[o4][row] = o4 ? -__builtin_inff() : rm;
          wave_l[o4][row] = o4 ? 0.0f : rl;
        }
        for (int e = 0; e < E; ++e) {
          const int d = E * lane + e;
          const int at = FMT == KV_Q4 ? (d & ~7) | place4(d & 7) : d;
          ((float*)(lds + o4 * F::kWaveLds))[row * D + at] = o4 ? 0.0f : acc[e];
        }
      }
    }
    __syncthreads();
  }
  // per row: the common maximum, the waves' weights against it, their sum
  if (threadIdx.x < 16 * RT) {
    const int row = threadIdx.x;
    float most = wave_m[0][row];
#pragma unroll
    for (int i = 1; i < 4; ++i) most = fmaxf(most, wave_m[i][row]);
    const float base = most == -__builtin_inff() ? 0.0f : most;
    float total = 0.0f, f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i] = __builtin_amdgcn_exp2f(wave_m[i][row] - base);
      total += wave_l[i][row] * f[i];
    }
    const float norm = !whole ? 1.0f : total != 0.0f ? 1.0f / total : 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) wave_l[i][row] = f[i] * norm;
    if (!whole && row < w.rows) {
      p.stats[(slot0 + row) * 2] = most;
      p.stats[(slot0 + row) * 2 + 1] = total;
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < w.rows * (D / 4); e += 256) {
    const int row = e / (D / 4), d = e % (D / 4) * 4;
    float sum[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float f = wave_l[i][row];
      const float* from = (const float*)(lds + i * F::kWaveLds) + row * D;
      if constexpr (FMT == KV_Q4) {
#pragma unroll
        for (int c = 0; c < 4; ++c) sum[c] += from[(d & ~7) | place4((d & 4) + c)] * f;
      } else {
        const float4v v = *(const float4v*)(from + d);
#pragma unroll
        for (int c = 0; c < 4; ++c) sum[c] += v[c] * f;
      }
    }
    if (whole) {
      uint16_t* to = (uint16_t*)p.y + (size_t)(w.start + row / p.group) * p.y_stride +
                     (size_t)(kvh * p.group + row % p.group) * D + d;
      const u32x2 y = {pack2(p.q_type, sum[0], sum[1]), pack2(p.q_type, sum[2], sum[3])};
      if (p.y_vec) {
        *(u32x2*)to = y;
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) to[c] = (uint16_t)(y[c / 2] >> (16 * (c & 1)));
      }
    } else {
      *(float4v*)(p.part + (slot0 + row) * D + d) = float4v{sum[0], sum[1], sum[2], sum[3]};
    }
  }
}

}  // namespace exl3
