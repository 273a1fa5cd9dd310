// Attention of many rows (tokens x heads of a group) over the cache: prefill chunks.
// The matrix cores bound it.
//
// A workgroup (4 waves) takes 128 rows of one sequence and cache head, 32 per wave, and
// walks the cache in tiles of TK tokens that its waves share in LDS (16-bit rows; codes
// are decoded once per workgroup on the way in).  Per tile and wave:
//   S^T = K Q^T   32x32x16 MFMAs, K from LDS as the A operand, the wave's queries in
//                 registers as the B operand.  Lane l holds scores of query l % 32 only, so
//                 a row's maximum and sum stay in the lane (its other half in lane l ^ 32);
//   P             rounded to 16 bits, already the next product's B operand, its sum f32 of the
//                 unrounded ones, the maximum with kSlack, as in attn_few_kernel;
//   O^T += V^T P^T  V read from LDS transposed.
// Shaped scores (S, exl3_attn.hpp): a bias is where S^T's sums start; a cap puts four instructions a
// score behind the first product.
// The next tile's loads are in flight meanwhile, straight into the other half of LDS or,
// coded ones, into registers and from there decoded behind the products: one barrier per
// tile.  Two workgroups share a CU (heads of 64: three), so that one's exponentials run beside
// the other's products.
//
// Coded values are one or two f16 by the queries' type (scale_parts): two double the products,
// in tiles half as long where the others' would leave one workgroup a CU.  With one, f16
// results are off by 5.3e-4 to 8.1e-4 in the 2-norm, with two by 2.9e-4, where rounding the
// exact ones takes 2.1e-4.
//
// Measured (us, TFLOP/s of the products that the mask leaves; one box): 2048 tokens over 16384
// bf16 ones, 32 heads of 128 on 8: 496, 1040 -- a large product of the library's runs at 1238 --
// with the matrix units busy half of the cycles and the exponentials beside them; 2048 over
// 8192 bf16 998 TFLOP/s, f16 952, 8 bits 815 in one part and 477 in two, 4 bits 820 and 410; heads
// of 64 733 to 757, 610 / 431, 514 / 370 (half the products per exponential); of 256 630, 475 / 348,
// 486 / 337 (one workgroup a CU: its registers).  Six prompts of 496 to 1500 tokens, heads of 64,
// window 512: 46 us, 432 TFLOP/s, masked tiles and two rounds of short workgroups.
// Shaped, 2048 tokens over 8192, us on two machines, plain | biased | capped | both | with a prefix only:
//   bf16 heads of 128       239, 252 | 248, 260 | 288, 302 | 311, 326 | 240, 252
//   f16 heads of 64         153, 159 | 161, 167 | 208, 222 | 232, 233 | 154, 159
//   bf16 heads of 256       684, 678 | 750, 743 | 781, 746 | 806, 798 | 709, 720
//   bf16 over 8 bits        294, 308 | 292, 306 | 350, 365 | 363, 376 | 295, 309
//   f16 over 8 bits         504, 526 | 490, 512 | 554, 578 | 547, 570 | 507, 528
//   bf16 over 4 bits        293, 305 | 292, 304 | 348, 364 | 362, 370 | 294, 305
//   f16 over 4 bits         593, 603 | 606, 602 | 659, 662 | 682, 677 | 593, 601
// Kernels that looked for a bias under each cap and started a prefix' sums from a bias of zero (another
// machine): capped 318 for 310, heads of 64 229, of 256 845; with a prefix only 267 for 259, 173, 808.
// Where rows are done one by one (below, values that are not finite and some rows do not see) a
// workgroup takes its rows times its tokens: one NaN in the newest of 8192 tokens makes 2048 rows'
// 0.29 ms 268 ms.
#pragma once

#include "exl3_attn.hpp"

namespace exl3 {

constexpr int kManyRows = 128;

template <int FMT, typename T, int D, int PARTS>
struct Many {
  static constexpr bool kRaw = FMT >= 9;
  static constexpr int kTokens = D * PARTS >= 256 ? 32 : 64;            // of a tile
  static constexpr int kRow = kRaw ? 2 * D : FMT == KV_Q8 ? D : D / 2;  // bytes of a cached head
  static constexpr int kLanes = kRow / 16;                              // lanes that load a row
  static constexpr int kRows = 64 / kLanes;                             // rows of a wave's load
  static constexpr int kMine = kTokens / 4;                             // a wave's rows of a tile
  static constexpr int kLoads = kMine > kRows ? kMine / kRows : 1;
  static constexpr int kTile = kTokens * D * 2;                         // bytes in LDS
  static constexpr int kHalf = 2 * PARTS * kTile;                       // keys' parts, values' parts
  static constexpr int kLds = 2 * kHalf;
  static constexpr int kGroups = D == 256 ? 1 : D == 64 && PARTS == 1 ? 3 : 2;  // workgroups that share a CU

  struct Loads {  // of coded caches
    u32x4 k[kLoads], v[kLoads];
    uint32_t ks[kLoads], vs[kLoads];  // (16-bit elements would go through scratch)
  };

  // Byte of 16-byte chunk c of row t.  A key read takes one chunk of 16 rows at a time, a
  // value read 64 bytes of 4 rows: both fall into different banks.
  static __device__ __forceinline__ int key_swizzle(int t) { return D == 64 ? (t >> 1) & 7 : t & 15; }
  static __device__ __forceinline__ int value_swizzle(int t) { return D == 64 ? ((t >> 1) & 1) << 2 : (t & 3) << 2; }
  static __device__ __forceinline__ int key_place(int t, int c) { return t * D * 2 + ((c ^ key_swizzle(t)) << 4); }
  static __device__ __forceinline__ int value_place(int t, int c) { return t * D * 2 + ((c ^ value_swizzle(t)) << 4); }

  // Wave w loads rows kMine w .. of a tile, all of one page: its row of load u.
  static __device__ __forceinline__ int row_of(int u, int lane) { return u * kRows + lane / kLanes; }

  // 16-bit caches: the wave's rows of the tile at t0 from page `page` straight into LDS
  // (keys and values of rows `first` on); whoever waits for them waits with vmcnt.  A load
  // fills 1 KB in lane order, so a lane fetches the chunk that belongs at its place.
  static __device__ __forceinline__ void copy(const AttnParams& p, int kvh, int page, int t, int first, int lane,
                                              uint8_t* keys, uint8_t* values) {
    const KvCacheView& c = p.cache;
    const int ch = lane % kLanes;
    const size_t h = (size_t)max(page, 0) * c.kv_heads + kvh;
    const size_t at = ((h << c.page_shift) + (t & ((1 << c.page_shift) - 1))) * kRow;
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int r = row_of(u, lane), to = (first + u * kRows) * D * 2;
      lds_dma16_s(c.k + at, r * kRow + ((ch ^ key_swizzle(first + r)) << 4), lds_offset(keys) + to);
      lds_dma16_s(c.v + at, r * kRow + ((ch ^ value_swizzle(first + r)) << 4), lds_offset(values) + to);
    }
  }
  // Their values on an edge, once they are there: rows outside [lo, hi) become zeros.
  // Returns whether the others hold a value that is not finite.
  static __device__ __forceinline__ bool clear(uint8_t* values, int first, int lane, int lo, int hi) {
    bool bad = false;
#pragma unroll 1
    for (int u = 0; u < kLoads; ++u) {
      const int t = first + row_of(u, lane);
      u32x4* at = (u32x4*)(values + (first + u * kRows) * D * 2 + lane * 16);
      const u32x4 v = *at;
      if (t >= lo && t < hi)
        bad = bad || not_finite<T>(v);
      else
        *at = u32x4{0, 0, 0, 0};
    }
    return bad;
  }

  // Coded caches: the same rows into registers.
  static __device__ __forceinline__ void load(const AttnParams& p, int kvh, int page, int t, int lane, Loads& x) {
    const KvCacheView& c = p.cache;
    const int ch = lane % kLanes;
    const size_t h = (size_t)max(page, 0) * c.kv_heads + kvh;
    const int slot = t & ((1 << c.page_shift) - 1);
    const uint8_t* k = c.k + ((h << c.page_shift) + slot) * kRow;
    const uint8_t* v = c.v + ((h << c.page_shift) + slot) * kRow;
    const size_t s = ((h * (D / 32)) << c.page_shift) + slot;
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int r = kRows > kMine ? row_of(u, lane) & (kMine - 1) : row_of(u, lane);
      const int g = ((ch * (16 * D / kRow) / 32) << c.page_shift) + r;
      x.k[u] = *(const u32x4*)(k + r * kRow + ch * 16);
      x.v[u] = *(const u32x4*)(v + r * kRow + ch * 16);
      x.ks[u] = (c.ks + s)[g];
      x.vs[u] = (c.vs + s)[g];
    }
  }
  // Eight channels of a lane's load, times a scale.
  static __device__ __forceinline__ u32x4 decoded(const u32x4& w, _Float16 s, int i) {
    if constexpr (FMT == KV_Q8) {
      const uint32_t a = w[2 * i], b = w[2 * i + 1];
      return decode8(a, b, s);
    }
    const uint32_t a = w[i & 3];
    return decode4(a, s);
  }
  // And decoded to LDS, with what clear() does on an edge.
  static __device__ __forceinline__ bool put(const Loads& x, uint8_t* keys, uint8_t* values, int first, int lane,
                                             bool edge, int lo, int hi) {
    constexpr int n = FMT == KV_Q8 ? 2 : 4;  // 16-byte chunks of a lane's load
    const int ch = lane % kLanes;
    bool bad = false;
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int t = first + row_of(u, lane);
      if (kRows > kMine && row_of(u, lane) >= kMine) continue;
      const bool live = !edge || (t >= lo && t < hi);
      if (edge && live) bad = bad || past_f16<FMT>(x.vs[u]);
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const int kat = key_place(t, ch * n + i), vat = value_place(t, ch * n + i);
        _Float16 hi, lo;
        scale_parts<FMT, PARTS>(x.ks[u], hi, lo);
        *(u32x4*)(keys + kat) = decoded(x.k[u], hi, i);
        if constexpr (PARTS == 2) *(u32x4*)(keys + kTile + kat) = decoded(x.k[u], lo, i);
        scale_parts<FMT, PARTS>(x.vs[u], hi, lo);
        const u32x4 none = {0, 0, 0, 0};
        *(u32x4*)(values + vat) = live ? decoded(x.v[u], hi, i) : none;
        if constexpr (PARTS == 2) *(u32x4*)(values + kTile + vat) = live ? decoded(x.v[u], lo, i) : none;
      }
    }
    return bad;
  }
};

// One-dimensional grid of tiles x splits x kv heads, the heads fastest (blocks go to the
// XCDs in turn, so a head's tiles share few L2s), a sequence's last and longest tiles first.
template <int FMT, typename T, int D, int PARTS, int S>
__global__ __launch_bounds__(256)
__attribute__((amdgpu_waves_per_eu(Many<FMT, T, D, PARTS>::kGroups, Many<FMT, T, D, PARTS>::kGroups)))
void attn_many_kernel(AttnParams p, int tiles) {
  typedef Many<FMT, T, D, PARTS> F;
  typedef typename T::V8 V8;
  constexpr int TK = F::kTokens, NT = TK / 32;
  extern __shared__ __align__(16) uint8_t lds[];
  __shared__ int retry, page_on[2][4];  // [half of LDS][wave whose rows they are]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kvh = blockIdx.x % p.cache.kv_heads, rest = blockIdx.x / p.cache.kv_heads;
  const int split = rest % p.splits, tile = tiles - 1 - rest / p.splits;
  int row0;
  const Work w = tile_work<S>(p, tile, kManyRows, row0);
  const int rows = min(w.rows - row0, kManyRows);
  if (rows <= 0) return;
  const Seen top = row_sees<S>(p, w, row0), end = row_sees<S>(p, w, row0 + rows - 1);
  const int lo = top.lo & ~15, seen = max(end.hi - lo, 0), size = split_tokens(p, seen);
  const int t0 = (int)min((int64_t)lo + (int64_t)split * size, (int64_t)INT32_MAX - 4095);
  const int t1 = (int)min((int64_t)t0 + size, (int64_t)end.hi);
  const size_t slot0 = ((size_t)(tile * p.splits + split) * p.cache.kv_heads + kvh) * kManyRows;
  if (p.splits > 1 && t0 >= t1) {
    for (int e = threadIdx.x; e < 2 * rows; e += 256)
      p.stats[slot0 * 2 + e] = e & 1 ? 0.0f : -__builtin_inff();
    return;
  }
  if (threadIdx.x == 0) retry = 0;

  const int n = lane & 31, h = lane >> 5;
  // this wave's rows, what all of them see and what any of them sees
  const int wrow = row0 + 32 * wave;
  const bool busy = 32 * wave < rows;
  const int mine = min(wrow + n, row0 + rows - 1);  // rows past the last repeat it; nobody reads them
  const Seen see = row_sees<S>(p, w, mine);
  const Seen wtop = row_sees<S>(p, w, min(wrow, row0 + rows - 1));
  const Seen wend = row_sees<S>(p, w, min(wrow + 31, row0 + rows - 1));
  V8 q[D / 16];
  float scale2 = p.scale2;  // of rows that were scaled times the inverse
  {
    constexpr bool kScaled = !F::kRaw && PARTS == 1;  // bf16 queries, to fit f16
    const size_t qi = (size_t)(w.start + mine / p.group) * p.q_stride +
                      (size_t)(kvh * p.group + mine % p.group) * D;
    u32x4 raw[D / 16];
    float factor = 1.0f, most = 0.0f;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) raw[s] = load_q8(p, qi + 16 * s + 8 * h);
    if constexpr (kScaled) {
#pragma unroll
      for (int s = 0; s < D / 16; ++s) most = largest_bf16(raw[s], most);
      most = fmaxf(most, xor_lanes<32>(most));
      const uint32_t e = fit_exponent<S>(most);
      factor = fit_factor(e);
      scale2 = fit_scale(p.scale2, e);
    }
#pragma unroll
    for (int s = 0; s < D / 16; ++s) q[s] = query_operand<FMT == KV_Q4 ? KV_Q8 : FMT, T, kScaled>(raw[s], factor);
  }
  // of shaped scores: the row's bias, its position less this lane's first token of a tile
  constexpr bool kCap = S == kCapped || S == kBoth;
  float slope2 = S == kEarly || S == kBoth || S == kLate ? slope_of(p, kvh * p.group + mine % p.group) : 0.0f;
  const int at = w.first + mine / p.group - 4 * h, nearest = w.first + wrow / p.group;
  const float rate = kCap ? cap_rate(p, scale2) : 0.0f;
  if (kCap) scale2 = 2.0f * p.cap2;
  if (S == kEarly || S == kBoth) slope2 /= scale2;
  float16v o[D / 32];
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt) o[dt] = float16v{};
  float m = kNothing, l = 0.0f;
  bool again = false;
  // of the wave, and what scores are multiplied by as weights; far (kFar): less than 0 and 1
  float slack = kSlack + T::kRoom, unit = S == kLate ? 1.0f : scale2;

  typename F::Loads x;
  const int off = F::kMine * wave;  // of this wave's rows in a tile
  // biased scores mostly rise towards the row's own position: newest tiles first, so that the running
  // maximum rarely moves (2048 biased rows over 8192 tokens, us: heads of 128 the other way 279, this one
  // 250; of 64 183 and 159; of 256 993 and 755)
  constexpr bool kBack = S == kEarly || S == kBoth || S == kLate;
  const int first = kBack && t0 < t1 ? t0 + (t1 - t0 - 1) / TK * TK : t0, step = kBack ? -TK : TK;
  auto entry_at = [&](int t) { return table_entry(p, w, kBack ? max((t + off) & ~15, 0) : (t + off) & ~15, t1); };
  auto page_at = [&](int entry, int t) { return page_ok(p, entry, (t + off) & ~15, t1); };
  // starts the loads of the tile at t, and ends them in half `half` of LDS
  auto fetch = [&](int t, int page, int half) __attribute__((always_inline)) {
    uint8_t* buf = lds + half * F::kHalf;
    if constexpr (F::kRaw)
      F::copy(p, kvh, page, t + off, off, lane, buf, buf + PARTS * F::kTile);
    else
      F::load(p, kvh, page, t + off, lane, x);
  };
  auto stage = [&](int t, int page, int half) __attribute__((always_inline)) {
    uint8_t* buf = lds + half * F::kHalf;
    // an edge: some row of the workgroup does not see some token of the tile
    const bool edge = t < end.lo || t + TK > min(top.hi, t1) || page < 0;
    const int lo = top.lo - t, hi = page < 0 ? 0 : min(end.hi, t1) - t;
    bool bad = false;
    if constexpr (F::kRaw) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      if (edge) bad = F::clear(buf + PARTS * F::kTile, off, lane, lo, hi);
    } else {
      bad = F::put(x, buf, buf + PARTS * F::kTile, off, lane, edge, lo, hi);
    }
    again = again || (bad && (top.lo < end.lo || top.hi < end.hi));
    if (lane == 0) page_on[half][wave] = page >= 0;
  };
  int page = -1, next = -1;  // of the tile in flight; the table's entry for the one behind it
  if (t0 < t1) {
    next = entry_at(first);
    page = page_at(next, first);
    fetch(first, page, 0);
    next = entry_at(first + step);
    stage(first, page, 0);
  }
  // the queries are here before the loop: a wait for them inside it would be one for the
  // tile in flight
#pragma unroll
  for (int st = 0; st < D / 16; ++st) asm volatile("" : "+v"(q[st]));
  int cur = 0;
  for (int t = first; t < t1 && (!kBack || t >= t0); t += step, cur ^= 1) {
    __syncthreads();
    const uint8_t* keys = lds + cur * F::kHalf;
    const uint8_t* values = keys + PARTS * F::kTile;
    // always, so that no later wait has to count both ways (behind the end: the pool's first
    // page, and nobody uses it)
    page = page_at(next, t + step);
    fetch(t + step, page, cur ^ 1);
    if (busy && t < wend.hi && t + TK > wtop.lo) {
      // The compiler orders these reads and products for few registers, each product right
      // behind its read; pin() keeps kDepth reads ahead of the products.
      constexpr int N = NT * PARTS, QK = N * (D / 16), kDepth = 4;
      float16v s[N];  // of part c of block a: s[a + NT c]
      auto key = [&](int i) __attribute__((always_inline)) {
        const int a = i % NT, c = i / NT % PARTS, st = i / N;
        return *(const V8*)(keys + c * F::kTile + F::key_place(32 * a + n, 2 * st + h));
      };
      V8 kf[kDepth];
#pragma unroll
      for (int i = 0; i < kDepth; ++i) kf[i] = key(i);
      if constexpr (S == kEarly) {
        const float away = (float)(at - t);
        // well behind all rows one instruction each: rounded at the tile's border, from where a token
        // lies at most twice as far as the nearest one, it is off by 2^-23 of itself
        if (t + 2 * TK <= nearest) {
          const float from = -slope2 * away;
#pragma unroll
          for (int i = 0; i < 16 * NT; ++i)
            s[i / 16][i % 16] = fmaf(slope2, (float)(32 * (i / 16) + 8 * (i % 16 / 4) + i % 4), from);
        } else {
#pragma unroll
          for (int i = 0; i < 16 * NT; ++i)
            s[i / 16][i % 16] = -slope2 * fabsf(away - (float)(32 * (i / 16) + 8 * (i % 16 / 4) + i % 4));
        }
      }
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int i = 0; i < QK; ++i) {
        pin();
        if (i < N && (S != kEarly || i >= NT)) s[i] = float16v{};
        s[i % N] = T::mfma32(kf[i % kDepth], q[i / N], s[i % N]);
        if (i + kDepth < QK) kf[i % kDepth] = key(i + kDepth);
      }
      if constexpr (PARTS == 2) {
#pragma unroll
        for (int a = 0; a < NT; ++a) s[a] += s[a + NT];
      }
      // product i of the second kind: 16 tokens, part of their values, 32 channels
      constexpr int DT = D / 32, PV = TK / 16 * PARTS * DT;
      auto value = [&](int i) __attribute__((always_inline)) {
        const int ks = i / (PARTS * DT), c = i / DT % PARTS, dt = i % DT;
        const int tok = 16 * ks + 4 * h + ((lane >> 2) & 3);
        const int chunk = dt * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1), half = (lane & 1) * 8;
        const uint8_t* from = values + c * F::kTile + half;
        const u32x2 lo = lds_transpose4(from + F::value_place(tok, chunk));
        const u32x2 hi = lds_transpose4(from + F::value_place(tok + 8, chunk));
        const u32x4 r = {lo[0], lo[1], hi[0], hi[1]};
        return __builtin_bit_cast(V8, r);
      };
      V8 vf[DT];
#pragma unroll
      for (int i = 0; i < DT; ++i) vf[i] = value(i);
      pin();
      __builtin_amdgcn_s_setprio(0);
      if constexpr (kCap) {
#pragma unroll
        for (int i = 0; i < 16 * NT; ++i) s[i / 16][i % 16] = squashed(s[i / 16][i % 16], rate);
      }
      if constexpr (S == kBoth) {
        pin();  // caps first: both at once 320 us for 311 (2048 rows over 8192, heads of 128), 240 for 235 (of 64)
        const float away = (float)(at - t);
#pragma unroll
        for (int i = 0; i < 16 * NT; ++i)
          s[i / 16][i % 16] = biased(s[i / 16][i % 16], slope2, away - (float)(32 * (i / 16) + 8 * (i % 16 / 4) + i % 4));
      }
      if constexpr (S == kLate) {
        const float away = (float)(at - t);
#pragma unroll
        for (int i = 0; i < 16 * NT; ++i)
          s[i / 16][i % 16] = biased(capped(p, s[i / 16][i % 16] * scale2), slope2,
                                     away - (float)(32 * (i / 16) + 8 * (i % 16 / 4) + i % 4));
      }
      if (t < wend.lo || t + TK > min(wtop.hi, t1)) {
        // token r of the tile is one of the row's `n` from `lo` on
        const int lo = see.lo - t - 4 * h, n = max(min(see.hi, t1) - see.lo, 0);
#pragma unroll
        for (int a = 0; a < NT; ++a)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int r = 32 * a + 8 * (i / 4) + i % 4;
            s[a][i] = (uint32_t)(r - lo) < (uint32_t)n ? s[a][i] : -__builtin_inff();
          }
      }
      // where a page is missing, so are its tokens
      const int* on = page_on[cur];
      if (!__builtin_amdgcn_readfirstlane(on[0] & on[1] & on[2] & on[3])) {
#pragma unroll
        for (int a = 0; a < NT; ++a)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            s[a][i] = on[(2 * a + i / 8) * 16 / F::kMine] ? s[a][i] : -__builtin_inff();
      }
      float most = s[0][0];
#pragma unroll
      for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int i = 0; i < 16; ++i) most = fmaxf(most, s[a][i]);
      if constexpr (S != kLate) most *= scale2;
      if (__any(most - m > slack)) {
        most = fmaxf(most, xor_lanes<32>(most));
        const float up = fmaxf(m, most - T::kRoom);
        const float f = __builtin_amdgcn_exp2f(m - up);
        m = up;
        l *= f;
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) o[dt] *= f;
        if constexpr (S != kLate) slack = slack_at(up, slack);
        if (S != kLate && slack < 0.0f) {
          unit = 1.0f;
#pragma unroll
          for (int a = 0; a < NT; ++a)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[a][i] *= scale2;
        }
      }
      V8 w8, following;
      auto weight = [&](int ks, int i) __attribute__((always_inline)) {
        const float e = __builtin_amdgcn_exp2f(fmaf(s[ks / 2][8 * (ks & 1) + i], unit, -m));
        l += e;
        return (typename T::E)e;
      };
#pragma unroll
      for (int i = 0; i < 8; ++i) following[i] = weight(0, i);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int i = 0; i < PV; ++i) {
        const int ks = i / (PARTS * DT), dt = i % DT;
        if (i % (PARTS * DT) == 0) w8 = following;
        pin();
        o[dt] = T::mfma32(vf[dt], w8, o[dt]);
        if (i + DT < PV) vf[dt] = value(i + DT);
        if (i % (PARTS * DT) < DT && ks + 1 < TK / 16) {  // beside it the next 16 tokens' weights
#pragma unroll
          for (int e = 0; e < 8 / DT; ++e) following[dt * (8 / DT) + e] = weight(ks + 1, dt * (8 / DT) + e);
        }
      }
      pin();
      __builtin_amdgcn_s_setprio(0);
    }
    if (kBack ? t > t0 : t + TK < t1)
      stage(t + step, page, cur ^ 1);
    else if (F::kRaw)
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // LDS is not left to loads in flight
    next = entry_at(t + 2 * step);
  }
  if (again) retry = 1;
  __syncthreads();
  l += xor_lanes<32>(l);
  if (retry) {
    // values that some rows see and others do not were not finite (a zero weight times an
    // infinity is no zero): one row at a time, touching only what it sees
    constexpr int E = D / 64;
    for (int r = wave; r < rows; r += 4) {
      const int row = row0 + r;
      const Seen s = row_sees<S>(p, w, row);
      float rm, rl, acc[E];
      row_pass<E, S>(p, w, kvh, row, max(s.lo, t0), min(s.hi, t1), lane, rm, rl, acc);
      const size_t yi = (size_t)(w.start + row / p.group) * p.y_stride +
                        (size_t)(kvh * p.group + row % p.group) * D + E * lane;
      for (int e = 0; e < E; ++e) {
        if (p.splits == 1)
          store1(p.y, p.q_type, yi + e, rl != 0.0f ? acc[e] / rl : 0.0f);
        else
          p.part[(slot0 + r) * D + E * lane + e] = acc[e];
      }
      if (p.splits > 1 && lane == 0) {
        p.stats[(slot0 + r) * 2] = rm;
        p.stats[(slot0 + r) * 2 + 1] = rl;
      }
    }
    return;
  }
  if (32 * wave + n >= rows) return;
  if (p.splits > 1) {
    float* out = p.part + (slot0 + 32 * wave + n) * D;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *(float4v*)(out + 32 * dt + 8 * i + 4 * h) =
            float4v{o[dt][4 * i], o[dt][4 * i + 1], o[dt][4 * i + 2], o[dt][4 * i + 3]};
    if (h == 0) {
      p.stats[(slot0 + 32 * wave + n) * 2] = seen_max(m);
      p.stats[(slot0 + 32 * wave + n) * 2 + 1] = l;
    }
    return;
  }
  const float inv = l != 0.0f ? 1.0f / l : 0.0f;
  const size_t yi = (size_t)(w.start + mine / p.group) * p.y_stride +
                    (size_t)(kvh * p.group + mine % p.group) * D;
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint16_t y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float v = o[dt][4 * i + e] * inv;
        y[e] = p.q_type == DT_F16 ? f2h(v) : f2bf(v);
      }
      uint16_t* to = (uint16_t*)p.y + yi + 32 * dt + 8 * i + 4 * h;
      if (p.y_vec) {
        *(u32x2*)to = u32x2{(uint32_t)y[0] | (uint32_t)y[1] << 16, (uint32_t)y[2] | (uint32_t)y[3] << 16};
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) to[e] = y[e];
      }
    }
}

}  // namespace exl3
