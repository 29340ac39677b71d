// Attention of one new token a sequence over the paged cache: work units and their spans, the 16-bit cache's stream of keys,
// the kernels that a stream makes, and the launch plan.  decode.hip tells the whole.
#pragma once

#include "attend.hpp"
#include "shared.hpp"

#include <algorithm>
#include <type_traits>

namespace latent {
namespace attend {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kStep = 32;               // keys of a wave's step
constexpr int kTile = kStep * kWaves;   // keys of a work item
constexpr int kMaxGroups = 512;         // workgroups of a launch: two on every CU
// Over 8-bit caches twice as many, whose waves have half the bytes under way (35 sequences of 16 to 16000: 66 us, 70 with 512; 64 of
// 8000: 216 and 236; but 32 of 3400 61 and 57, which are even spans either way).
constexpr uint32_t kMaxGroups8 = 1024;

struct DecodeParams {
  Cache cache;
  const char* q;
  char* out;
  float* lse;
  const int32_t* lengths;
  int64_t q_token, q_head, o_token, o_head;  // bytes
  uint32_t B, Hq, G, D;
  uint32_t chunks;     // chunks of a head's query heads
  uint32_t rows;       // query heads of a chunk (the last may have fewer)
  uint32_t U;          // units of a sequence: n_kv_head * chunks
  bool whole;          // a workgroup a unit
  float scale_log2;
  // Workspace: parts [groups][2][rows] (max, sum), [groups][2][rows][D] rows, and for each unit its first workgroup and number of parts.
  float* part_ml;
  float* part_acc;
  int2* unit_parts;
};
// What only 8-bit caches and shared prefixes take, apart from what every launch has to fetch (96 sequences of up to 2500 tokens, 20 heads of 64 over
// one: 17.0 us the whole call, 17.1 with all of it in one structure).
struct MoreParams : DecodeParams {
  Scales scales;  // of an 8-bit cache
  // kAfter: keys here begin at position `ahead`, which cache.pages and cache.max_len leave out; what rows have seen before it is `prior`.  Every
  // unit leaves its rows, those that one workgroup has whole by themselves: sums [units][rows][2] and rows [units][rows][D].
  Prior prior;
  // kTable streams: the first pages of every sequence, which its row of cache.pages need not name.
  const int32_t* prefix;
  uint32_t prefix_pages;
  float* unit_ml;
  float* unit_acc;
  uint32_t ahead;
};
template <bool kMore>
using Params = std::conditional_t<kMore, MoreParams, DecodeParams>;

template <bool kAfter>
__device__ __forceinline__ uint32_t length_of(const Params<kAfter>& p, uint32_t b) {
  const int32_t n = p.lengths[b];
  if constexpr (kAfter) return n < static_cast<int64_t>(p.ahead) ? 0u : min(static_cast<uint32_t>(n) - p.ahead, p.cache.max_len);
  return n < 0 ? 0u : min(static_cast<uint32_t>(n), p.cache.max_len);
}

// The workgroup's span of tiles and the sequence it starts in.
struct Span {
  uint32_t begin, end;  // of all tiles
  uint32_t per;         // tiles of a workgroup
  uint32_t b;           // first sequence
  uint32_t base;        // tiles (of one unit each) of the sequences before it
};

__device__ __forceinline__ uint32_t wave_scan(uint32_t v, int lane) {  // inclusive
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const uint32_t o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  return v;
}

__device__ __forceinline__ uint32_t tiles_of(uint32_t len) { return (len + kTile - 1) / kTile; }

template <bool kAfter>
__device__ __forceinline__ Span find_span(const Params<kAfter>& p, int lane) {
  uint32_t total = 0;
  for (uint32_t b0 = 0; b0 < p.B; b0 += kWave) {
    const uint32_t b = b0 + lane;
    total += b < p.B ? tiles_of(length_of<kAfter>(p, b)) : 0;
  }
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) total += __shfl_xor(total, d);
  total *= p.U;
  Span s;
  s.per = max(1u, (total + gridDim.x - 1) / gridDim.x);
  s.begin = min(total, s.per * blockIdx.x);
  s.end = min(total, s.begin + s.per);
  s.b = 0;
  s.base = 0;
  if (s.begin == s.end) return s;
  const uint32_t at = s.begin / p.U;  // the sequence's tiles cover [base U, (base + its tiles) U)
  for (uint32_t b0 = 0; b0 < p.B; b0 += kWave) {
    const uint32_t b = b0 + lane, n = b < p.B ? tiles_of(length_of<kAfter>(p, b)) : 0;
    const uint32_t upto = s.base + wave_scan(n, lane);
    const uint64_t past = __ballot(upto > at);
    if (past) {
      const int first = __builtin_ctzll(past);
      s.b = b0 + first;
      s.base = __shfl(upto - n, first);
      break;
    }
    s.base = __shfl(upto, kWave - 1);
  }
  return s;
}

template <int kMT, int kVec>
struct Rows {  // a wave's running softmax: lane (query lane & 15, dims 4 kVec (lane >> 4) ..)
  float m[kMT], l[kMT];  // l: this lane's keys; sums and rows are times 2^kLift
  f32x4 acc[kMT][kVec];
};

// Pairs eight loaded value rows into the operand of product i: dword a holds keys 2a, 2a + 1 at element i.
template <int kVec>
__device__ __forceinline__ u32x4 pair_rows(const uint32_t (&v)[8][kVec / 2], int i) {
  u32x4 r;
#pragma unroll
  for (int a = 0; a < 4; ++a)
    r[a] = __builtin_amdgcn_perm(v[2 * a + 1][i / 2], v[2 * a][i / 2], (i & 1) ? 0x07060302u : 0x05040100u);
  return r;
}

// Rows of a cache that is larger than what the last-level cache keeps from step to step pass it by.
template <bool kOnce, typename T>
__device__ __forceinline__ T load_row(const char* at) {
  if constexpr (kOnce) return __builtin_nontemporal_load(reinterpret_cast<const T*>(at));
  return *reinterpret_cast<const T*>(at);
}

template <typename E_, int kDP_, bool kExact_, int kMT_, bool kPage8, bool kOnce, bool kTable>
struct Stream {
  typedef E_ E;
  static constexpr int kDP = kDP_, kMT = kMT_, kVec = kDP / 16, kK = kDP / 32;
  static constexpr bool kExact = kExact_;
  static constexpr int kRound = kDP <= 128 ? kMT : 1;  // row blocks that the waves exchange at once
  static constexpr int kPerSimd = kDP == 256 ? 1 : 2;  // waves
  static constexpr bool kMore = kTable;
  // The first of the eight dimensions that lane quarter kq holds of product s.
  static __device__ __forceinline__ int q_dim(int s, int kq) { return 32 * s + 8 * kq; }

  const Params<kMore>& p;
  int lane, kq;
  uint32_t len;
  const int32_t* pages;
  const char* kbase;
  const char* vbase;
  __device__ __forceinline__ Stream(const Params<kMore>& p, int lane, int kq, uint32_t len, uint32_t b, uint32_t hk)
      : p(p), lane(lane), kq(kq), len(len), pages(p.cache.pages + b * p.cache.pages_stride), kbase(p.cache.k + hk * p.cache.k_head),
        vbase(p.cache.v + hk * p.cache.v_head) {}

  // Where a step's keys lie: a page and the row in it.  Eight neighbours from a
  // multiple of eight share a page where pages hold multiples of eight rows.
  struct Place {
    int32_t page;  // outside [0, n_pages): masked
    uint32_t row;
  };
  struct Places {
    Place k[kPage8 ? 1 : 2], v[kPage8 ? 1 : 8];
  };
  __device__ __forceinline__ Place place_of(uint32_t key) const {
    const uint32_t slot = p.cache.by_page.of(key);
    const int32_t* of = pages;
    if constexpr (kTable) of = slot < p.prefix_pages ? p.prefix : pages;
    return {key < len ? of[slot] : -1, key - slot * p.cache.page_size};
  }
  // Row m of score block blk is key 8 (m / 4) + 4 blk + m % 4 of the step: lane (query, kq) then holds keys 8 kq .. + 7.
  __device__ __forceinline__ uint32_t k_key(uint32_t kb, int blk) const { return kb + 8 * ((lane & 15) >> 2) + 4 * blk + (lane & 3); }
  __device__ __forceinline__ Places places(uint32_t kb) const {
    Places r;
    if constexpr (kPage8) {
      r.k[0] = place_of(kb + 8 * ((lane & 15) >> 2));
      r.v[0] = place_of(kb + 8 * kq);
    } else {
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) r.k[blk] = place_of(k_key(kb, blk));
#pragma unroll
      for (int j = 0; j < 8; ++j) r.v[j] = place_of(kb + 8 * kq + j);
    }
    return r;
  }
  __device__ __forceinline__ bool valid(uint32_t key, int32_t page) const {
    return key < len && static_cast<uint32_t>(page) < p.cache.n_pages;
  }

  __device__ __forceinline__ void load_k(uint32_t kb, const Places& at, u32x4 (&k)[2][kK]) const {
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      const Place pl = at.k[kPage8 ? 0 : blk];
      const uint32_t row_in = kPage8 ? pl.row + 4 * blk + (lane & 3) : pl.row;
      const char* row = valid(k_key(kb, blk), pl.page) ? kbase + pl.page * p.cache.k_page + row_in * p.cache.k_row
                                                       : reinterpret_cast<const char*>(kZeroRow);
#pragma unroll
      for (int s = 0; s < kK; ++s) {
        const int d = 32 * s + 8 * kq;
        if constexpr (kExact) {
          k[blk][s] = load_row<kOnce, u32x4>(row + 2 * d);
        } else {
          const u32x4 x = load_row<kOnce, u32x4>(row + 2 * min(d, static_cast<int>(p.D) - 8));
          k[blk][s] = d < static_cast<int>(p.D) ? x : u32x4{0, 0, 0, 0};
        }
      }
    }
  }
  // Returns the mask of this lane's eight keys.
  __device__ __forceinline__ uint32_t load_v(uint32_t kb, const Places& at, uint32_t (&v)[8][kVec / 2]) const {
    uint32_t mask = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const Place pl = at.v[kPage8 ? 0 : j];
      const uint32_t row_in = kPage8 ? pl.row + j : pl.row;
      const bool ok = valid(kb + 8 * kq + j, pl.page);
      mask |= static_cast<uint32_t>(ok) << j;
      const char* row = ok ? vbase + pl.page * p.cache.v_page + row_in * p.cache.v_row : reinterpret_cast<const char*>(kZeroRow);
      const int d0 = kVec * (lane & 15);
      if constexpr (kVec == 4) {
        const u32x2 x = load_row<kOnce, u32x2>(row + 2 * (kExact ? d0 : min(d0, static_cast<int>(p.D) - 4)));
        const bool in = kExact || d0 < static_cast<int>(p.D);
        v[j][0] = in ? x[0] : 0;
        v[j][1] = in ? x[1] : 0;
      } else {
#pragma unroll
        for (int w = 0; w < kVec / 8; ++w) {
          const int d = d0 + 8 * w;
          const u32x4 x = load_row<kOnce, u32x4>(row + 2 * (kExact ? d : min(d, static_cast<int>(p.D) - 8)));
          const bool in = kExact || d < static_cast<int>(p.D);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[j][4 * w + e] = in ? x[e] : 0;
        }
      }
    }
    return mask;
  }

  __device__ __forceinline__ void run(uint32_t first, uint32_t last, const u32x4 (&q)[kMT][kK], Rows<kMT, kVec>& r) const {
    // Steps first, first + kTile, ... below last (a wave's share of the segment).
    if (first >= last) return;
    u32x4 k[2][kK];
    uint32_t v[8][kVec / 2];
    Places at = places(first);
    load_k(first, at, k);
    uint32_t mask = load_v(first, at, v);
    uint32_t next = first + kTile;
    if (next < last) at = places(next);
    for (uint32_t kb = first; kb < last; kb = next, next += kTile) {
      f32x4 s[kMT][2];
#pragma unroll
      for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
          s[mt][blk] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int st = 0; st < kK; ++st) s[mt][blk] = E::mfma16(k[blk][st], q[mt][st], s[mt][blk]);
        }
      if (next < last) load_k(next, at, k);
      u32x4 prob[kMT];
#pragma unroll
      for (int mt = 0; mt < kMT; ++mt) {
        float x[8], top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[j] = (mask >> j) & 1 ? s[mt][j >> 2][j & 3] * p.scale_log2 : -INFINITY;
          top = fmaxf(top, x[j]);
        }
        top = fmaxf(r.m[mt], op_over(top, 16, 64, OpMax{}));
        const float mm = finite_max(top), f = exp2_fast(r.m[mt] - mm), from = mm - E::kLift;
        r.m[mt] = top;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[j] = exp2_fast(x[j] - from);
          sum += x[j];
        }
        r.l[mt] = r.l[mt] * f + sum;
#pragma unroll
        for (int i = 0; i < kVec; ++i) r.acc[mt][i] *= f;
#pragma unroll
        for (int a = 0; a < 4; ++a) prob[mt][a] = pack2<E>(x[2 * a], x[2 * a + 1]);
      }
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const u32x4 vt = pair_rows<kVec>(v, i);
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt) r.acc[mt][i] = E::mfma16(vt, prob[mt], r.acc[mt][i]);
      }
      if (next < last) {
        mask = load_v(next, at, v);
        if (next + kTile < last) at = places(next + kTile);
      }
    }
  }
};

// The output of a row: sums x and l under the maximum m (times 2^kLift).
template <typename E>
__device__ __forceinline__ void finish(const DecodeParams& p, uint32_t b, uint32_t h, uint32_t c, const f32x4 (&x)[2], float m, float l) {
  const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
  u32x4 y;
#pragma unroll
  for (int a = 0; a < 4; ++a) y[a] = pack2<E>(x[a >> 1][2 * (a & 1)] * inv, x[a >> 1][2 * (a & 1) + 1] * inv);
  *reinterpret_cast<u32x4*>(p.out + b * p.o_token + h * p.o_head + 16 * c) = y;
  if (p.lse && c == 0) p.lse[static_cast<int64_t>(b) * p.Hq + h] = l == 0.f ? -INFINITY : (m - E::kLift + __log2f(l)) * kLn2;
}

template <typename S, bool kAfter>
__global__ void __launch_bounds__(kThreads, S::kPerSimd) decode_kernel(Params<S::kMore || kAfter> p) {
  using E = typename S::E;
  constexpr int kDP = S::kDP, kMT = S::kMT, kVec = kDP / 16, kK = kDP / 32, kPad = kDP + 4, kRound = S::kRound;
  constexpr bool kExact = S::kExact;
  __shared__ float ml[kWaves][kMT * 16][2];
  __shared__ float rows[kWaves][kRound * 16][kPad];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  const int n16 = lane & 15, kq = lane >> 4;

  // Zeros for query heads [h0, h1) of sequence b, which has no keys.
  auto write_zeros = [&](uint32_t b, uint32_t h0, uint32_t h1) {
    for (uint32_t i = threadIdx.x; i < (h1 - h0) * (p.D / 8); i += kThreads) {
      const uint32_t h = h0 + i / (p.D / 8), c = i % (p.D / 8);
      *reinterpret_cast<u32x4*>(p.out + b * p.o_token + h * p.o_head + 16 * c) = u32x4{0, 0, 0, 0};
      if (p.lse && c == 0) p.lse[static_cast<int64_t>(b) * p.Hq + h] = -INFINITY;
    }
  };
  uint32_t cur, last, per = 1, b, u, tile = 0, len, nt;
  if (p.whole) {
    b = blockIdx.x / p.U;
    u = blockIdx.x % p.U;
    len = length_of<kAfter>(p, b);
    nt = tiles_of(len);
    cur = 0;
    last = nt;
    if (kAfter && threadIdx.x == 0) p.unit_parts[blockIdx.x] = int2{0, len != 0};
    if (kAfter && len == 0) return;
    if (len == 0) {
      const uint32_t h0 = u / p.chunks * p.G + (u % p.chunks) * p.rows;
      write_zeros(b, h0, min(h0 + p.rows, (u / p.chunks + 1) * p.G));
      return;
    }
  } else {
    // Sequences without keys: units of no parts, rows of zeros.
    for (b = blockIdx.x; b < p.B; b += gridDim.x) {
      if (length_of<kAfter>(p, b) != 0) continue;
      if (!kAfter) write_zeros(b, 0, p.Hq);
      for (uint32_t i = threadIdx.x; i < p.U; i += kThreads) p.unit_parts[b * p.U + i] = int2{0, 0};
    }
    const Span span = find_span<kAfter>(p, lane);
    cur = span.begin;
    last = span.end;
    per = span.per;
    if (cur == last) return;
    b = span.b;
    len = length_of<kAfter>(p, b);
    nt = tiles_of(len);
    u = (cur - span.base * p.U) / nt;
    tile = (cur - span.base * p.U) % nt;
  }
  while (cur < last) {
    const uint32_t n = min(nt - tile, last - cur);
    const uint32_t hk = u / p.chunks, r0 = (u % p.chunks) * p.rows, nr = min(p.rows, p.G - r0);
    const S st(p, lane, kq, len, b, hk);
    u32x4 q[kMT][kK];
    Rows<kMT, kVec> r;
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt) {
      const uint32_t row = mt * 16 + n16;
      const char* src = p.q + b * p.q_token + (hk * p.G + r0 + min(row, nr - 1)) * p.q_head;
#pragma unroll
      for (int s = 0; s < kK; ++s) {
        const int d = S::q_dim(s, kq);
        const bool in = row < nr && (kExact || d < static_cast<int>(p.D));
        const u32x4 x = *reinterpret_cast<const u32x4*>(src + 2 * (kExact ? d : min(d, static_cast<int>(p.D) - 8)));
        q[mt][s] = in ? x : u32x4{0, 0, 0, 0};
      }
      r.m[mt] = -INFINITY;
      r.l[mt] = 0.f;
#pragma unroll
      for (int i = 0; i < kVec; ++i) r.acc[mt][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    st.run(tile * kTile + wave * kStep, min(len, (tile + n) * kTile), q, r);

    // The four waves' rows under one maximum.
    const bool whole = tile == 0 && n == nt;
    const uint32_t slot = tile == 0 ? 1 : 0;  // a workgroup's last unit may begin here, its first may end here
    const int64_t part = (static_cast<int64_t>(blockIdx.x) * 2 + slot) * p.rows;
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt) {
      r.l[mt] = op_over(r.l[mt], 16, 64, OpAdd{});
      if (kq == 0) {
        ml[wave][mt * 16 + n16][0] = r.m[mt];
        ml[wave][mt * 16 + n16][1] = r.l[mt];
      }
    }
    __syncthreads();
#pragma unroll
    for (int mt0 = 0; mt0 < kMT; mt0 += kRound) {
#pragma unroll
      for (int mm = 0; mm < kRound; ++mm) {
        const int mt = mt0 + mm;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) top = fmaxf(top, ml[w][mt * 16 + n16][0]);
        const float f = exp2_fast(r.m[mt] - finite_max(top));
#pragma unroll
        for (int rr = 0; rr < 4; ++rr)
#pragma unroll
          for (int i = 0; i < kVec; ++i) rows[wave][mm * 16 + n16][4 * kVec * kq + kVec * rr + i] = r.acc[mt][i][rr] * f;
      }
      __syncthreads();
      const uint32_t live = min(kRound * 16, max(0, static_cast<int>(nr) - mt0 * 16));
      for (uint32_t i = threadIdx.x; i < live * (p.D / 8); i += kThreads) {
        const uint32_t row = mt0 * 16 + i / (p.D / 8), c = i % (p.D / 8);
        float m = -INFINITY, l = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) m = fmaxf(m, ml[w][row][0]);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) l += ml[w][row][1] * exp2_fast(ml[w][row][0] - finite_max(m));
        f32x4 x[2] = {};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          x[0] += *reinterpret_cast<const f32x4*>(&rows[w][row - mt0 * 16][8 * c]);
          x[1] += *reinterpret_cast<const f32x4*>(&rows[w][row - mt0 * 16][8 * c + 4]);
        }
        if (!kAfter && whole) {
          finish<E>(p, b, hk * p.G + r0 + row, c, x, m, l);
        } else {
          const bool alone = kAfter && whole;
          const int64_t at = (alone ? (static_cast<int64_t>(b) * p.U + u) * p.rows : part) + row;
          float *acc = p.part_acc, *ml = p.part_ml;
          if constexpr (kAfter) acc = alone ? p.unit_acc : acc, ml = alone ? p.unit_ml : ml;
          f32x4* dst = reinterpret_cast<f32x4*>(acc + at * p.D + 8 * c);
          ml += 2 * at;
          dst[0] = x[0];
          dst[1] = x[1];
          if (c == 0) {
            ml[0] = m;
            ml[1] = l;
          }
        }
      }
      __syncthreads();
    }
    if (!p.whole && tile == 0 && threadIdx.x == 0)
      p.unit_parts[b * p.U + u] = int2{static_cast<int>(blockIdx.x), static_cast<int>((cur + nt - 1) / per - blockIdx.x + 1)};
    cur += n;
    tile = 0;
    if (++u == p.U && cur < last) {
      u = 0;
      do len = length_of<kAfter>(p, ++b);
      while (len == 0 && b + 1 < p.B);
      nt = tiles_of(len);
    }
  }
}

// Joins the parts of a unit: lane i of blockIdx.y holds eight elements of one row, each wave a share of the parts.
// A single pass under a running maximum, four parts in flight.
constexpr int kJoinWaves = 16;
template <typename E, bool kAfter>
__global__ void __launch_bounds__(kJoinWaves * kWave) join_kernel(Params<kAfter> p) {
  __shared__ float sm[kJoinWaves][10][kWave];
  const uint32_t unit = blockIdx.x, b = unit / p.U, u = unit % p.U;
  const int2 parts = p.unit_parts[unit];
  if (!kAfter && parts.y < 2) return;
  int count = parts.y;
  if constexpr (kAfter) count += p.prior.parts;
  const uint32_t hk = u / p.chunks, r0 = (u % p.chunks) * p.rows, nr = min(p.rows, p.G - r0);
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  // A part's pieces of one row are neighbours, the prior's those of neighbouring rows (kAfter).
  const uint32_t pieces = p.D / 8, item = blockIdx.y * kWave + lane, row_at = kAfter ? item % p.rows : item / pieces;
  const uint32_t row = min(row_at, nr - 1), c = kAfter ? min(item / p.rows, pieces - 1) : item % pieces;
  float m = -INFINITY, l = 0.f;
  f32x4 x[2] = {};
  const int waves = blockDim.x / kWave;
  // kAfter: the prior's parts of this row lie in the prompt kernels' layout: thread 64 wave + 32 half + row % 32 has dimensions 8 c + 4 half ..
  const uint32_t pr = b * p.G + r0 + row, tile = pr / 128, thread = pr % 128 / 32 * 64 + pr % 32, Hkv = p.Hq / p.G, width = p.D <= 64 ? 64 : p.D <= 128 ? 128 : 256;
  int64_t pfirst = 0, pstep = 0;
  if constexpr (kAfter) {
    pfirst = static_cast<int64_t>(p.prior.tiles - 1 - static_cast<int>(tile)) * Hkv + hk;
    pstep = static_cast<int64_t>(p.prior.tiles) * Hkv;
  }
  for (int i0 = wave; i0 < count; i0 += 4 * waves) {
    float pm[4], pl[4];
    f32x4 px[4][2];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = min(i0 + j * waves, count - 1);
      auto own = [&](const float* part_ml, const float* part_acc, int64_t part) {
        const int64_t at = part * p.rows + row;
        const f32x4* src = reinterpret_cast<const f32x4*>(part_acc + at * p.D + 8 * c);
        pm[j] = part_ml[2 * at];
        pl[j] = part_ml[2 * at + 1];
        px[j][0] = src[0];
        px[j][1] = src[1];
      };
      const int64_t part = static_cast<int64_t>(parts.x + i) * 2 + (i == 0 ? 1 : 0);
      if constexpr (kAfter) {
        if (i >= parts.y) {
          const int64_t at = pfirst + (i - parts.y) * pstep;
          const f32x4 ml = reinterpret_cast<const f32x4*>(p.prior.ml)[at * 256 + thread];
          const f32x4* src = reinterpret_cast<const f32x4*>(p.prior.acc) + at * (width / 8 * 256) + c * 256 + thread;
          // Its rows are to be divided by the sum of the rounded weights, the second of ml, and count with the full one.
          const float by = ml[1] > 0.f ? ml[2] / ml[1] : ml[1] == 0.f ? 0.f : ml[1];
          pm[j] = ml[0] - p.prior.up + E::kLift;
          pl[j] = ml[2];
          px[j][0] = src[0] * by;
          px[j][1] = src[32] * by;
        } else if (parts.y == 1) {
          own(p.unit_ml, p.unit_acc, unit);
        } else {
          own(p.part_ml, p.part_acc, part);
        }
      } else {
        own(p.part_ml, p.part_acc, part);
      }
      if (i0 + j * waves >= count) {
        pm[j] = -INFINITY;
        pl[j] = 0.f;
      }
    }
    // All loads are under way before the first is looked at: left alone, the first part's rows are fetched once its maximum is there, a second
    // latency (those 96 sequences 17.3 us).
    if constexpr (!kAfter) {
#pragma unroll
      for (int j = 0; j < 4; ++j) asm volatile("" : "+v"(px[j][0]), "+v"(px[j][1]));
    }
    const float top = fmaxf(fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3])), m), mm = finite_max(top), f = exp2_fast(m - mm);
    m = top;
    l *= f;
    x[0] *= f;
    x[1] *= f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float w = exp2_fast(pm[j] - mm);
      if (pm[j] == -INFINITY && pl[j] == pl[j]) continue;  // no keys (a repeated last part among them), and no NaN to pass on
      l += w * pl[j];
      x[0] += px[j][0] * w;
      x[1] += px[j][1] * w;
    }
  }
  sm[wave][0][lane] = m;
  sm[wave][1][lane] = l;
#pragma unroll
  for (int e = 0; e < 8; ++e) sm[wave][2 + e][lane] = x[e >> 2][e & 3];
  __syncthreads();
  if (wave != 0 || item >= p.rows * pieces || row_at >= nr) return;
  float y[8] = {};
  m = -INFINITY;
  for (int w = 0; w < waves; ++w) m = fmaxf(m, sm[w][0][lane]);
  l = 0.f;
  for (int w = 0; w < waves; ++w) {
    const float f = exp2_fast(sm[w][0][lane] - finite_max(m));
    l += f * sm[w][1][lane];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] += f * sm[w][2 + e][lane];
  }
  const f32x4 sums[2] = {{y[0], y[1], y[2], y[3]}, {y[4], y[5], y[6], y[7]}};
  finish<E>(p, b, hk * p.G + r0 + row, c, sums, m, l);
}

struct Plan {
  int mt;
  uint32_t chunks, rows, U, groups;
  bool whole, once;
  size_t ml_bytes, acc_bytes, unit_bytes;
};

// Up to kWholeTiles tiles of the longest sequence a page table holds each unit is one workgroup's: the parts and the second
// launch cost more than the tiles one after the other (301 tokens: 13.6 us in parts, 8.7 whole).  Twice as many where
// the units alone fill the chip (32 sequences of up to 1000 tokens, 8 heads: 22.9 and 21.1 us; 12 sequences 13.4 and 20.0).
constexpr int64_t kWholeTiles = 4, kManyWholeTiles = 8;
// A call that may read more than this finds nothing of it in the last-level cache (256 MB) at the next step, and its loads leave
// what others keep there alone (131071 tokens, 537 MB: 113 -> 103 us; 3.8 GB: 684 -> 658; 32 MB would go from 18.0 to 19.6).
constexpr int64_t kOnceBytes = 256 << 20;
constexpr int64_t kMaxUnits = 1 << 22;  // workgroups of a launch

// size: bytes of a cache element; most: workgroups of a launch.
Plan plan_for(const latent_attn_decode_args& a, int64_t size = 2, uint32_t most = kMaxGroups) {
  Plan pl{};
  const uint32_t G = static_cast<uint32_t>(a.n_head / a.n_kv_head);
  pl.mt = G > 16 ? 2 : 1;
  pl.chunks = (G + 16 * pl.mt - 1) / (16 * pl.mt);
  pl.rows = std::min<uint32_t>(G, 16 * pl.mt);
  pl.U = static_cast<uint32_t>(a.n_kv_head) * pl.chunks;
  const int64_t tiles = (a.cache.max_pages * a.cache.page_size + kTile - 1) / kTile;
  const int64_t items = a.cache.n_seq * pl.U * tiles;
  const int64_t units = a.cache.n_seq * pl.U;
  const int64_t row = 2 * size * a.n_kv_head * a.head_dim;  // bytes of a position
  pl.once = std::min(a.cache.n_seq * a.cache.max_pages, a.cache.n_pages) > kOnceBytes / (row * a.cache.page_size);
  pl.whole = tiles <= kWholeTiles || (tiles <= kManyWholeTiles && units >= 256 && units <= 1024);
  if (pl.whole) {
    pl.groups = static_cast<uint32_t>(units);
    return pl;
  }
  pl.groups = static_cast<uint32_t>(std::min<int64_t>(items, most));
  const size_t parts = static_cast<size_t>(pl.groups) * 2 * pl.rows;
  auto up = [](size_t n) { return (n + 15) & ~size_t{15}; };
  pl.ml_bytes = up(parts * 2 * sizeof(float));
  pl.acc_bytes = up(parts * a.head_dim * sizeof(float));
  pl.unit_bytes = up(static_cast<size_t>(a.cache.n_seq) * pl.U * sizeof(int2));
  return pl;
}

int validate(const latent_attn_decode_args& a) {
  const int st = check_heads(a.n_head, a.n_kv_head, a.head_dim, a.dtype);
  if (st != LATENT_OK) return st;
  if (a.n_head == 0 || !(a.scale > 0.f) || !(a.scale < INFINITY)) return LATENT_E_INVALID;
  const int sc = check_cache(a.cache);
  if (sc != LATENT_OK) return sc;
  // Tiles and output rows are counted in 32 bits.
  const Plan pl = plan_for(a);
  if (a.cache.n_seq * pl.U > kMaxUnits) return LATENT_E_UNSUPPORTED;
  const int64_t tiles = (a.cache.max_pages * a.cache.page_size + kTile - 1) / kTile;
  if (a.cache.n_seq * pl.U > INT32_MAX / std::max<int64_t>(1, tiles) - kMaxGroups) return LATENT_E_UNSUPPORTED;
  return LATENT_OK;
}


// The checks of a call and its parameters.  size: bytes of a cache element; 1: what the call does is done (no sequences).
int decode_params(const latent_attn_decode_args& a, int64_t size, const Plan& pl, DecodeParams* out) {
  if (!a.q || !a.out || !a.lengths) return LATENT_E_INVALID;
  const bool keys = a.cache.max_pages > 0 && a.cache.n_pages > 0;
  if (keys && (!a.cache.k || !a.cache.v || !a.cache.pages)) return LATENT_E_INVALID;
  if (!aligned16(a.q) || !aligned16(a.out) || !aligned16(a.workspace)) return LATENT_E_UNSUPPORTED;
  for (int64_t s : {a.q_token_stride, a.q_head_stride, a.out_token_stride, a.out_head_stride})
    if (!stride_ok(s)) return LATENT_E_UNSUPPORTED;
  if ((a.n_head > 1 && !a.out_head_stride) || (a.cache.n_seq > 1 && !a.out_token_stride)) return LATENT_E_INVALID;
  if (!pl.whole && (!a.workspace || a.workspace_bytes < pl.ml_bytes + pl.acc_bytes + pl.unit_bytes)) return LATENT_E_WORKSPACE;
  DecodeParams& p = *out;
  p.cache = device_cache(a.cache, size);
  if (!keys) p.cache.max_len = 0;
  p.q = static_cast<const char*>(a.q);
  p.out = static_cast<char*>(a.out);
  p.lse = a.lse;
  p.lengths = a.lengths;
  p.q_token = a.q_token_stride * 2, p.q_head = a.q_head_stride * 2;
  p.o_token = a.out_token_stride * 2, p.o_head = a.out_head_stride * 2;
  p.B = static_cast<uint32_t>(a.cache.n_seq);
  p.Hq = static_cast<uint32_t>(a.n_head);
  p.G = static_cast<uint32_t>(a.n_head / a.n_kv_head);
  p.D = static_cast<uint32_t>(a.head_dim);
  p.chunks = pl.chunks;
  p.rows = pl.rows;
  p.U = pl.U;
  p.whole = pl.whole;
  p.scale_log2 = a.scale * kLog2e;
  char* ws = static_cast<char*>(a.workspace);
  p.part_ml = reinterpret_cast<float*>(ws);
  p.part_acc = reinterpret_cast<float*>(ws + pl.ml_bytes);
  p.unit_parts = reinterpret_cast<int2*>(ws + pl.ml_bytes + pl.acc_bytes);
  return LATENT_OK;
}

// The second launch, where units were left in parts.
template <bool kAfter>
void launch_join(const Plan& pl, const Params<kAfter>& p, bool f16, hipStream_t s) {
  if (pl.whole && !kAfter) return;
  // A unit has about groups / units parts, four in flight a wave.  Of few parts two waves join soonest (96 units of six:
  // 16.8 us the whole call, 17.1 with one or four), of hundreds sixteen (one unit of 235: 16.6, 23.1 with four).
  const uint32_t units = p.B * p.U;
  uint32_t waves = pl.groups > 16 * units ? kJoinWaves : pl.groups > 8 * units ? 4 : 2;
  // The prior's parts are as many for each unit (5 sequences, 16 parts, 40 units: 5.1 us by eight waves, 7.2 by four; 512 units 12.0 and 10.0).
  if constexpr (kAfter) {
    if (p.prior.parts > 8) waves = std::max<uint32_t>(waves, units <= 256 ? 8 : 4);
  }
  const dim3 grid(units, (p.rows * (p.D / 8) + kWave - 1) / kWave), block(kWave * waves);
  if (f16)
    hipLaunchKernelGGL((join_kernel<F16, kAfter>), grid, block, 0, s, p);
  else
    hipLaunchKernelGGL((join_kernel<BF16, kAfter>), grid, block, 0, s, p);
}

// The same call over the positions behind a shared prefix of n_prefix pages.
latent_attn_decode_args behind(const latent_attn_decode_args& a, int64_t n_prefix) {
  latent_attn_decode_args r = a;
  r.cache.max_pages -= n_prefix;
  if (r.cache.pages) r.cache.pages += n_prefix;
  return r;
}
// The workspace behind a shared prefix: a decode's, every unit's parts among it, and the rows of units that one workgroup has whole.
struct After {
  Plan plan;
  size_t unit_bytes, ml_bytes, acc_bytes;
  size_t all() const { return plan.ml_bytes + plan.acc_bytes + unit_bytes + ml_bytes + acc_bytes; }
};
After plan_after(const latent_attn_decode_args& own, int64_t size, uint32_t most) {
  After r{plan_for(own, size, most), 0, 0, 0};
  auto up = [](size_t n) { return (n + 15) & ~size_t{15}; };
  const size_t units = static_cast<size_t>(own.cache.n_seq) * r.plan.U, rows = units * r.plan.rows;
  r.unit_bytes = up(units * sizeof(int2));
  r.ml_bytes = up(rows * 2 * sizeof(float));
  r.acc_bytes = rows * own.head_dim * sizeof(float);
  return r;
}
int after_params(const latent_attn_decode_args& a, int64_t n_prefix, int64_t size, const After& w, const Prior& prior, void* workspace, MoreParams* p) {
  latent_attn_decode_args own = behind(a, n_prefix);
  own.workspace = workspace;
  own.workspace_bytes = SIZE_MAX;
  const int st = decode_params(own, size, w.plan, p);
  char* more = static_cast<char*>(workspace) + w.plan.ml_bytes + w.plan.acc_bytes;
  p->unit_parts = reinterpret_cast<int2*>(more);
  p->unit_ml = reinterpret_cast<float*>(more + w.unit_bytes);
  p->unit_acc = reinterpret_cast<float*>(more + w.unit_bytes + w.ml_bytes);
  p->prior = prior;
  p->ahead = static_cast<uint32_t>(n_prefix * a.cache.page_size);
  return st;
}

}  // namespace
}  // namespace attend
}  // namespace latent
