// The 8-bit cache's stream of keys for the decode kernels.
//
//   score[j] = scale ks[j] (q . kcode[j]),   out = sum_j (p[j] vs[j]) vcode[j] / sum_j p[j]
//
// Codes become exact elements of the queries' type in registers, four of a dword in two instructions (e4m3; whole numbers take
// three for bf16's pairs, as they have no conversion of their own), so that a row costs its D bytes and a scale, and products are the 16-bit ones.
// A lane quarter holds a quarter of a key's dimensions, which is as good an order of the sum as any as long as the queries
// have it too, and is 16 adjacent bytes a load.  Values arrive as VEC bytes a lane for eight keys; four keys' dwords are
// transposed by byte permutes, after which a key pair's codes are neighbours.
//
// A probability times its value's scale has a full significand where the largest probability alone is one: rounded once it would
// put its half step on a row that one key makes.  Its rounding's remainder, rounded too, is a second operand: the matrix units, idle
// nine tenths of the time here, take both (one key of bf16: off by 0.0029 of the row's size without, 0.0017, the output's rounding, with).
//
// Measured (heads of 128, 32 over 8 unless said): 301 tokens 8.0 us, 35 sequences of 16 to 16000 (228 MB) 66 us, 64 of 8000 214 us over e4m3 and
// 217 over int8 (362 over a 16-bit cache), 64 of 10000 to 20000, 64 heads, f16 over int8, 392 us (5.0 TB/s).  Bound by HBM, behind 15 to 20 us of
// launch, prologue and join; rows of a head that are together in a page, instead of all heads' of a position, go at 5.6 TB/s.
#pragma once

#include "decode.hpp"

namespace latent {
namespace attend {
namespace {

// Bytes i of four dwords, as dword i.
__device__ __forceinline__ void transpose4(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t (&t)[4]) {
  const uint32_t ab0 = __builtin_amdgcn_perm(b, a, 0x05010400u), ab1 = __builtin_amdgcn_perm(b, a, 0x07030602u);
  const uint32_t cd0 = __builtin_amdgcn_perm(d, c, 0x05010400u), cd1 = __builtin_amdgcn_perm(d, c, 0x07030602u);
  t[0] = __builtin_amdgcn_perm(cd0, ab0, 0x05040100u);
  t[1] = __builtin_amdgcn_perm(cd0, ab0, 0x07060302u);
  t[2] = __builtin_amdgcn_perm(cd1, ab1, 0x05040100u);
  t[3] = __builtin_amdgcn_perm(cd1, ab1, 0x07060302u);
}

template <typename E_, typename Q, int kDP_, int kMT_, bool kOnce, bool kTable>
struct Stream8 {
  typedef E_ E;
  static constexpr int kDP = kDP_, kMT = kMT_, kVec = kDP / 16, kK = kDP / 32, kKLoads = kDP / 64, kVWords = kVec / 4;
  static constexpr bool kExact = false;
  static constexpr int kRound = kDP <= 128 ? kMT : 1;
  static constexpr int kPerSimd = kDP == 256 ? 1 : 2;
  static constexpr bool kMore = true;
  static __device__ __forceinline__ int q_dim(int s, int kq) { return kDP / 4 * kq + 8 * s; }

  const MoreParams& p;
  int lane, kq;
  uint32_t len;
  const int32_t* pages;
  uint64_t kbase, vbase, kscale, vscale;
  __device__ __forceinline__ Stream8(const MoreParams& p, int lane, int kq, uint32_t len, uint32_t b, uint32_t hk)
      : p(p), lane(lane), kq(kq), len(len), pages(p.cache.pages + b * p.cache.pages_stride),
        kbase(reinterpret_cast<uint64_t>(p.cache.k + hk * p.cache.k_head)), vbase(reinterpret_cast<uint64_t>(p.cache.v + hk * p.cache.v_head)),
        kscale(reinterpret_cast<uint64_t>(p.scales.k + hk * p.scales.k_head)), vscale(reinterpret_cast<uint64_t>(p.scales.v + hk * p.scales.v_head)) {}

  // Eight neighbours from a multiple of eight share a page: those that this lane reads keys of, and those that it holds scores of.
  struct Place {
    int32_t page;  // outside [0, n_pages): masked
    uint32_t row;
  };
  struct Places {
    Place k, v;
  };
  __device__ __forceinline__ Place place_of(uint32_t key) const {
    const uint32_t slot = p.cache.by_page.of(key);
    return {key < len ? (kTable && slot < p.prefix_pages ? p.prefix : pages)[slot] : -1, key - slot * p.cache.page_size};
  }
  __device__ __forceinline__ Places places(uint32_t kb) const { return {place_of(kb + 8 * ((lane & 15) >> 2)), place_of(kb + 8 * kq)}; }
  __device__ __forceinline__ bool there(const Place& at) const { return static_cast<uint32_t>(at.page) < p.cache.n_pages; }

  // What a step reads.  Rows behind the last are read as zeros, scales of a part of eight as they stand there: their keys are masked.
  struct Buffer {
    u32x4 k[2][kKLoads];
    uint32_t v[8][kVWords];
    f32x4 kscale[2], vscale[2];
    Places at;      // of the step that is loaded next
    uint32_t mask;  // the keys of this lane that exist
  };
  template <typename T>
  static __device__ __forceinline__ T load(uint64_t at) {  // global, which a pointer that may be the zeros' would not be seen to be
    return *reinterpret_cast<const __attribute__((address_space(1))) T*>(at);
  }
  template <typename T>
  static __device__ __forceinline__ T load_code(uint64_t at) {
    if constexpr (kOnce) return __builtin_nontemporal_load(reinterpret_cast<const __attribute__((address_space(1))) T*>(at));
    return load<T>(at);
  }
  // Whether all keys of a step exist: then none of its addresses and scores needs a look.
  __device__ __forceinline__ bool whole(uint32_t kb, const Places& at) const { return kb + kStep <= len && __all(there(at.k) && there(at.v)); }

  __device__ __forceinline__ void load_k(uint32_t kb, bool all, Buffer& b) const {
    const uint32_t r = b.at.k.row + (lane & 3);
    uint64_t row[2];
    row[0] = kbase + b.at.k.page * p.cache.k_page + r * p.cache.k_row;
    row[1] = row[0] + 4 * p.cache.k_row;
    uint64_t s = kscale + b.at.v.page * p.scales.k_page + 4 * b.at.v.row;
    if (!all) {
      // Row m of score block blk is key 8 (m / 4) + 4 blk + m % 4 of the step: lane (query, kq) then holds keys 8 kq .. + 7.
      const uint32_t key = kb + 8 * ((lane & 15) >> 2) + (lane & 3);
      const uint64_t zero = reinterpret_cast<uint64_t>(kZeroRow);
      row[0] = key < len && there(b.at.k) ? row[0] : zero;
      row[1] = key + 4 < len && there(b.at.k) ? row[1] : zero;
      s = there(b.at.v) ? s : zero;
    }
#pragma unroll
    for (int blk = 0; blk < 2; ++blk)
#pragma unroll
      for (int i = 0; i < kKLoads; ++i) b.k[blk][i] = load_code<u32x4>(row[blk] + min(kDP / 4 * kq + 16 * i, static_cast<int>(p.D) - 16));
    b.kscale[0] = load<f32x4>(s);
    b.kscale[1] = load<f32x4>(s + 16);
  }
  __device__ __forceinline__ void load_v(uint32_t kb, bool all, Buffer& b) const {
    const uint64_t first = vbase + b.at.v.page * p.cache.v_page + b.at.v.row * p.cache.v_row + min(kVec * (lane & 15), static_cast<int>(p.D) - kVec);
    uint64_t s = vscale + b.at.v.page * p.scales.v_page + 4 * b.at.v.row;
    const uint64_t zero = reinterpret_cast<uint64_t>(kZeroRow);
    uint64_t row[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) row[j] = first + j * p.cache.v_row;
    b.mask = 0xFFu;
    if (!all) {
      s = there(b.at.v) ? s : zero;
      b.mask = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool ok = kb + 8 * kq + j < len && there(b.at.v);
        b.mask |= static_cast<uint32_t>(ok) << j;
        row[j] = ok ? row[j] : zero;
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (kVWords == 1) {
        b.v[j][0] = load_code<uint32_t>(row[j]);
      } else if constexpr (kVWords == 2) {
        const u32x2 x = load_code<u32x2>(row[j]);
        b.v[j][0] = x[0];
        b.v[j][1] = x[1];
      } else {
        const u32x4 x = load_code<u32x4>(row[j]);
#pragma unroll
        for (int w = 0; w < 4; ++w) b.v[j][w] = x[w];
      }
    }
    b.vscale[0] = load<f32x4>(s);
    b.vscale[1] = load<f32x4>(s + 16);
  }

  // The step in buffer b, and into it, as its parts fall free, the next one.
  // f16 holds a probability times its value's scale against a power of two (its bits in `base`) below the largest scale so far: like the
  // probabilities (kLift, one less for the factor below two) they then come near the type's largest, whatever the values' size.
  static constexpr bool kLifted = E::kLift != 0.f;
  __device__ __forceinline__ void step(Buffer& b, uint32_t next, uint32_t last, const u32x4 (&q)[kMT][kK], Rows<kMT, kVec>& r, uint32_t& base) const {
    f32x4 s[kMT][2];
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) s[mt][blk] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int st = 0; st < kK; ++st)
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) {
        const uint32_t w0 = b.k[blk][st / 2][2 * (st & 1)], w1 = b.k[blk][st / 2][2 * (st & 1) + 1];
        const u32x4 x{Q::template pair<E, false>(w0), Q::template pair<E, true>(w0), Q::template pair<E, false>(w1), Q::template pair<E, true>(w1)};
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt) s[mt][blk] = E::mfma16(x, q[mt][st], s[mt][blk]);
      }
    float ks[8], vs[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      ks[j] = b.kscale[j >> 2][j & 3] * p.scale_log2;
      vs[j] = b.vscale[j >> 2][j & 3];
    }
    const bool more = next < last;
    const bool all_next = more && whole(next, b.at);
    if (more) load_k(next, all_next, b);
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
      for (int j = 0; j < 8; ++j) s[mt][j >> 2][j & 3] *= ks[j];
    if (__any(b.mask != 0xFFu)) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool ok = b.mask >> j & 1;
        vs[j] = ok ? vs[j] : 0.f;
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt) s[mt][j >> 2][j & 3] = ok ? s[mt][j >> 2][j & 3] : -INFINITY;
      }
    }
    float rebase = 1.f;
    if constexpr (kLifted) {
      float most = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) most = fmaxf(most, vs[j]);
      if (__any(!held<E, Q>(most))) {
        most = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          vs[j] = held<E, Q>(vs[j]) ? vs[j] : __uint_as_float(0x7FC00000u);
          most = fmaxf(most, vs[j]);
        }
      }
      const uint32_t up = max(base, __float_as_uint(op_over(most, 16, 64, OpMax{})) & 0x7F800000u);
      const float inv = __uint_as_float(0x7E800000u - up);  // half over the power: 2^k has the exponent bits 127 + k, 253 less those are 2^(-1 - k)'s
      rebase = __uint_as_float(0x3F800000u + base - up);
      base = up;
#pragma unroll
      for (int j = 0; j < 8; ++j) vs[j] *= inv;
    }
    u32x4 prob[kMT], rest[kMT];
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt) {
      float x[8], top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 8; ++j) top = fmaxf(top, s[mt][j >> 2][j & 3]);
      top = fmaxf(r.m[mt], op_over(top, 16, 64, OpMax{}));
      const float mm = finite_max(top), f = exp2_fast(r.m[mt] - mm), from = mm - E::kLift;
      r.m[mt] = top;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] = exp2_fast(s[mt][j >> 2][j & 3] - from);
        sum += x[j];
        x[j] *= vs[j];
      }
      r.l[mt] = r.l[mt] * f + sum;
      const float fa = f * rebase;
      if (__any(fa != 1.f)) {  // the largest scores come early: most steps change neither
#pragma unroll
        for (int i = 0; i < kVec; ++i) r.acc[mt][i] *= fa;
      }
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        prob[mt][a] = pack2<E>(x[2 * a], x[2 * a + 1]);
        rest[mt][a] = pack2<E>(x[2 * a] - unpack_lo<E>(prob[mt][a]), x[2 * a + 1] - unpack_hi<E>(prob[mt][a]));
      }
    }
#pragma unroll
    for (int w = 0; w < kVWords; ++w) {
      uint32_t lo[4], hi[4];
      transpose4(b.v[0][w], b.v[1][w], b.v[2][w], b.v[3][w], lo);
      transpose4(b.v[4][w], b.v[5][w], b.v[6][w], b.v[7][w], hi);
      u32x4 x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = u32x4{Q::template pair<E, false>(lo[i]), Q::template pair<E, true>(lo[i]), Q::template pair<E, false>(hi[i]), Q::template pair<E, true>(hi[i])};
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt) r.acc[mt][4 * w + i] = E::mfma16(x[i], prob[mt], r.acc[mt][4 * w + i]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt) r.acc[mt][4 * w + i] = E::mfma16(x[i], rest[mt], r.acc[mt][4 * w + i]);
    }
    if (more) {
      load_v(next, all_next, b);
      if (next + kTile < last) b.at = places(next + kTile);
    }
  }

  __device__ __forceinline__ void run(uint32_t first, uint32_t last, const u32x4 (&q)[kMT][kK], Rows<kMT, kVec>& r) const {
    if (first >= last) return;
    uint32_t base = 0x2B800000u;  // 2^-40, below which a value is nothing to f16; bf16 has fp32's range and no need
    Buffer b;
    b.at = places(first);
    const bool all = whole(first, b.at);
    load_k(first, all, b);
    load_v(first, all, b);
    if (first + kTile < last) b.at = places(first + kTile);
    for (uint32_t kb = first; kb < last; kb += kTile) step(b, kb + kTile, last, q, r, base);
    if constexpr (kLifted) {  // back from what `inv` took
      const float f = __uint_as_float(base) * 2.f;
#pragma unroll
      for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
        for (int i = 0; i < kVec; ++i) r.acc[mt][i] *= f;
    }
  }
};

// f(S{}) with the stream type of a call: the only variants are the types, the rows' padded width, the products' columns, and whether
// the rows pass the last-level cache by.
template <typename T>
struct Type {
  typedef T type;
};
template <bool kTable, typename F>
void with_stream8(const latent_attn_decode_args& a, int32_t code, const Plan& pl, F f) {
  using std::integral_constant;
  auto once = [&](auto e, auto q, auto dp, auto mt) {
    constexpr int kDP = decltype(dp)::value, kMT = decltype(mt)::value;
    pl.once ? f(Type<Stream8<decltype(e), decltype(q), kDP, kMT, true, kTable>>{}) : f(Type<Stream8<decltype(e), decltype(q), kDP, kMT, false, kTable>>{});
  };
  auto rows = [&](auto e, auto q, auto dp) { pl.mt == 1 ? once(e, q, dp, integral_constant<int, 1>{}) : once(e, q, dp, integral_constant<int, 2>{}); };
  auto dims = [&](auto e, auto q) {
    a.head_dim <= 64    ? rows(e, q, integral_constant<int, 64>{})
    : a.head_dim <= 128 ? rows(e, q, integral_constant<int, 128>{})
                        : rows(e, q, integral_constant<int, 256>{});
  };
  auto codes = [&](auto e) { code == LATENT_CODE_INT8 ? dims(e, Int8{}) : dims(e, E4M3{}); };
  a.dtype == LATENT_F16 ? codes(F16{}) : codes(BF16{});
}

}  // namespace
}  // namespace attend
}  // namespace latent
