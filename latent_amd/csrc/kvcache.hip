// Appending a step's keys and values to the paged cache, rotated on the way.
//
//   (a, b) -> (a c - b s, b c + a s),  c, s = rope[position][0 / 1][pair]
//
// for the pairs of a head's leading rot_dim dimensions, of k and (into q_out) of
// q; v and the rest are copied.  Products and sums are fp32, each element is
// rounded once.
//
// Bound by memory: a token's (n_head + 2 n_kv_head) D elements are read and
// written once.  A thread moves 2 x 16 bytes of a head (the two halves of eight
// pairs, or 16 neighbours) and goes on to the next heads of its token with the
// same 16 table values: read again for each head they would be twice the bytes
// of the data itself.  Measured: 8190 tokens of 80 heads of 128 bf16 68 us (5.0 TB/s,
// a copy's rate); one token 2.9 us of GPU, 5.1 a call.  Heads or rotations that are no multiples of 16 take a kernel of one pair a
// thread in accesses of two bytes (8192 tokens of 48 heads: rotation of 20 of 128 dimensions 191 us, of 128 41; heads of 72 62,
// of 80 31): one step's tokens cost a launch either way (32 tokens of heads of 72: 4.6 us).
#include "attend.hpp"

#include <algorithm>

namespace latent {
namespace attend {
namespace {

constexpr int kThreads = 256;

struct AppendParams {
  Cache cache;  // k, v written
  const char* q;
  char* q_out;
  const char* k;
  const char* v;
  int64_t q_token, q_head, qo_token, qo_head, k_token, k_head, v_token, v_head;  // bytes
  const int32_t* positions;
  const int32_t* seqs;
  const float* rope;
  uint32_t rope_rows;  // positions below it are in the table (any, without a table)
  uint32_t n_seq, T, Hq, Hkv, D, rot;
  uint32_t units;   // work items of a head
  uint32_t groups;  // head groups of a token
};

enum Kind { kHalf, kInterleaved, kScalar };

// Page of a token and the row in it, or false.
__device__ __forceinline__ bool find_row(const Cache& cache, const int32_t* seqs, uint32_t n_seq, uint32_t t, uint32_t pos, uint32_t* page,
                                         uint32_t* off) {
  const uint32_t seq = seqs ? static_cast<uint32_t>(seqs[t]) : t;
  if (seq >= n_seq || pos >= cache.max_len) return false;
  const uint32_t slot = cache.by_page.of(pos);
  *off = pos - slot * cache.page_size;
  *page = static_cast<uint32_t>(cache.pages[seq * cache.pages_stride + slot]);
  return *page < cache.n_pages;
}
// Cache row of a token (byte offsets of head 0), or false.
__device__ __forceinline__ bool cache_row(const AppendParams& p, uint32_t t, uint32_t pos, int64_t* k, int64_t* v) {
  uint32_t page, off;
  if (!find_row(p.cache, p.seqs, p.n_seq, t, pos, &page, &off)) return false;
  *k = page * p.cache.k_page + off * p.cache.k_row;
  *v = page * p.cache.v_page + off * p.cache.v_row;
  return true;
}

// Where head h of token t is read and written; h counts q, then k, then v heads.
__device__ __forceinline__ bool head_rows(const AppendParams& p, uint32_t t, uint32_t h, bool stored, int64_t krow,
                                          int64_t vrow, const char** src, char** dst) {
  if (h < p.Hq) {
    *src = p.q + t * p.q_token + h * p.q_head;
    *dst = p.q_out + t * p.qo_token + h * p.qo_head;
    return true;
  }
  h -= p.Hq;
  if (h < p.Hkv) {
    *src = p.k + t * p.k_token + h * p.k_head;
    *dst = const_cast<char*>(p.cache.k) + krow + h * p.cache.k_head;
  } else {
    h -= p.Hkv;
    *src = p.v + t * p.v_token + h * p.v_head;
    *dst = const_cast<char*>(p.cache.v) + vrow + h * p.cache.v_head;
  }
  return stored;
}

template <typename E>
__device__ __forceinline__ void rotate8(u32x4& a, u32x4& b, const f32x4 c[2], const f32x4 s[2]) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float a0 = unpack_lo<E>(a[w]), a1 = unpack_hi<E>(a[w]), b0 = unpack_lo<E>(b[w]), b1 = unpack_hi<E>(b[w]);
    const float c0 = c[w >> 1][2 * (w & 1)], c1 = c[w >> 1][2 * (w & 1) + 1];
    const float s0 = s[w >> 1][2 * (w & 1)], s1 = s[w >> 1][2 * (w & 1) + 1];
    a[w] = pack2<E>(a0 * c0 - b0 * s0, a1 * c1 - b1 * s1);
    b[w] = pack2<E>(b0 * c0 + a0 * s0, b1 * c1 + a1 * s1);
  }
}

template <typename E>
__device__ __forceinline__ void rotate8_neighbours(u32x4& x, const f32x4& c, const f32x4& s) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float a = unpack_lo<E>(x[w]), b = unpack_hi<E>(x[w]);
    x[w] = pack2<E>(a * c[w] - b * s[w], b * c[w] + a * s[w]);
  }
}

// kHeads heads of one token, 16 elements of each: units 0 .. rot / 16 - 1 hold
// rotated pairs, the others (and v) are copied.
template <typename E, int kKind, int kHeads>
__global__ void __launch_bounds__(kThreads) append_kernel(AppendParams p) {
  const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t t = i / (p.units * p.groups);
  if (t >= p.T) return;
  const uint32_t g = i / p.units % p.groups, u = i % p.units;
  const uint32_t pos = static_cast<uint32_t>(p.positions[t]);
  if (pos >= p.rope_rows) return;
  const uint32_t h0 = g * kHeads, H = p.Hq + 2 * p.Hkv;
  int64_t krow = 0, vrow = 0;
  const bool stored = h0 + kHeads > p.Hq && cache_row(p, t, pos, &krow, &vrow);
  const bool turned = u < p.rot / 16;
  // Byte offsets of the unit's two 16-byte pieces in a head.
  const uint32_t a0 = kKind == kHalf && turned ? 16 * u : 32 * u;
  const uint32_t b0 = kKind == kHalf && turned ? p.rot + 16 * u : 32 * u + 16;
  f32x4 c[2], s[2];
  if (turned) {
    const f32x4* row = reinterpret_cast<const f32x4*>(p.rope + static_cast<int64_t>(pos) * p.rot);
    c[0] = row[2 * u], c[1] = row[2 * u + 1];
    s[0] = row[p.rot / 8 + 2 * u], s[1] = row[p.rot / 8 + 2 * u + 1];
  }
  const char* src[kHeads];
  char* dst[kHeads];
  bool live[kHeads];
  u32x4 a[kHeads], b[kHeads];
#pragma unroll
  for (int j = 0; j < kHeads; ++j) {
    live[j] = h0 + j < H && head_rows(p, t, h0 + j, stored, krow, vrow, &src[j], &dst[j]);
    if (live[j]) {
      a[j] = *reinterpret_cast<const u32x4*>(src[j] + a0);
      b[j] = *reinterpret_cast<const u32x4*>(src[j] + b0);
    }
  }
#pragma unroll
  for (int j = 0; j < kHeads; ++j) {
    if (!live[j]) continue;
    u32x4 x = a[j], y = b[j];
    // v heads' units are copied at the offsets of a rotated unit: all units of a head cover it either way.
    if (turned && h0 + j < p.Hq + p.Hkv) {
      if constexpr (kKind == kHalf) {
        rotate8<E>(x, y, c, s);
      } else {
        rotate8_neighbours<E>(x, c[0], s[0]);
        rotate8_neighbours<E>(y, c[1], s[1]);
      }
    }
    *reinterpret_cast<u32x4*>(dst[j] + a0) = x;
    *reinterpret_cast<u32x4*>(dst[j] + b0) = y;
  }
}

// Any even rot_dim and any D: one pair, or one element beyond them, a thread.
template <typename E>
__global__ void __launch_bounds__(kThreads) append_scalar_kernel(AppendParams p, bool interleaved) {
  const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t t = i / (p.units * p.groups);
  if (t >= p.T) return;
  const uint32_t h = i / p.units % p.groups, u = i % p.units;
  const uint32_t pos = static_cast<uint32_t>(p.positions[t]);
  if (pos >= p.rope_rows) return;
  int64_t krow = 0, vrow = 0;
  const bool stored = h >= p.Hq && cache_row(p, t, pos, &krow, &vrow);
  const char* src;
  char* dst;
  if (!head_rows(p, t, h, stored, krow, vrow, &src, &dst)) return;
  const uint16_t* x = reinterpret_cast<const uint16_t*>(src);
  uint16_t* y = reinterpret_cast<uint16_t*>(dst);
  const uint32_t half = p.rot / 2;
  if (u >= half) {
    y[half + u] = x[half + u];
    return;
  }
  const uint32_t a = interleaved ? 2 * u : u, b = interleaved ? 2 * u + 1 : u + half;
  uint16_t xa = x[a], xb = x[b];
  if (h < p.Hq + p.Hkv) {
    const float* row = p.rope + static_cast<int64_t>(pos) * p.rot;
    const float c = row[u], s = row[half + u], fa = unpack_lo<E>(xa), fb = unpack_lo<E>(xb);
    const uint32_t w = pack2<E>(fa * c - fb * s, fb * c + fa * s);
    xa = static_cast<uint16_t>(w);
    xb = static_cast<uint16_t>(w >> 16);
  }
  y[a] = xa;
  y[b] = xb;
}

// ---- 8-bit caches ----------------------------------------------------------------
// A head's row is kLanes lanes', eight numbers each: they rotate them (each lane reads its numbers' partners itself),
// find the row's largest magnitude by lane exchanges and store eight codes each, the first the scale.
//
// The rotation's products and sums are rounded one by one, and the scaling is a reciprocal and a product a row and a product a number: the
// codes are then the same whoever computes them, to the bit, and a test can ask for that.  A number half way between two codes may
// get either, which are as near (a division a number, which would see it, took 80 us for 8190 tokens and their reading back instead of 78).
//
// Bound by memory: 8190 tokens of 64 + 2x8 heads of 128 64 us, 14 to read them back (78 both, 4.8 TB/s); one token 3.4 and 2.5 us of GPU.

// The largest v of kLanes neighbouring lanes.
template <int kLanes>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
  auto dpp = [](uint32_t x, auto ctrl) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), decltype(ctrl)::value, 0xF, 0xF, false));
  };
  v = max(v, dpp(v, std::integral_constant<int, 0xB1>{}));   // lane ^ 1
  v = max(v, dpp(v, std::integral_constant<int, 0x4E>{}));   // lane ^ 2
  v = max(v, dpp(v, std::integral_constant<int, 0x141>{}));  // mirrored in eight lanes
  if (kLanes > 8) v = max(v, dpp(v, std::integral_constant<int, 0x140>{}));  // in sixteen
  if (kLanes > 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(r[0], r[1]);
  }
  return v;
}

template <typename E>
__device__ __forceinline__ void widen(const u32x4& x, float (&y)[8]) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    y[2 * w] = unpack_lo<E>(x[w]);
    y[2 * w + 1] = unpack_hi<E>(x[w]);
  }
}

// Numbers d0 .. d0 + 7 of a row, rotated: half tables and partners a number at a time where they are no multiples of eight.
template <typename E, int kKind>
__device__ __forceinline__ void rotated8(const uint16_t* row, const u32x4& own, const u32x4& other, uint32_t d0, const AppendParams& p, bool inter,
                                         const float* table, const float (&c)[8], const float (&s)[8], float (&y)[8]) {
#pragma clang fp contract(off)
  float x[8];
  widen<E>(own, x);
  const uint32_t half = p.rot / 2;
  if constexpr (kKind == kHalf) {
    float o[8];
    widen<E>(other, o);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float a = x[e] * c[e], b = o[e] * s[e];
      y[e] = d0 < half ? a - b : a + b;
    }
  } else if constexpr (kKind == kInterleaved) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float ac = x[e] * c[e / 2], bs = x[e + 1] * s[e / 2], bc = x[e + 1] * c[e / 2], as = x[e] * s[e / 2];
      y[e] = ac - bs;
      y[e + 1] = bc + as;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t d = d0 + e;
      y[e] = x[e];
      if (d >= p.rot) continue;
      const bool first = inter ? !(d & 1) : d < half;
      const uint32_t i = inter ? d / 2 : first ? d : d - half, with = inter ? d ^ 1 : first ? d + half : d - half;
      const float a = x[e] * table[i], b = unpack_lo<E>(row[with]) * table[half + i];
      y[e] = first ? a - b : a + b;
    }
  }
}

// Queries may be rotated where they stand, and a lane reads numbers that its row's other lanes write: all of them belong to one wave, in which
// nothing that is written behind this fence is written before what stands in front of it is read.
__device__ __forceinline__ void row_is_read() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

template <typename E, typename Q, int kKind, int kLanes, int kHeads>
__global__ void __launch_bounds__(kThreads) append8_kernel(AppendParams p, Scales scales, bool inter) {
  static_assert(kWave % kLanes == 0, "a row's lanes are of one wave");
  const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t u = i % kLanes, t = i / kLanes / p.groups, g = i / kLanes % p.groups;
  if (t >= p.T) return;
  const uint32_t pos = static_cast<uint32_t>(p.positions[t]);
  if (pos >= p.rope_rows) return;
  const uint32_t h0 = g * kHeads, H = p.Hq + 2 * p.Hkv, d0 = 8 * u, half = p.rot / 2;
  uint32_t page = 0, off = 0;
  const bool stored = h0 + kHeads > p.Hq && find_row(p.cache, p.seqs, p.n_seq, t, pos, &page, &off);
  const bool in = d0 < p.D, turned = in && d0 < p.rot;
  const float* table = p.rope + static_cast<int64_t>(pos) * p.rot;
  float c[8], s[8];
  uint32_t other = d0;
  if (kKind != kScalar && turned) {
    const uint32_t i0 = kKind == kInterleaved ? d0 / 2 : d0 < half ? d0 : d0 - half;
    if (kKind == kHalf) other = d0 < half ? d0 + half : d0 - half;
#pragma unroll
    for (int e = 0; e < (kKind == kHalf ? 8 : 4); e += 4) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(table + i0 + e), y = *reinterpret_cast<const f32x4*>(table + half + i0 + e);
#pragma unroll
      for (int j = 0; j < 4; ++j) c[e + j] = x[j], s[e + j] = y[j];
    }
  }
  const char* src[kHeads];
  u32x4 x[kHeads], y[kHeads];
#pragma unroll
  for (int j = 0; j < kHeads; ++j) {
    const uint32_t h = h0 + j;
    src[j] = h < p.Hq ? p.q + t * p.q_token + h * p.q_head
             : h < p.Hq + p.Hkv ? p.k + t * p.k_token + (h - p.Hq) * p.k_head
                                : p.v + t * p.v_token + (h - p.Hq - p.Hkv) * p.v_head;
    const bool live = h < H && in && (h < p.Hq || stored);
    x[j] = live ? *reinterpret_cast<const u32x4*>(src[j] + 2 * d0) : u32x4{0, 0, 0, 0};
    if (kKind == kHalf) y[j] = live && turned && h < p.Hq + p.Hkv ? *reinterpret_cast<const u32x4*>(src[j] + 2 * other) : u32x4{0, 0, 0, 0};
  }
  row_is_read();
#pragma unroll
  for (int j = 0; j < kHeads; ++j) {
    const uint32_t h = h0 + j;
    if (h >= H) return;
    float r[8];
    if (turned && h < p.Hq + p.Hkv)
      rotated8<E, kKind>(reinterpret_cast<const uint16_t*>(src[j]), x[j], y[j], d0, p, inter, table, c, s, r);
    else
      widen<E>(x[j], r);
    if (kKind == kScalar) row_is_read();
    if (h < p.Hq) {
      if (in) {
        u32x4 o;
#pragma unroll
        for (int w = 0; w < 4; ++w) o[w] = pack2<E>(r[2 * w], r[2 * w + 1]);
        *reinterpret_cast<u32x4*>(p.q_out + t * p.qo_token + h * p.qo_head + 2 * d0) = o;
      }
      continue;
    }
    if (!stored) return;
    uint32_t most = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) most = max(most, __float_as_uint(r[e]) & 0x7FFFFFFFu);
    most = lanes_max<kLanes>(most);
    const bool finite = most < 0x7F800000u;
    const float m = fmaxf(__uint_as_float(most), 0x1p-100f), by = Q::kTop * (1.f / m);
    u32x2 codes{0, 0};
    if (finite) {
      float z[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) z[e] = r[e] * by;
      codes = u32x2{Q::codes(z), Q::codes(z + 4)};
    }
    const bool key = h < p.Hq + p.Hkv;
    const uint32_t hk = h - p.Hq - (key ? 0 : p.Hkv);
    char* to = const_cast<char*>(key ? p.cache.k + page * p.cache.k_page + off * p.cache.k_row + hk * p.cache.k_head
                                     : p.cache.v + page * p.cache.v_page + off * p.cache.v_row + hk * p.cache.v_head);
    if (in) *reinterpret_cast<u32x2*>(to + d0) = codes;
    char* sc = const_cast<char*>(key ? scales.k + page * scales.k_page + hk * scales.k_head : scales.v + page * scales.v_page + hk * scales.v_head);
    if (u == 0) reinterpret_cast<float*>(sc)[off] = finite ? m / Q::kTop : __uint_as_float(0x7FC00000u);
  }
}

// ---- reading back ----------------------------------------------------------------
struct ReadParams {
  Cache cache;
  Scales scales;
  char* k;
  char* v;
  int64_t k_token, k_head, v_token, v_head;  // bytes
  const int32_t* positions;
  const int32_t* seqs;
  uint32_t n_seq, T, Hkv, D;
};

// Eight numbers of a key or value row a thread.  Q: void for a 16-bit cache.
template <typename E, typename Q>
__global__ void __launch_bounds__(kThreads) read_kernel(ReadParams p) {
  const uint32_t i = blockIdx.x * kThreads + threadIdx.x, pieces = p.D / 8;
  const uint32_t u = i % pieces, h = i / pieces % (2 * p.Hkv), t = i / pieces / (2 * p.Hkv);
  if (t >= p.T) return;
  const bool key = h < p.Hkv;
  const uint32_t hk = key ? h : h - p.Hkv;
  uint32_t page, off;
  u32x4 o{0, 0, 0, 0};
  if (find_row(p.cache, p.seqs, p.n_seq, t, static_cast<uint32_t>(p.positions[t]), &page, &off)) {
    const char* from = key ? p.cache.k + page * p.cache.k_page + off * p.cache.k_row + hk * p.cache.k_head
                           : p.cache.v + page * p.cache.v_page + off * p.cache.v_row + hk * p.cache.v_head;
    if constexpr (std::is_void<Q>::value) {
      o = *reinterpret_cast<const u32x4*>(from + 16 * u);
    } else {
      const char* sc = key ? p.scales.k + page * p.scales.k_page + hk * p.scales.k_head : p.scales.v + page * p.scales.v_page + hk * p.scales.v_head;
      const float s = reinterpret_cast<const float*>(sc)[off];
      const u32x2 w = *reinterpret_cast<const u32x2*>(from + 8 * u);
#pragma unroll
      for (int a = 0; a < 4; ++a) o[a] = pack2<E>(Q::value(w[a >> 1], 2 * (a & 1)) * s, Q::value(w[a >> 1], 2 * (a & 1) + 1) * s);
    }
  }
  *reinterpret_cast<u32x4*>((key ? p.k + t * p.k_token + hk * p.k_head : p.v + t * p.v_token + hk * p.v_head) + 16 * u) = o;
}

int validate(const latent_kv_append_args& a) {
  const int st = check_heads(a.n_head, a.n_kv_head, a.head_dim, a.dtype);
  if (st != LATENT_OK) return st;
  if (a.n_tokens < 0) return LATENT_E_INVALID;
  if (a.rope_kind != LATENT_ROPE_HALF && a.rope_kind != LATENT_ROPE_INTERLEAVED) return LATENT_E_INVALID;
  if (a.rope && (a.rope_rows < 0 || a.rot_dim <= 0 || a.rot_dim % 2 || a.rot_dim > a.head_dim)) return LATENT_E_INVALID;
  if (a.n_tokens > (1 << 24) || a.rope_rows > INT32_MAX) return LATENT_E_UNSUPPORTED;
  // Work items are counted in 32 bits.
  if (a.n_tokens * (a.n_head + 2 * a.n_kv_head) * a.head_dim > (int64_t{1} << 32) - 4096) return LATENT_E_UNSUPPORTED;
  return check_cache(a.cache);
}

}  // namespace
}  // namespace attend
}  // namespace latent

using namespace latent;
using namespace latent::attend;

namespace {

// The checks of an append, and its parameters.  size: bytes of a cache element.
int append_params(const latent_kv_append_args& a, int64_t size, AppendParams* out) {
  const int st = validate(a);
  if (st != LATENT_OK) return st;
  if (a.n_tokens == 0) return LATENT_OK;
  const bool q = a.n_head > 0;
  if (!a.k || !a.v || !a.positions || (q && (!a.q || !a.q_out))) return LATENT_E_INVALID;
  if (a.cache.n_pages > 0 && (!a.cache.k || !a.cache.v)) return LATENT_E_INVALID;
  if (a.cache.n_seq > 0 && a.cache.max_pages > 0 && !a.cache.pages) return LATENT_E_INVALID;
  for (const void* ptr : {a.q, static_cast<const void*>(a.q_out), a.k, a.v, static_cast<const void*>(a.rope)})
    if (!aligned16(ptr)) return LATENT_E_UNSUPPORTED;
  for (int64_t s : {a.k_token_stride, a.k_head_stride, a.v_token_stride, a.v_head_stride})
    if (!stride_ok(s)) return LATENT_E_UNSUPPORTED;
  if (q)
    for (int64_t s : {a.q_token_stride, a.q_head_stride, a.q_out_token_stride, a.q_out_head_stride})
      if (!stride_ok(s)) return LATENT_E_UNSUPPORTED;
  // What is written may not be one place for several rows.
  const latent_kv_cache& c = a.cache;
  if ((a.n_kv_head > 1 && (!c.k_head_stride || !c.v_head_stride)) || (c.page_size > 1 && (!c.k_row_stride || !c.v_row_stride)) ||
      (c.n_pages > 1 && (!c.k_page_stride || !c.v_page_stride)) || (a.n_head > 1 && !a.q_out_head_stride) ||
      (q && a.n_tokens > 1 && !a.q_out_token_stride))
    return LATENT_E_INVALID;
  AppendParams& p = *out;
  p.cache = device_cache(a.cache, size);
  p.q = static_cast<const char*>(a.q);
  p.q_out = static_cast<char*>(a.q_out);
  p.k = static_cast<const char*>(a.k);
  p.v = static_cast<const char*>(a.v);
  p.q_token = a.q_token_stride * 2, p.q_head = a.q_head_stride * 2;
  p.qo_token = a.q_out_token_stride * 2, p.qo_head = a.q_out_head_stride * 2;
  p.k_token = a.k_token_stride * 2, p.k_head = a.k_head_stride * 2;
  p.v_token = a.v_token_stride * 2, p.v_head = a.v_head_stride * 2;
  p.positions = a.positions;
  p.seqs = a.seqs;
  p.rope = a.rope;
  p.rope_rows = a.rope ? static_cast<uint32_t>(a.rope_rows) : 1u << 31;
  p.n_seq = static_cast<uint32_t>(a.cache.n_seq);
  p.T = static_cast<uint32_t>(a.n_tokens);
  p.Hq = static_cast<uint32_t>(a.n_head);
  p.Hkv = static_cast<uint32_t>(a.n_kv_head);
  p.D = static_cast<uint32_t>(a.head_dim);
  p.rot = a.rope ? static_cast<uint32_t>(a.rot_dim) : 0;
  return LATENT_OK;
}

}  // namespace

extern "C" int latent_kv_append(const latent_kv_append_args* args, latent_stream_t stream) {
  if (!args) return LATENT_E_INVALID;
  const latent_kv_append_args& a = *args;
  AppendParams p{};
  const int st = append_params(a, 2, &p);
  if (st != LATENT_OK || a.n_tokens == 0) return st;
  const uint32_t H = p.Hq + 2 * p.Hkv;
  const bool f16 = a.dtype == LATENT_F16, inter = a.rope_kind == LATENT_ROPE_INTERLEAVED;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  (void)hipGetLastError();
  auto launch = [&](auto kernel, auto... more) {
    const uint64_t items = static_cast<uint64_t>(p.T) * p.groups * p.units;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>((items + kThreads - 1) / kThreads)), dim3(kThreads), 0, s, p, more...);
  };
  if (p.D % 16 || p.rot % 16) {
    p.units = p.D - p.rot / 2;
    p.groups = H;
    f16 ? launch(append_scalar_kernel<F16>, inter) : launch(append_scalar_kernel<BF16>, inter);
    return hipGetLastError() == hipSuccess ? LATENT_OK : LATENT_E_HIP;
  }
  p.units = p.D / 16;
  // Four heads a thread once that leaves every CU a workgroup.
  const bool wide = static_cast<uint64_t>(p.T) * H * p.units >= 4 * 256 * kThreads;
  p.groups = wide ? (H + 3) / 4 : H;
  auto pick = [&](auto e) {
    using E = decltype(e);
    if (inter)
      wide ? launch(append_kernel<E, kInterleaved, 4>) : launch(append_kernel<E, kInterleaved, 1>);
    else
      wide ? launch(append_kernel<E, kHalf, 4>) : launch(append_kernel<E, kHalf, 1>);
  };
  f16 ? pick(F16{}) : pick(BF16{});
  return hipGetLastError() == hipSuccess ? LATENT_OK : LATENT_E_HIP;
}

extern "C" int latent_kv_append_q8(const latent_kv_append_args* args, const latent_kv_scales* scales, latent_stream_t stream) {
  if (!args || !scales) return LATENT_E_INVALID;
  const latent_kv_append_args& a = *args;
  int st = validate(a);
  if (st == LATENT_OK) st = check_codes(a.cache, *scales, a.head_dim);
  if (st != LATENT_OK) return st;
  AppendParams p{};
  st = append_params(a, 1, &p);
  if (st != LATENT_OK || a.n_tokens == 0) return st;
  if (a.cache.n_pages > 0 && (!scales->k || !scales->v)) return LATENT_E_INVALID;
  if ((a.n_kv_head > 1 && (!scales->k_head_stride || !scales->v_head_stride)) ||
      (a.cache.n_pages > 1 && (!scales->k_page_stride || !scales->v_page_stride)))
    return LATENT_E_INVALID;
  const Scales sc = device_scales(*scales);
  const bool inter = a.rope_kind == LATENT_ROPE_INTERLEAVED;
  const uint32_t H = p.Hq + 2 * p.Hkv, lanes = p.D <= 64 ? 8 : p.D <= 128 ? 16 : 32;
  // Four heads a thread once that leaves every CU a workgroup.
  const bool wide = static_cast<uint64_t>(p.T) * H * lanes >= 4 * 256 * kThreads;
  p.groups = wide ? (H + 3) / 4 : H;
  const uint64_t items = static_cast<uint64_t>(p.T) * p.groups * lanes;
  if (items > (uint64_t{1} << 32) - kThreads) return LATENT_E_UNSUPPORTED;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  (void)hipGetLastError();
  auto launch = [&](auto e, auto q, auto kind, auto l) {
    constexpr int kKind = decltype(kind)::value, kLanes = decltype(l)::value;
    const dim3 grid(static_cast<unsigned>((items + kThreads - 1) / kThreads));
    if (wide)
      hipLaunchKernelGGL((append8_kernel<decltype(e), decltype(q), kKind, kLanes, 4>), grid, dim3(kThreads), 0, s, p, sc, inter);
    else
      hipLaunchKernelGGL((append8_kernel<decltype(e), decltype(q), kKind, kLanes, 1>), grid, dim3(kThreads), 0, s, p, sc, inter);
  };
  using std::integral_constant;
  auto with_lanes = [&](auto e, auto q, auto kind) {
    lanes == 8 ? launch(e, q, kind, integral_constant<int, 8>{})
    : lanes == 16 ? launch(e, q, kind, integral_constant<int, 16>{}) : launch(e, q, kind, integral_constant<int, 32>{});
  };
  auto with_kind = [&](auto e, auto q) {
    if (p.rot % 16)
      with_lanes(e, q, integral_constant<int, kScalar>{});
    else
      inter ? with_lanes(e, q, integral_constant<int, kInterleaved>{}) : with_lanes(e, q, integral_constant<int, kHalf>{});
  };
  auto with_code = [&](auto e) { scales->code == LATENT_CODE_INT8 ? with_kind(e, Int8{}) : with_kind(e, E4M3{}); };
  a.dtype == LATENT_F16 ? with_code(F16{}) : with_code(BF16{});
  return hipGetLastError() == hipSuccess ? LATENT_OK : LATENT_E_HIP;
}

extern "C" int latent_kv_read(const latent_kv_read_args* args, const latent_kv_scales* scales, latent_stream_t stream) {
  if (!args) return LATENT_E_INVALID;
  const latent_kv_read_args& a = *args;
  int st = check_heads(a.n_kv_head, a.n_kv_head, a.head_dim, a.dtype);
  if (st != LATENT_OK) return st;
  if (a.n_tokens < 0) return LATENT_E_INVALID;
  if (a.n_tokens > (1 << 24) || a.n_tokens * 2 * a.n_kv_head * a.head_dim > (int64_t{1} << 35) - 8 * kThreads) return LATENT_E_UNSUPPORTED;
  st = check_cache(a.cache);
  if (st == LATENT_OK && scales) st = check_codes(a.cache, *scales, a.head_dim);
  if (st != LATENT_OK || a.n_tokens == 0) return st;
  if (!a.k || !a.v || !a.positions) return LATENT_E_INVALID;
  if (a.cache.n_pages > 0 && (!a.cache.k || !a.cache.v || (scales && (!scales->k || !scales->v)))) return LATENT_E_INVALID;
  if (a.cache.n_seq > 0 && a.cache.max_pages > 0 && !a.cache.pages) return LATENT_E_INVALID;
  if (!aligned16(a.k) || !aligned16(a.v)) return LATENT_E_UNSUPPORTED;
  for (int64_t s : {a.k_token_stride, a.k_head_stride, a.v_token_stride, a.v_head_stride})
    if (!stride_ok(s)) return LATENT_E_UNSUPPORTED;
  if ((a.n_kv_head > 1 && (!a.k_head_stride || !a.v_head_stride)) || (a.n_tokens > 1 && (!a.k_token_stride || !a.v_token_stride)))
    return LATENT_E_INVALID;
  ReadParams p{};
  p.cache = device_cache(a.cache, scales ? 1 : 2);
  if (scales) p.scales = device_scales(*scales);
  p.k = static_cast<char*>(a.k);
  p.v = static_cast<char*>(a.v);
  p.k_token = a.k_token_stride * 2, p.k_head = a.k_head_stride * 2;
  p.v_token = a.v_token_stride * 2, p.v_head = a.v_head_stride * 2;
  p.positions = a.positions;
  p.seqs = a.seqs;
  p.n_seq = static_cast<uint32_t>(a.cache.n_seq);
  p.T = static_cast<uint32_t>(a.n_tokens);
  p.Hkv = static_cast<uint32_t>(a.n_kv_head);
  p.D = static_cast<uint32_t>(a.head_dim);
  const uint64_t items = static_cast<uint64_t>(p.T) * 2 * p.Hkv * (p.D / 8);
  const dim3 grid(static_cast<unsigned>((items + kThreads - 1) / kThreads));
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  (void)hipGetLastError();
  auto launch = [&](auto e) {
    using E = decltype(e);
    if (!scales)
      hipLaunchKernelGGL((read_kernel<E, void>), grid, dim3(kThreads), 0, s, p);
    else if (scales->code == LATENT_CODE_INT8)
      hipLaunchKernelGGL((read_kernel<E, Int8>), grid, dim3(kThreads), 0, s, p);
    else
      hipLaunchKernelGGL((read_kernel<E, E4M3>), grid, dim3(kThreads), 0, s, p);
  };
  a.dtype == LATENT_F16 ? launch(F16{}) : launch(BF16{});
  return hipGetLastError() == hipSuccess ? LATENT_OK : LATENT_E_HIP;
}
