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

// Cache row of a token (byte offsets of head 0), or false.
__device__ __forceinline__ bool cache_row(const AppendParams& p, uint32_t t, uint32_t pos, int64_t* k, int64_t* v) {
  const uint32_t seq = p.seqs ? static_cast<uint32_t>(p.seqs[t]) : t;
  if (seq >= p.n_seq || pos >= p.cache.max_len) return false;
  const uint32_t slot = p.cache.by_page.of(pos), off = pos - slot * p.cache.page_size;
  const uint32_t page = static_cast<uint32_t>(p.cache.pages[seq * p.cache.pages_stride + slot]);
  if (page >= p.cache.n_pages) return false;
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

extern "C" int latent_kv_append(const latent_kv_append_args* args, latent_stream_t stream) {
  if (!args) return LATENT_E_INVALID;
  const latent_kv_append_args& a = *args;
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
  AppendParams p{};
  p.cache = device_cache(a.cache);
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
