// Attention of whole prompts: packed sequences, causal, grouped heads, keys and
// values packed or in the paged cache.
//
//   out[i] = sum_j softmax_j(scale q[i] . k[j]) v[j],  j <= i + m - n  (n queries, m keys)
//
// A workgroup takes 128 rows of one sequence and key/value head.  Row r is query
// token r / G, query head r % G of the group: all heads that read the same keys
// share the tiles, and a few tokens of many heads fill a tile as well as many of
// one.  Keys come in tiles of 64 through LDS, one pass, with the running maximum
// and sum of the softmax; the next tile is on its way into registers meanwhile.
//
// Each wave owns 32 rows.  scores^T = K Q^T on 32x32x16 products leaves every
// lane the scores of one row (lane % 32) for keys 8 (r / 4) + 4 (lane / 32) + r % 4,
// so maximum and sum are per-lane loops and one exchange between lane halves, and
// eight consecutive registers, rounded, are the operand of out^T = V^T P^T as
// they stand; the value operand is read transposed from LDS in that key order.
#include "attend.hpp"

#include <algorithm>
#include <type_traits>

namespace latent {
namespace attend {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kRowsWave = 32;
constexpr int kRowsTile = kRowsWave * kWaves;
constexpr int kKeys = 64;  // keys of a tile
// The exponentials' reference follows the running maximum only when it is passed by more than this (log2): the sums are
// rescaled a few times a row instead of with almost every tile.  Probabilities then reach 2^8 before the
// division by their sum, which costs no precision (f16 holds up to 2^15).
constexpr float kSlack = 8.f;

struct PromptParams {
  Cache cache;  // packed keys: k, v, k_row, k_head, v_row, v_head alone
  const char* q;
  char* out;
  float* lse;
  const int32_t* starts;
  const int32_t* k_starts;  // packed
  const int32_t* lengths;   // paged
  int64_t q_token, q_head, o_token, o_head;  // bytes
  int32_t T, n_keys, B, Hq, Hkv, G, D;
  bool causal;
  float scale_log2;
};

// Rows [s0, s0 + n) of sequence b.
__device__ __forceinline__ int2 rows_of(const int32_t* starts, int b, int most) {
  const int s0 = min(max(starts[b], 0), most), s1 = min(max(starts[b + 1], s0), most);
  return int2{s0, s1 - s0};
}

__device__ __forceinline__ int tiles_of(const PromptParams& p, int b) {
  return static_cast<int>((static_cast<int64_t>(rows_of(p.starts, b, p.T).y) * p.G + kRowsTile - 1) / kRowsTile);
}

// Sequence and tile of work item x, or false behind the last.
__device__ __forceinline__ bool find_tile(const PromptParams& p, int x, int lane, int* b, int* tile) {
  int base = 0;
  for (int b0 = 0; b0 < p.B; b0 += kWave) {
    const int n = b0 + lane < p.B ? tiles_of(p, b0 + lane) : 0;
    int upto = n;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const int o = __shfl_up(upto, d);
      if (lane >= d) upto += o;
    }
    upto += base;
    const uint64_t past = __ballot(upto > x);
    if (past) {
      const int first = __builtin_ctzll(past);
      *b = b0 + first;
      *tile = __shfl(upto, first) - 1 - x;  // the last rows see the most keys: they start first
      return true;
    }
    base = __shfl(upto, kWave - 1);
  }
  return false;
}

// A tile in LDS: rows of kC 16-byte pieces, permuted so that the lanes of a read spread over all banks: a key row's
// pieces for neighbouring keys; 64 bytes of four neighbouring value rows.  Piece c of row `key` lies at place c ^ *_turn(key).
template <int kDP>
struct Shared {
  static constexpr int kC = kDP / 8;
  static constexpr uint32_t kTile = kKeys * kDP * 2;
  u32x4 k[2][kKeys * kC];
  u32x4 v[2][kKeys * kC];
  // Infinities and NaN among values must not reach the rows that do not see their keys: 0 times them is NaN.  Tiles
  // that some rows see in part hold 0 in their place; the keys they belong to are noted here, and added to
  // the rows that do see them.
  unsigned long long bad[2];
  static __device__ __forceinline__ int k_turn(int key) { return kC >= 16 ? key & 15 : (key >> 1) & 7; }
  static __device__ __forceinline__ int v_turn(int key) { return kC >= 16 ? 4 * (key & 3) : 4 * ((key >> 1) & 1); }
};

typedef short s16x4 __attribute__((ext_vector_type(4)));

// Four 16-bit rows of 16 columns, read by 16 lanes: lane i's address is row i / 4, columns 4 (i % 4) .. + 3; it gets
// column i of the four rows.
__device__ __forceinline__ u32x2 read_transposed(uint32_t at) {
  typedef __attribute__((address_space(3))) s16x4* Lds;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds) static_cast<uintptr_t>(at)));
}

// 0xFFFF in the places of a dword's infinities and NaN.
template <typename E>
__device__ __forceinline__ uint32_t nonfinite(uint32_t w) {
  constexpr uint32_t kExp = __is_same(E, F16) ? 0x7C00u : 0x7F80u;
  return ((w & kExp) == kExp ? 0xFFFFu : 0u) | ((w >> 16 & kExp) == kExp ? 0xFFFF0000u : 0u);
}

template <typename E, int kDP, bool kPaged, bool kLse>
__global__ void __launch_bounds__(kThreads, kDP == 256 ? 1 : 2) prompt_kernel(PromptParams p) {
  typedef Shared<kDP> S;
  constexpr int kC = S::kC, kSteps = kDP / 16, kBlocks = kDP / 32;
  constexpr int kRowsLoad = kWave / kC, kLoads = kKeys / kWaves / kRowsLoad;  // rows of a direct load; loads of a wave and tile
  constexpr uint32_t kRow = kDP * 2;
  __shared__ S sm;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid >> 6), l32 = lane & 31, h = lane >> 5;
  const int hk = blockIdx.x % p.Hkv;
  int b, tile;
  if (!find_tile(p, blockIdx.x / p.Hkv, lane, &b, &tile)) return;
  const int2 qs = rows_of(p.starts, b, p.T);
  const int n = qs.y;
  int k0 = 0, m;
  if constexpr (kPaged) {
    m = min(max(p.lengths[b], 0), static_cast<int>(p.cache.max_len));
  } else {
    const int2 ks = rows_of(p.k_starts, b, p.n_keys);
    k0 = ks.x;
    m = ks.y;
  }
  const int32_t* pages = kPaged ? p.cache.pages + b * p.cache.pages_stride : nullptr;
  const char* kbase = p.cache.k + hk * p.cache.k_head + k0 * p.cache.k_row;
  const char* vbase = p.cache.v + hk * p.cache.v_head + k0 * p.cache.v_row;

  // This lane's row, and how many keys it sees.
  const int64_t all = static_cast<int64_t>(n) * p.G, row0 = static_cast<int64_t>(tile) * kRowsTile;
  const int64_t row = row0 + wave * kRowsWave + l32;
  const bool live = row < all;
  const int64_t rc = live ? row : all - 1;
  const int tok = static_cast<int>(rc / p.G), head = hk * p.G + static_cast<int>(rc % p.G);
  auto sees = [&](int64_t r) { return p.causal ? max(0, min(m, static_cast<int>(min(r, all - 1) / p.G) + m - n + 1)) : m; };
  const int vis = sees(rc);
  const int64_t w0 = row0 + wave * kRowsWave;
  const int all_see = __builtin_amdgcn_readfirstlane(sees(row0));                 // keys that every row of the workgroup sees
  const int wave_all = __builtin_amdgcn_readfirstlane(sees(w0));                  // of the wave
  const int wave_any = __builtin_amdgcn_readfirstlane(w0 < all ? sees(w0 + kRowsWave - 1) : 0);
  const int end = __builtin_amdgcn_readfirstlane(sees(row0 + kRowsTile - 1));     // keys that some row sees

  u32x4 q[kSteps];
  {
    const char* src = p.q + (qs.x + tok) * p.q_token + head * p.q_head;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int d = 16 * s + 8 * h;
      const u32x4 x = *reinterpret_cast<const u32x4*>(src + 2 * min(d, p.D - 8));
      q[s] = live && d < p.D ? x : u32x4{0, 0, 0, 0};
    }
  }

  // Loading: load i of a wave covers kRowsLoad rows from 16 wave + i kRowsLoad; lane l takes the piece that belongs at place
  // l % kC of row l / kC.  Offsets within a tile for packed rows; the pieces of a row for any.
  const int lrow = 16 * wave + lane / kC, lpos = lane % kC;
  uint32_t koff[kPaged ? 1 : kLoads], voff[kPaged ? 1 : kLoads];
  if constexpr (!kPaged) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int key = lrow + i * kRowsLoad;
      koff[i] = key * static_cast<uint32_t>(p.cache.k_row) + 16 * (lpos ^ S::k_turn(key));
      voff[i] = key * static_cast<uint32_t>(p.cache.v_row) + 16 * (lpos ^ S::v_turn(key));
    }
  }
  const uint32_t lds_k = lds_addr(sm.k[0][0]) + wave * (S::kTile / kWaves), lds_v = lds_addr(sm.v[0][0]) + wave * (S::kTile / kWaves);
  const bool exact = p.D == kDP;
  // K or V rows kt .. kt + 63 into buffer buf.
  auto load = [&](bool values, int kt, int buf) {
    const uint32_t to = (values ? lds_v : lds_k) + buf * S::kTile;
    if constexpr (!kPaged) {
      if (kt + kKeys <= end && exact) {
        const char* from = values ? vbase + kt * p.cache.v_row : kbase + kt * p.cache.k_row;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) dma16s(from, values ? voff[i] : koff[i], to + i * (kWave * 16));
        return;
      }
    }
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int row_in = lrow + i * kRowsLoad, key = kt + row_in, c = lpos ^ (values ? S::v_turn(row_in) : S::k_turn(row_in));
      bool ok = key < end;
      const char* from;
      if constexpr (kPaged) {
        const uint32_t pg = static_cast<uint32_t>(key) / p.cache.page_size, off = static_cast<uint32_t>(key) - pg * p.cache.page_size;
        const uint32_t page = ok ? static_cast<uint32_t>(pages[pg]) : 0xFFFFFFFFu;
        ok = page < p.cache.n_pages;
        from = values ? vbase + page * p.cache.v_page + off * p.cache.v_row : kbase + page * p.cache.k_page + off * p.cache.k_row;
      } else {
        from = values ? vbase + key * p.cache.v_row : kbase + key * p.cache.k_row;
      }
      from = ok && 8 * c < p.D ? from + 16 * c : reinterpret_cast<const char*>(kZeroRow);
      dma16(from, to + i * (kWave * 16));
    }
  };

  // Lane parts of the operands' LDS addresses.
  uint32_t kat[kSteps], vat[kBlocks];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) kat[s] = lds_addr(sm.k[0][0]) + l32 * kRow + 16 * ((2 * s + h) ^ S::k_turn(l32));
  {
    const int i16 = lane & 15, row_in = 4 * h + (i16 >> 2);
#pragma unroll
    for (int i = 0; i < kBlocks; ++i)
      vat[i] = lds_addr(sm.v[0][0]) + row_in * kRow + 16 * ((4 * i + 2 * ((lane >> 4) & 1) + ((i16 & 3) >> 1)) ^ S::v_turn(row_in)) + 8 * (i16 & 1);
  }

  f32x16 acc[kBlocks];
#pragma unroll
  for (int i = 0; i < kBlocks; ++i) acc[i] = f32x16{};
  // top: what the exponentials are taken against, within kSlack of the maximum.  The row is divided by the sum of the rounded
  // probabilities that weigh its values, so that their roundings cancel as far as they agree (a row of one key is that
  // key's value); the log-sum-exp, where it is asked for, takes the sum of the unrounded ones.
  float top = -INFINITY, sum = 0.f, full = 0.f;

  auto step = [&](int t, auto bufc) {
    constexpr int buf = decltype(bufc)::value;
    const int kt = t * kKeys;
    pipeline_barrier();  // this tile is there, the other buffer read
    if (kt + kKeys < end) {
      load(false, kt + kKeys, buf ^ 1);
      load(true, kt + kKeys, buf ^ 1);
    }
    const bool part_seen = kt + kKeys > all_see;
    if (part_seen) {
#pragma unroll
      for (int i = 0; i < kKeys * kC / kThreads; ++i) {
        const int at = tid + i * kThreads;
        const uint32_t addr = lds_addr(sm.v[buf][0]) + 16 * at;
        const u32x4 x = lds_ld<u32x4>(addr);
        u32x4 is;
#pragma unroll
        for (int a = 0; a < 4; ++a) is[a] = nonfinite<E>(x[a]);
        if (is[0] | is[1] | is[2] | is[3]) {
          lds_st(addr, x & ~is);
          atomicOr(&sm.bad[buf], 1ull << (at / kC));
        }
      }
      lds_barrier();
      if (tid == 0) sm.bad[buf ^ 1] = 0;
    }
    if (kt >= wave_any) return;  // the other waves' rows see this tile
    f32x16 s[2] = {};
#pragma unroll
    for (int st = 0; st < kSteps; ++st)
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) s[blk] = E::mfma32(lds_ld<u32x4>(kat[st] + buf * S::kTile + blk * 32 * kRow), q[st], s[blk]);
    uint64_t exists = ~uint64_t{0};
    if constexpr (kPaged) {
      const int key = kt + lane;
      exists = __ballot(key < end && static_cast<uint32_t>(pages[static_cast<uint32_t>(key) / p.cache.page_size]) < p.cache.n_pages);
    }
    if (!(kt + kKeys <= wave_all && exists == ~uint64_t{0})) {
#pragma unroll
      for (int blk = 0; blk < 2; ++blk)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = 32 * blk + 8 * (r >> 2) + 4 * h + (r & 3);
          if (kt + key >= vis || !((exists >> key) & 1)) s[blk][r] = -INFINITY;
        }
    }
    float m2[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int r = 0; r < 16; ++r)
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) m2[blk] = fmaxf(m2[blk], s[blk][r]);
    const float t2 = op_over(fmaxf(m2[0], m2[1]), 32, 64, OpMax{}) * p.scale_log2;
    if (__any(t2 > top + kSlack)) {
      const float up = fmaxf(top, t2), f = exp2_fast(top - finite_max(up));
      top = up;
      sum *= f;
      full *= f;
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) acc[i] *= f;
    }
    const float mm = finite_max(top);
    float part[2] = {0.f, 0.f};
    u32x4 prob[4];
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const float x = exp2_fast(s[kk >> 1][8 * (kk & 1) + 2 * a] * p.scale_log2 - mm);
        const float y = exp2_fast(s[kk >> 1][8 * (kk & 1) + 2 * a + 1] * p.scale_log2 - mm);
        prob[kk][a] = pack2<E>(x, y);
        sum = E::add2(prob[kk][a], sum);
        if constexpr (kLse) {
          part[0] += x;
          part[1] += y;
        }
      }
    if constexpr (kLse) full += part[0] + part[1];
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)  // 16 keys
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) {
        const uint32_t at = vat[i] + buf * S::kTile + 16 * kk * kRow;
        const u32x2 lo = read_transposed(at), hi = read_transposed(at + 8 * kRow);
        acc[i] = E::mfma32(u32x4{lo[0], lo[1], hi[0], hi[1]}, prob[kk], acc[i]);
      }
    if (part_seen) {  // what was cleared, to the rows that see it
      for (uint64_t bad = sm.bad[buf]; bad; bad &= bad - 1) {
        const int key = kt + __builtin_ctzll(bad);
        int64_t vo;
        if constexpr (kPaged) {
          const uint32_t pg = static_cast<uint32_t>(key) / p.cache.page_size;
          vo = pages[pg] * p.cache.v_page + (static_cast<uint32_t>(key) - pg * p.cache.page_size) * p.cache.v_row;
        } else {
          vo = key * p.cache.v_row;
        }
#pragma unroll
        for (int i = 0; i < kBlocks; ++i)
#pragma unroll
          for (int rr = 0; rr < 4; ++rr) {
            const int d = 32 * i + 8 * rr + 4 * h;
            if (d >= p.D) continue;
            const u32x2 x = *reinterpret_cast<const u32x2*>(vbase + vo + 2 * d);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t w = x[e >> 1], is = nonfinite<E>(w);
              const bool add = key < vis && (e & 1 ? is >> 16 : is & 0xFFFFu);
              acc[i][4 * rr + e] += add ? (e & 1 ? unpack_hi<E>(w) : unpack_lo<E>(w)) : 0.f;
            }
          }
      }
    }
  };

  if (end > 0) {
    if (tid < 2) sm.bad[tid] = 0;
    load(false, 0, 0);
    load(true, 0, 0);
    const int tiles = (end + kKeys - 1) / kKeys;
    for (int t = 0; t < tiles; t += 2) {
      step(t, std::integral_constant<int, 0>{});
      if (t + 1 < tiles) step(t + 1, std::integral_constant<int, 1>{});
    }
  }

  if (!live) return;
  sum = op_over(sum, 32, 64, OpAdd{});
  const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
  char* dst = p.out + (qs.x + tok) * p.o_token + head * p.o_head;
#pragma unroll
  for (int i = 0; i < kBlocks; ++i)
#pragma unroll
    for (int rr = 0; rr < 4; ++rr) {
      const int d = 32 * i + 8 * rr + 4 * h;
      if (d < p.D)
        *reinterpret_cast<u32x2*>(dst + 2 * d) = u32x2{pack2<E>(acc[i][4 * rr] * inv, acc[i][4 * rr + 1] * inv),
                                                       pack2<E>(acc[i][4 * rr + 2] * inv, acc[i][4 * rr + 3] * inv)};
    }
  if constexpr (kLse) {
    full = op_over(full, 32, 64, OpAdd{});
    if (h == 0) p.lse[static_cast<int64_t>(qs.x + tok) * p.Hq + head] = full == 0.f ? -INFINITY : (top + __log2f(full)) * kLn2;
  }
}

int validate(const latent_attn_prompt_args& a) {
  const int st = check_heads(a.n_head, a.n_kv_head, a.head_dim, a.dtype);
  if (st != LATENT_OK) return st;
  if (a.n_head == 0 || !(a.scale > 0.f) || !(a.scale < INFINITY)) return LATENT_E_INVALID;
  if (a.n_tokens < 0 || a.n_keys < 0 || a.cache.n_seq < 0) return LATENT_E_INVALID;
  if (a.n_tokens > (1 << 28) || a.n_keys > (1 << 28)) return LATENT_E_UNSUPPORTED;
  if (a.cache.n_seq > (1 << 20)) return LATENT_E_UNSUPPORTED;
  // Workgroups are counted in 31 bits.
  const int64_t G = a.n_head / a.n_kv_head, tiles = (a.n_tokens * G + kRowsTile - 1) / kRowsTile + a.cache.n_seq;
  if (tiles * a.n_kv_head > INT32_MAX) return LATENT_E_UNSUPPORTED;
  return a.k ? LATENT_OK : check_cache(a.cache);
}

}  // namespace
}  // namespace attend
}  // namespace latent

using namespace latent;
using namespace latent::attend;

extern "C" int latent_attn_prompt(const latent_attn_prompt_args* args, latent_stream_t stream) {
  if (!args) return LATENT_E_INVALID;
  const latent_attn_prompt_args& a = *args;
  const int st = validate(a);
  if (st != LATENT_OK) return st;
  if (a.n_tokens == 0 || a.cache.n_seq == 0) return LATENT_OK;
  if (!a.q || !a.out || !a.starts) return LATENT_E_INVALID;
  for (int64_t s : {a.q_token_stride, a.q_head_stride, a.out_token_stride, a.out_head_stride})
    if (!stride_ok(s)) return LATENT_E_UNSUPPORTED;
  if (!aligned16(a.q) || !aligned16(a.out)) return LATENT_E_UNSUPPORTED;
  if ((a.n_head > 1 && !a.out_head_stride) || (a.n_tokens > 1 && !a.out_token_stride)) return LATENT_E_INVALID;
  PromptParams p{};
  const bool paged = !a.k;
  if (paged) {
    if (!a.lengths) return LATENT_E_INVALID;
    p.cache = device_cache(a.cache);
    if (a.cache.n_pages == 0)
      p.cache.max_len = 0;
    else if (p.cache.max_len && (!a.cache.k || !a.cache.v || !a.cache.pages))
      return LATENT_E_INVALID;
  } else {
    if (!a.v || !a.k_starts) return LATENT_E_INVALID;
    for (int64_t s : {a.k_token_stride, a.k_head_stride, a.v_token_stride, a.v_head_stride})
      if (!stride_ok(s)) return LATENT_E_UNSUPPORTED;
    if (!aligned16(a.k) || !aligned16(a.v)) return LATENT_E_UNSUPPORTED;
    // A tile's rows are addressed from its first in 32 bits.
    if (a.n_keys > 1 && (a.k_token_stride > (1 << 24) || a.v_token_stride > (1 << 24))) return LATENT_E_UNSUPPORTED;
    p.cache.k = static_cast<const char*>(a.k);
    p.cache.v = static_cast<const char*>(a.v);
    p.cache.k_row = a.k_token_stride * 2, p.cache.k_head = a.k_head_stride * 2;
    p.cache.v_row = a.v_token_stride * 2, p.cache.v_head = a.v_head_stride * 2;
  }
  p.q = static_cast<const char*>(a.q);
  p.out = static_cast<char*>(a.out);
  p.lse = a.lse;
  p.starts = a.starts;
  p.k_starts = a.k_starts;
  p.lengths = a.lengths;
  p.q_token = a.q_token_stride * 2, p.q_head = a.q_head_stride * 2;
  p.o_token = a.out_token_stride * 2, p.o_head = a.out_head_stride * 2;
  p.T = static_cast<int32_t>(a.n_tokens);
  p.n_keys = static_cast<int32_t>(a.n_keys);
  p.B = static_cast<int32_t>(a.cache.n_seq);
  p.Hq = static_cast<int32_t>(a.n_head);
  p.Hkv = static_cast<int32_t>(a.n_kv_head);
  p.G = p.Hq / p.Hkv;
  p.D = static_cast<int32_t>(a.head_dim);
  p.causal = a.causal != 0;
  p.scale_log2 = a.scale * kLog2e;
  // A sequence's rows round up to whole tiles: at most one more each.
  const int64_t tiles = (a.n_tokens * p.G + kRowsTile - 1) / kRowsTile + std::min<int64_t>(a.cache.n_seq, a.n_tokens) - 1;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  (void)hipGetLastError();
  auto launch = [&](auto e, auto dp) {
    constexpr int kDP = decltype(dp)::value;
    using E = decltype(e);
    const dim3 grid(static_cast<unsigned>(std::max<int64_t>(1, tiles) * p.Hkv));
    auto go = [&](auto paged_c) {
      constexpr bool kPaged = decltype(paged_c)::value;
      if (p.lse)
        hipLaunchKernelGGL((prompt_kernel<E, kDP, kPaged, true>), grid, dim3(kThreads), 0, s, p);
      else
        hipLaunchKernelGGL((prompt_kernel<E, kDP, kPaged, false>), grid, dim3(kThreads), 0, s, p);
    };
    paged ? go(std::true_type{}) : go(std::false_type{});
  };
  auto with_type = [&](auto e) {
    if (p.D <= 64)
      launch(e, std::integral_constant<int, 64>{});
    else if (p.D <= 128)
      launch(e, std::integral_constant<int, 128>{});
    else
      launch(e, std::integral_constant<int, 256>{});
  };
  a.dtype == LATENT_F16 ? with_type(F16{}) : with_type(BF16{});
  return hipGetLastError() == hipSuccess ? LATENT_OK : LATENT_E_HIP;
}
