// Attention of whole prompts: work items, tiles in LDS, the join of split units, and the launch plan.  prompt.hip tells the whole.
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
constexpr int kRowsWave = 32;
constexpr int kRowsTile = kRowsWave * kWaves;
// The exponentials' reference follows the running maximum only when it is passed by more than kSlack (log2): the sums are
// rescaled a few times a row instead of with almost every tile.  Probabilities are taken times 2^kUp so that with
// that they end at f16's 2^15, where the small ones keep their bits, and at bf16's 1, where no product with a value can overflow.
template <typename E>
struct Scale {
  static constexpr float kSlack = __is_same(E, F16) ? 2.f : 8.f, kUp = E::kLift - kSlack;
};

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
  Divisor by_group;  // row / G
  bool causal;
  float scale_log2;
  // Splitting (see find_item): parts that the workspace holds, 0 for none.
  int32_t max_parts;
  float items;      // that are to have work
  int32_t least;    // keys of a sequence up to which it stays whole
  f32x4* part_acc;  // [max_parts][4 * 32-dimension blocks][256]
  f32x4* part_ml;   // [max_parts][256]: reference, sum, full sum
  Scales scales;    // of an 8-bit cache
  // kPrefix: one sequence of all T tokens over the first n_keys positions of the cache, of which token t sees lengths[t]; every item
  // of prefix_chunk keys leaves a part.
  int32_t prefix_chunk;
};

// Rows [s0, s0 + n) of sequence b.
__device__ __forceinline__ int2 rows_of(const int32_t* starts, int b, int most) {
  const int s0 = min(max(starts[b], 0), most), s1 = min(max(starts[b + 1], s0), most);
  return int2{s0, s1 - s0};
}

template <bool kPrefix>
__device__ __forceinline__ int2 queries_of(const PromptParams& p, int b) {
  if constexpr (kPrefix) return int2{0, p.T};
  return rows_of(p.starts, b, p.T);
}
// Keys of sequence b: first row (packed) and number.
template <bool kPaged, bool kPrefix>
__device__ __forceinline__ int2 keys_of(const PromptParams& p, int b) {
  if constexpr (kPrefix) return int2{0, p.n_keys};
  if constexpr (kPaged) return int2{0, min(max(p.lengths[b], 0), static_cast<int>(p.cache.max_len))};
  return rows_of(p.k_starts, b, p.n_keys);
}

__device__ __forceinline__ int row_tiles(const PromptParams& p, int n) {
  return (n * p.G + kRowsTile - 1) / kRowsTile;
}
// v, computed from here on: what only a rare branch needs is not kept in registers beside the common path's.
__device__ __forceinline__ int opaque(int v) {
  asm volatile("" : "+v"(v));
  return v;
}
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
// Keys that row r of a sequence of n queries and m keys sees.
__device__ __forceinline__ int keys_seen(const PromptParams& p, int n, int m, int r) {
  return p.causal ? max(0, min(m, static_cast<int>(p.by_group.of(min(r, n * p.G - 1))) + m - n + 1)) : m;
}

// ---- work items ------------------------------------------------------------------
// A unit is a row tile of one sequence and key/value head.  Sequences go from the longest to the shortest, row tiles
// from the last (which sees the most keys) to the first, so that short units fill the end of the launch.  Where the units
// of all sequences are few against their keys, long ones are split: `chunk` keys an item (whole tiles), at least kChunk and so many
// that about `items` items have work; each item of a split unit leaves a part (reference, sums, unnormalised rows), and
// join_kernel adds them up.  Items of one chunk follow one another: they read the same keys, at about the same time, on the
// same XCD (equal spans of the line of all key tiles, each workgroup's keys its own, balanced as well and ran three
// times longer: 14 prompts of up to 2000 tokens 375 us, 190 us a unit a workgroup).  Against chunks of 512 those of 256 took
// 29.0 us instead of 39.7 (two prompts of 699 tokens, 4 heads of 256), 18.0 of 20.9 (2000 tokens, 2 heads); of 128, 27.5 and 20.4.
// Every wave finds its item by itself, from the sequences in its lanes; more than 64 sequences are taken as they come.
constexpr int kChunk = 256, kChunkStep = 64;
// Sequence `lane`: its row tiles, keys, and the parts of its units.
struct Line {
  int s0, n, k0, m;
  int tiles, parts, chunk;
  uint64_t order;  // longer sequences first, equal ones as they come
};
template <bool kPaged, bool kPrefix>
__device__ __forceinline__ Line line_of(const PromptParams& p, int lane) {
  Line l{};
  if (lane < p.B) {
    const int2 q = queries_of<kPrefix>(p, lane), k = keys_of<kPaged, kPrefix>(p, lane);
    l = {q.x, q.y, k.x, k.y, row_tiles(p, q.y)};
  }
  l.order = static_cast<uint64_t>(l.m) << 6 | (kWave - 1 - lane);
  l.parts = 1;
  l.chunk = INT32_MAX;
  if constexpr (kPrefix) {
    l.chunk = p.prefix_chunk;
    l.parts = max(1, (l.m + l.chunk - 1) / l.chunk);
  } else if (p.max_parts) {
    // Both kernels cut the keys by this sum and have to agree to the last bit, whatever the compiler makes of either: no contraction.
#pragma clang fp contract(off)
    float work = static_cast<float>(l.tiles) * static_cast<float>(l.m);
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) work += __shfl_xor(work, d);
    // chunk > work Hkv / items: split units are less than `items`, and their parts, m / chunk + 1 < 2 m / chunk each, less
    // than twice that (1.001 is for the rounding of the sum).
    l.chunk = uniform(max(kChunk, (static_cast<int>(min(work * static_cast<float>(p.Hkv) * 1.001f / p.items, 1e9f)) / kChunkStep + 1) * kChunkStep));
    if (l.m > l.chunk && l.m > p.least) l.parts = (l.m + l.chunk - 1) / l.chunk;
  }
  return l;
}
// Items of the sequences in front of this lane's (longer ones first).
__device__ __forceinline__ int items_before(const PromptParams& p, const Line& l, int items) {
  int before = 0;
  for (int j = 0; j < p.B; ++j) {
    const uint64_t other = static_cast<uint64_t>(__builtin_amdgcn_readlane(l.m, j)) << 6 | (kWave - 1 - j);
    before += other > l.order ? __builtin_amdgcn_readlane(items, j) : 0;
  }
  return before;
}
struct Item {
  int b, tile, part, chunk;  // chunk: keys
  int s0, n, k0, m;          // the sequence's queries and keys
};
template <bool kPaged, bool kPrefix>
__device__ __forceinline__ Item find_item(const PromptParams& p, int x, int lane) {  // b < 0: behind the last
  if (!kPrefix && p.B > kWave) {
    int base = 0;
    for (int b0 = 0; b0 < p.B; b0 += kWave) {
      const int n = b0 + lane < p.B ? row_tiles(p, rows_of(p.starts, b0 + lane, p.T).y) : 0;
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
        const int b = b0 + first;
        const int2 q = rows_of(p.starts, b, p.T), k = keys_of<kPaged, kPrefix>(p, b);
        return {b, __builtin_amdgcn_readlane(upto, first) - 1 - x, 0, INT32_MAX, uniform(q.x), uniform(q.y), uniform(k.x), uniform(k.y)};
      }
      base = __builtin_amdgcn_readlane(upto, kWave - 1);
    }
    return {-1};
  }
  const Line l = line_of<kPaged, kPrefix>(p, lane);
  const int items = l.tiles * l.parts;
  const int before = items_before(p, l, items);
  const uint64_t mine = __ballot(x >= before && x - before < items);
  if (!mine) return {-1};
  const int b = __builtin_ctzll(mine), r = x - __builtin_amdgcn_readlane(before, b), t = __builtin_amdgcn_readlane(l.tiles, b);
  const int part = uniform(r / t);
  return {b, t - 1 - (r - part * t), part, __builtin_amdgcn_readlane(l.parts, b) > 1 ? l.chunk : INT32_MAX, __builtin_amdgcn_readlane(l.s0, b), __builtin_amdgcn_readlane(l.n, b),
          __builtin_amdgcn_readlane(l.k0, b), __builtin_amdgcn_readlane(l.m, b)};
}

// The keys that rows see, where each token has a length of its own (kPrefix): row r's, and the least of a workgroup's rows from row0 on.
__device__ __forceinline__ int prefix_seen(const PromptParams& p, int m, int r) {
  return max(0, min(m, p.lengths[p.by_group.of(min(r, p.T * p.G - 1))]));
}
__device__ __forceinline__ int least_of(int v) {
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) v = min(v, __shfl_xor(v, d));
  return uniform(v);
}

// Four outputs from dimension d on of a row of token t and head h, and its log-sum-exp.
template <typename E>
__device__ __forceinline__ void store4(const PromptParams& p, int t, int h, int d, float a, float b, float c, float e) {
  *reinterpret_cast<u32x2*>(p.out + t * p.o_token + h * p.o_head + 2 * d) = u32x2{pack2<E>(a, b), pack2<E>(c, e)};
}
template <typename E>
__device__ __forceinline__ void store_lse(const PromptParams& p, int t, int h, float top, float full) {
  p.lse[static_cast<int64_t>(t) * p.Hq + h] = full == 0.f ? -INFINITY : (top - Scale<E>::kUp + __log2f(full)) * kLn2;
}

// A tile in LDS: rows of kC 16-byte pieces, permuted so that the lanes of a read spread over all banks: a key row's
// pieces for neighbouring keys; 64 bytes of four neighbouring value rows.  Piece c of row `key` lies at place c ^ *_turn(key).
template <int kDP, int kKeys>
struct Shared {
  static constexpr int kC = kDP / 8;
  static constexpr uint32_t kTile = kKeys * kDP * 2;
  alignas(512) u32x4 k[2][kKeys * kC];
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

// Adds up the parts of a split unit, 32 dimensions a workgroup; threads as in prompt_kernel.
template <typename E, int kDP, bool kPaged, bool kLse>
__global__ void __launch_bounds__(kThreads) join_kernel(PromptParams p) {
  constexpr int kBlocks = kDP / 32;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), h = lane >> 5, i = blockIdx.y, hk = blockIdx.x % p.Hkv;
  // The split units in the order of their items.
  const Line l = line_of<kPaged, false>(p, lane);
  const int x0 = blockIdx.x / p.Hkv, units = l.parts > 1 ? l.tiles : 0;
  int count = units;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) count += __shfl_xor(count, d);
  if (x0 >= count) return;  // most of the grid, which has room for as many as there can be
  const int before = items_before(p, l, units);
  const uint64_t mine = __ballot(x0 >= before && x0 - before < units);
  if (!mine) return;
  const int b = __builtin_ctzll(mine), r = x0 - __builtin_amdgcn_readlane(before, b), t = __builtin_amdgcn_readlane(l.tiles, b);
  const int first = __builtin_amdgcn_readlane(items_before(p, l, l.tiles * l.parts), b) + r, tile = t - 1 - r;
  const int2 qs = queries_of<false>(p, b);
  const int n = qs.y, m = keys_of<kPaged, false>(p, b).y;
  const int parts = (keys_seen(p, n, m, tile * kRowsTile + kRowsTile - 1) + l.chunk - 1) / l.chunk;
  if (parts < 2) return;  // its rows see too little to be split
  const int row = tile * kRowsTile + (tid >> 6) * kRowsWave + (lane & 31);
  if (row >= n * p.G) return;
  const int at = first * p.Hkv + hk, step = t * p.Hkv;
  if (at + (parts - 1) * step >= p.max_parts) return;  // never, but for `starts` that descend
  float top = -INFINITY, sum = 0.f, full = 0.f;
  f32x4 x[4] = {};
  for (int j0 = 0; j0 < parts; j0 += 4) {
    f32x4 ml[4], a[4][4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t part = at + static_cast<int64_t>(min(j0 + k, parts - 1)) * step;
      ml[k] = p.part_ml[part * kThreads + tid];
      if (j0 + k >= parts) ml[k] = f32x4{-INFINITY, 0.f, 0.f, 0.f};
#pragma unroll
      for (int rr = 0; rr < 4; ++rr) a[k][rr] = p.part_acc[part * (4 * kBlocks * kThreads) + (4 * i + rr) * kThreads + tid];
    }
    const float up = fmaxf(fmaxf(fmaxf(ml[0][0], ml[1][0]), fmaxf(ml[2][0], ml[3][0])), top), mm = finite_max(up);
    const float f = exp2_fast(top - mm);
    top = up;
    sum *= f;
    full *= f;
#pragma unroll
    for (int rr = 0; rr < 4; ++rr) x[rr] *= f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (ml[k][0] == -INFINITY && ml[k][1] == ml[k][1]) continue;  // no keys, and no NaN to pass on
      const float g = exp2_fast(ml[k][0] - mm);
      sum += g * ml[k][1];
      full += g * ml[k][2];
#pragma unroll
      for (int rr = 0; rr < 4; ++rr) x[rr] += a[k][rr] * g;
    }
  }
  const int tok = p.by_group.of(row), head = hk * p.G + row - tok * p.G;
  const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
#pragma unroll
  for (int rr = 0; rr < 4; ++rr) {
    const int d = 32 * i + 8 * rr + 4 * h;
    if (d < p.D) store4<E>(p, qs.x + tok, head, d, x[rr][0] * inv, x[rr][1] * inv, x[rr][2] * inv, x[rr][3] * inv);
  }
  if constexpr (kLse) {
    if (i == 0 && h == 0) store_lse<E>(p, qs.x + tok, head, top, full);
  }
}

// Units may be split where keys are long and units few, as measured at D = 128 unless said otherwise, split and not:
//  - up to kShortKeys, where it saves little, units that leave CUs idle (716 tokens behind 6 cached ones, 184 units: 24.5 and 25.7 us;
//    four chunks of 354 to 517 tokens behind 5 to 210, 448 units: 35.5 and 27.8);
//  - beyond it long packed prompts, where the last rows see all keys and the first almost none, into more items than fit the chip
//    at once (8192 tokens, 256 units: 104 and 154 us; 512 units: 162 and 180; 2048 tokens, 384 units: 47.0 and 47.9; but 1300 tokens,
//    256 units: 37.5 and 32.0, and five prompts of 1300, 440 units: 51.2 and 41.1), fewer where a CU holds one workgroup (D = 256, 2048 tokens, 300 units: 98 and 110; 128 units
//    into 384 items 55, into 512 71);
//  - without the causal mask, where all units are alike, only those less than the CUs (256 units of 2048 keys: 51 and 45);
//  - sequences in the cache, of which the page table only bounds the lengths, up to 1024 (a chunk of 512 tokens behind 4000: 59 and
//    112, two of them 103 and 113, four 182 and 178; behind 30000: 305 and 706; 30 tokens behind 8000: 28 and 185).  Keys that
//    are fewer than the table has room for are split as well: the four chunks of the first line in a wider table take 35.5 us.
constexpr int64_t kFewKeys = 512, kShortKeys = 1024, kFew = 256, kFewPaged = 1024;
constexpr int64_t kLong = 1536;  // keys of a prompt, or of several on average
constexpr int kItems = 512, kItemsCausal = 640, kFewCausal = 640, kItemsWide = 384, kFewWide = 320;
struct Plan {
  int64_t units;  // at most
  bool split;
  int items;
  int64_t least;
  int parts;  // at most
  size_t acc_bytes, ml_bytes;
};
Plan plan_for(const latent_attn_prompt_args& a) {
  Plan pl{};
  const int64_t G = a.n_head / a.n_kv_head;
  // A sequence's rows round up to whole tiles: at most one more each.
  pl.units = std::max<int64_t>(0, (a.n_tokens * G + kRowsTile - 1) / kRowsTile + std::min<int64_t>(a.cache.n_seq, a.n_tokens) - 1) * a.n_kv_head;
  const bool packed = a.k || a.n_keys;
  const int64_t keys = packed ? a.n_keys : a.cache.max_pages * a.cache.page_size;
  const bool wide = a.head_dim > 128, slanted = packed && a.causal && keys >= kLong * std::max<int64_t>(1, a.cache.n_seq);
  const int64_t few = slanted ? (wide ? kFewWide : kFewCausal) : packed || keys <= kShortKeys ? kFew : kFewPaged;
  pl.split = keys > kFewKeys && keys <= (1 << 28) && pl.units < few && a.cache.n_seq <= kWave;
  if (!pl.split) return pl;
  pl.least = slanted && pl.units >= kFew ? kLong : 0;
  pl.items = slanted ? (wide ? kItemsWide : kItemsCausal) : kItems;
  // Parts are less than twice the items, and a unit has no more than chunks of kChunk in the keys.
  const int64_t by_unit = pl.units * ((keys + kChunk - 1) / kChunk);
  pl.parts = static_cast<int>(std::min<int64_t>(2 * pl.items, by_unit));
  // The size is that of the most items, with the mask or without.
  const size_t blocks = a.head_dim <= 64 ? 2 : a.head_dim <= 128 ? 4 : 8;
  const size_t parts = std::min<int64_t>(2 * (wide ? kItems : kItemsCausal), by_unit);
  pl.acc_bytes = parts * 4 * blocks * kThreads * sizeof(f32x4);
  pl.ml_bytes = parts * kThreads * sizeof(f32x4);
  return pl;
}

int validate(const latent_attn_prompt_args& a) {
  const int st = check_heads(a.n_head, a.n_kv_head, a.head_dim, a.dtype);
  if (st != LATENT_OK) return st;
  if (a.n_head == 0 || !(a.scale > 0.f) || !(a.scale < INFINITY)) return LATENT_E_INVALID;
  if (a.n_tokens < 0 || a.n_keys < 0 || a.cache.n_seq < 0) return LATENT_E_INVALID;
  if (a.n_tokens > (1 << 28) || a.n_keys > (1 << 28)) return LATENT_E_UNSUPPORTED;
  // Rows (tokens times the heads of a group) and, of a launch, threads are counted in 32 bits.
  if (a.n_tokens * (a.n_head / a.n_kv_head) > (1 << 30)) return LATENT_E_UNSUPPORTED;
  if (a.cache.n_seq > (1 << 20)) return LATENT_E_UNSUPPORTED;
  const int64_t G = a.n_head / a.n_kv_head, tiles = (a.n_tokens * G + kRowsTile - 1) / kRowsTile + a.cache.n_seq;
  if (tiles * a.n_kv_head > 1 << 23) return LATENT_E_UNSUPPORTED;
  return a.k || a.n_keys ? LATENT_OK : check_cache(a.cache);
}

// The checks of a call and its parameters.  size: bytes of a cache element.
int prompt_params(const latent_attn_prompt_args& a, int64_t size, const Plan& pl, PromptParams* out) {
  if (!a.q || !a.out || !a.starts) return LATENT_E_INVALID;
  for (int64_t s : {a.q_token_stride, a.q_head_stride, a.out_token_stride, a.out_head_stride})
    if (!stride_ok(s)) return LATENT_E_UNSUPPORTED;
  if (!aligned16(a.q) || !aligned16(a.out)) return LATENT_E_UNSUPPORTED;
  if ((a.n_head > 1 && !a.out_head_stride) || (a.n_tokens > 1 && !a.out_token_stride)) return LATENT_E_INVALID;
  PromptParams& p = *out;
  const bool paged = !a.k;
  if (paged) {
    if (a.n_keys || !a.lengths) return LATENT_E_INVALID;
    p.cache = device_cache(a.cache, size);
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
  p.by_group = divisor(p.G);
  p.D = static_cast<int32_t>(a.head_dim);
  p.causal = a.causal != 0;
  p.scale_log2 = a.scale * kLog2e;
  if (pl.split && a.workspace && a.workspace_bytes >= pl.acc_bytes + pl.ml_bytes) {
    if (!aligned16(a.workspace)) return LATENT_E_UNSUPPORTED;
    p.max_parts = pl.parts;
    p.items = static_cast<float>(pl.items);
    p.least = static_cast<int32_t>(pl.least);
    p.part_acc = static_cast<f32x4*>(a.workspace);
    p.part_ml = reinterpret_cast<f32x4*>(static_cast<char*>(a.workspace) + pl.acc_bytes);
  }
  return LATENT_OK;
}

// A decode's queries as one sequence over a shared prefix of n_prefix pages, without a mask.
latent_attn_prompt_args prefix_args(const latent_attn_decode_args& a, const int32_t* prefix, int64_t n_prefix) {
  latent_attn_prompt_args r{};
  r.cache = a.cache;
  r.cache.pages = prefix;
  r.cache.n_seq = 1;
  r.cache.max_pages = r.cache.pages_stride = n_prefix;
  r.q = a.q;
  r.out = a.out;          // not written: parts are
  r.starts = a.lengths;   // not read
  r.lengths = a.lengths;  // one a token
  r.q_token_stride = a.q_token_stride, r.q_head_stride = a.q_head_stride;
  r.out_token_stride = a.out_token_stride, r.out_head_stride = a.out_head_stride;
  r.n_tokens = a.cache.n_seq;
  r.n_head = a.n_head, r.n_kv_head = a.n_kv_head, r.head_dim = a.head_dim;
  r.dtype = a.dtype;
  r.scale = a.scale;
  return r;
}
int prefix_params(const latent_attn_prompt_args& a, int64_t size, const Prior& prior, PromptParams* p) {
  const int st = prompt_params(a, size, Plan{}, p);
  if (st != LATENT_OK) return st;
  p->n_keys = static_cast<int32_t>(p->cache.max_len);
  p->prefix_chunk = prior.chunk;
  p->max_parts = prior.parts * prior.tiles * p->Hkv;
  p->part_acc = reinterpret_cast<f32x4*>(prior.acc);
  p->part_ml = reinterpret_cast<f32x4*>(prior.ml);
  return LATENT_OK;
}

}  // namespace
}  // namespace attend
}  // namespace latent
