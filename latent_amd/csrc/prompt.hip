// Attention of whole prompts: packed sequences, causal, grouped heads, keys and
// values packed or in the paged cache.
//
//   out[i] = sum_j softmax_j(scale q[i] . k[j]) v[j],  j <= i + m - n  (n queries, m keys)
//
// A workgroup takes 128 rows of one sequence and key/value head.  Row r is query
// token r / G, query head r % G of the group: all heads that read the same keys
// share the tiles, and a few tokens of many heads fill a tile as well as many of
// one.  Keys come in tiles of 64 through LDS, one pass, with the running maximum
// and sum of the softmax; direct loads fill the other buffer with the next tile meanwhile.
//
// Each wave owns 32 rows.  scores^T = K Q^T on 32x32x16 products leaves every
// lane the scores of one row (lane % 32) for keys 8 (r / 4) + 4 (lane / 32) + r % 4,
// so maximum and sum are per-lane loops and one exchange between lane halves, and
// eight consecutive registers, rounded, are the operand of out^T = V^T P^T as
// they stand; the value operand is read transposed from LDS in that key order.
//
// Measured (bf16, heads of 128): 8192 tokens of 64 heads over 8 in 1030 to 1130 us by the
// card, 970 to 1070 TFLOP/s; 14 prompts of 162 to 2000 tokens, 32 heads, 191 us.  The long ones are
// bound by the power the products draw: where the 8192 took 1024 us, the same instructions over zeros took
// 832 (the card's 8192^3 matrix product: 1360 TFLOP/s, 1800 over zeros), and
// neither waits nor the order of products and exponentials shows in the time
// (scores a tile ahead with a few exponentials behind every product: 1049 us;
// three and four LDS buffers: the same; no wait for the loads at all: the same).
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
};

// Rows [s0, s0 + n) of sequence b.
__device__ __forceinline__ int2 rows_of(const int32_t* starts, int b, int most) {
  const int s0 = min(max(starts[b], 0), most), s1 = min(max(starts[b + 1], s0), most);
  return int2{s0, s1 - s0};
}

// Keys of sequence b: first row (packed) and number.
template <bool kPaged>
__device__ __forceinline__ int2 keys_of(const PromptParams& p, int b) {
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
template <bool kPaged>
__device__ __forceinline__ Line line_of(const PromptParams& p, int lane) {
  Line l{};
  if (lane < p.B) {
    const int2 q = rows_of(p.starts, lane, p.T), k = keys_of<kPaged>(p, lane);
    l = {q.x, q.y, k.x, k.y, row_tiles(p, q.y)};
  }
  l.order = static_cast<uint64_t>(l.m) << 6 | (kWave - 1 - lane);
  l.parts = 1;
  l.chunk = INT32_MAX;
  if (p.max_parts) {
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
template <bool kPaged>
__device__ __forceinline__ Item find_item(const PromptParams& p, int x, int lane) {  // b < 0: behind the last
  if (p.B > kWave) {
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
        const int2 q = rows_of(p.starts, b, p.T), k = keys_of<kPaged>(p, b);
        return {b, __builtin_amdgcn_readlane(upto, first) - 1 - x, 0, INT32_MAX, uniform(q.x), uniform(q.y), uniform(k.x), uniform(k.y)};
      }
      base = __builtin_amdgcn_readlane(upto, kWave - 1);
    }
    return {-1};
  }
  const Line l = line_of<kPaged>(p, lane);
  const int items = l.tiles * l.parts;
  const int before = items_before(p, l, items);
  const uint64_t mine = __ballot(x >= before && x - before < items);
  if (!mine) return {-1};
  const int b = __builtin_ctzll(mine), r = x - __builtin_amdgcn_readlane(before, b), t = __builtin_amdgcn_readlane(l.tiles, b);
  const int part = uniform(r / t);
  return {b, t - 1 - (r - part * t), part, __builtin_amdgcn_readlane(l.parts, b) > 1 ? l.chunk : INT32_MAX, __builtin_amdgcn_readlane(l.s0, b), __builtin_amdgcn_readlane(l.n, b),
          __builtin_amdgcn_readlane(l.k0, b), __builtin_amdgcn_readlane(l.m, b)};
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

// 0xFFFF in the places of a dword's infinities and NaN.
template <typename E>
__device__ __forceinline__ uint32_t nonfinite(uint32_t w) {
  constexpr uint32_t kExp = __is_same(E, F16) ? 0x7C00u : 0x7F80u;
  return ((w & kExp) == kExp ? 0xFFFFu : 0u) | ((w >> 16 & kExp) == kExp ? 0xFFFF0000u : 0u);
}

template <typename E, int kDP, int kKeys, bool kPaged, bool kLse>
__global__ void __launch_bounds__(kThreads, kDP == 256 ? 1 : 2) prompt_kernel(PromptParams p) {
  typedef Shared<kDP, kKeys> S;
  constexpr int kKeyBlocks = kKeys / 32, kC = S::kC, kSteps = kDP / 16, kBlocks = kDP / 32;
  constexpr int kRowsLoad = kWave / kC, kLoads = kKeys / kWaves / kRowsLoad;  // rows of a direct load; loads of a wave and tile
  constexpr uint32_t kRow = kDP * 2;
  __shared__ S sm;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid >> 6), l32 = lane & 31, h = lane >> 5;
  const int hk = blockIdx.x % p.Hkv;
  const Item it = find_item<kPaged>(p, blockIdx.x / p.Hkv, lane);
  if (it.b < 0) return;
  const int b = it.b, tile = it.tile, n = it.n, m = it.m;
  const int32_t* pages = kPaged ? p.cache.pages + b * p.cache.pages_stride : nullptr;
  const char* kbase = p.cache.k + hk * p.cache.k_head + it.k0 * p.cache.k_row;
  const char* vbase = p.cache.v + hk * p.cache.v_head + it.k0 * p.cache.v_row;

  // This lane's row, and how many keys it sees.
  const int all = n * p.G, row0 = tile * kRowsTile, w0 = row0 + wave * kRowsWave;
  const int vis = keys_seen(p, n, m, w0 + l32);
  const int all_see = uniform(keys_seen(p, n, m, row0));                      // keys that every row of the workgroup sees
  const int end = uniform(keys_seen(p, n, m, row0 + kRowsTile - 1));          // keys that some row sees
  const int wave_all = uniform(keys_seen(p, n, m, w0));                       // of the wave
  const int wave_any = uniform(w0 < all ? keys_seen(p, n, m, w0 + kRowsWave - 1) : 0);
  // This item's keys, and whether they are all of the unit's.
  const int begin = it.part ? it.part * it.chunk : 0;
  if (begin > 0 && begin >= end) return;
  const int stop = begin + min(end - begin, it.chunk);
  const bool whole_unit = begin == 0 && stop == end;

  u32x4 q[kSteps];
  {
    const int row = w0 + l32, rc = min(row, all - 1), tok = p.by_group.of(rc);
    const bool live = row < all;
    const char* src = p.q + (it.s0 + tok) * p.q_token + (hk * p.G + rc - tok * p.G) * p.q_head;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int d = 16 * s + 8 * h;
      const u32x4 x = *reinterpret_cast<const u32x4*>(src + 2 * min(d, p.D - 8));
      q[s] = live && d < p.D ? x : u32x4{0, 0, 0, 0};
    }
  }

  // Loading: load i of a wave covers kRowsLoad rows of its quarter of the tile; lane l takes the piece that belongs at place
  // l % kC of row l / kC.  Offsets within a tile for packed rows; the pieces of a row for any.
  const int lrow = kKeys / kWaves * wave + lane / kC, lpos = lane % kC;
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
  const bool exact = p.D == kDP, same_strides = p.cache.k_page == p.cache.v_page && p.cache.k_row == p.cache.v_row;
  // Paged: the page of key kt + lane of the tile that is loaded next, fetched a tile ahead.
  auto page_of = [&](int kt) -> uint32_t {
    const int key = kt + lane;
    return kPaged && key < stop ? static_cast<uint32_t>(pages[p.cache.by_page.of(key)]) : 0xFFFFFFFFu;
  };
  // Rows kt .. kt + kKeys - 1 of K and V into buffer buf.
  auto load = [&](int kt, int buf, uint32_t page_in_lane) {
    const uint32_t to_k = lds_k + buf * S::kTile, to_v = lds_v + buf * S::kTile;
    if constexpr (!kPaged) {
      if (kt + kKeys <= end) {
        const char *from_k = kbase + kt * p.cache.k_row, *from_v = vbase + kt * p.cache.v_row;
        if (exact) {
#pragma unroll
          for (int i = 0; i < kLoads; ++i) dma16s(from_k, koff[i], to_k + i * (kWave * 16));
#pragma unroll
          for (int i = 0; i < kLoads; ++i) dma16s(from_v, voff[i], to_v + i * (kWave * 16));
        } else {  // pieces beyond D stay the zeros they were set to
#pragma unroll
          for (int i = 0; i < kLoads; ++i) {
            const int row_in = lrow + i * kRowsLoad;
            if (8 * (lpos ^ S::k_turn(row_in)) < p.D) dma16s(from_k, koff[i], to_k + i * (kWave * 16));
            if (8 * (lpos ^ S::v_turn(row_in)) < p.D) dma16s(from_v, voff[i], to_v + i * (kWave * 16));
          }
        }
        return;
      }
    }
    if constexpr (kPaged) {
      // Lane l finds where row l lies, once for the tile; whoever loads a piece of the row asks it (four chunks of 354 to 517
      // tokens: 28.7 us with every load's address worked out by itself, 27.4 so).
      const uint32_t key = kt + opaque(lane), off = key - p.cache.by_page.of(key) * p.cache.page_size;
      const bool there = page_in_lane < p.cache.n_pages;
      const int64_t ko = there ? page_in_lane * p.cache.k_page + off * p.cache.k_row : 0;
      const int64_t vo = same_strides ? ko : there ? page_in_lane * p.cache.v_page + off * p.cache.v_row : 0;
      auto row = [](int64_t o, int of) {
        const uint32_t lo = __builtin_amdgcn_ds_bpermute(4 * of, static_cast<int>(o)), hi = __builtin_amdgcn_ds_bpermute(4 * of, static_cast<int>(o >> 32));
        return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
      };
      const uint64_t have = __ballot(there) | ~(~uint64_t{0} >> (64 - kKeys));
      const bool all = have == ~uint64_t{0} && exact;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int row_in = lrow + i * kRowsLoad, ck = lpos ^ S::k_turn(row_in), cv = lpos ^ S::v_turn(row_in);
        const int64_t kr = row(ko, row_in), vr = same_strides ? kr : row(vo, row_in);
        const char *from_k = kbase + kr + 16 * ck, *from_v = vbase + vr + 16 * cv;
        if (!all) {
          asm volatile("");
          const bool ok = have >> row_in & 1;
          const char* zero = reinterpret_cast<const char*>(kZeroRow);
          from_k = ok && 8 * ck < p.D ? from_k : zero;
          from_v = ok && 8 * cv < p.D ? from_v : zero;
        }
        dma16(from_k, to_k + i * (kWave * 16));
        dma16(from_v, to_v + i * (kWave * 16));
        __builtin_amdgcn_sched_barrier(0);  // all loads' addresses at once would not fit the registers
      }
      return;
    }
    const int ln = opaque(lane), lrow = kKeys / kWaves * wave + ln / kC, lpos = ln % kC;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int row_in = lrow + i * kRowsLoad, key = kt + row_in, ck = lpos ^ S::k_turn(row_in), cv = lpos ^ S::v_turn(row_in);
      const bool ok = key < end;
      const char* zero = reinterpret_cast<const char*>(kZeroRow);
      dma16(ok && 8 * ck < p.D ? kbase + key * p.cache.k_row + 16 * ck : zero, to_k + i * (kWave * 16));
      dma16(ok && 8 * cv < p.D ? vbase + key * p.cache.v_row + 16 * cv : zero, to_v + i * (kWave * 16));
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // Lane parts of the operands' LDS addresses.
  // Step s of a key row is 2 s + h pieces on, permuted by a constant: its address is the first's with 2 s put in by xor; block i of
  // a value row likewise, 4 i pieces on.
  const uint32_t kat = lds_addr(sm.k[0][0]) + l32 * kRow + 16 * (h ^ S::k_turn(l32));
  const int i16 = lane & 15, vrow = 4 * h + (i16 >> 2);
  const uint32_t vat = lds_addr(sm.v[0][0]) + vrow * kRow + 16 * ((2 * ((lane >> 4) & 1) + ((i16 & 3) >> 1)) ^ S::v_turn(vrow)) + 8 * (i16 & 1);

  f32x16 acc[kBlocks];
#pragma unroll
  for (int i = 0; i < kBlocks; ++i) acc[i] = f32x16{};
  // top: what the exponentials are taken against, within kSlack of the maximum.  The row is divided by the sum of the rounded
  // probabilities that weigh its values, so that their roundings cancel as far as they agree (a row of one key is that
  // key's value); the log-sum-exp, where it is asked for, takes the sum of the unrounded ones.
  float top = -INFINITY, sum = 0.f, full = 0.f;
  uint32_t page_now = 0, page_next = 0;  // paged: page_of this tile and the next

  auto step = [&](int kt, auto bufc) {
    constexpr int buf = decltype(bufc)::value;
    pipeline_barrier();  // this tile is there, the other buffer read
    constexpr uint64_t kAll = ~uint64_t{0} >> (64 - kKeys);
    uint64_t exists = kAll;
    if constexpr (kPaged) {
      exists = __ballot(page_now < p.cache.n_pages) & kAll;
      page_now = page_next;
    }
    if (kt + kKeys < stop) {
      load(kt + kKeys, buf ^ 1, page_now);
      if constexpr (kPaged) page_next = page_of(kt + 2 * kKeys);
    }
    __builtin_amdgcn_sched_barrier(0);  // the loads' addresses and the products' operands do not share the registers
    const bool part_seen = kt + kKeys > all_see;
    if (part_seen) {
#pragma unroll
      for (int i = 0; i < kKeys * kC / kThreads; ++i) {
        const int at = opaque(tid) + i * kThreads;
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
    f32x16 s[kKeyBlocks] = {};
#pragma unroll
    for (int st = 0; st < kSteps; ++st)
#pragma unroll
      for (int blk = 0; blk < kKeyBlocks; ++blk) s[blk] = E::mfma32(lds_ld<u32x4>((kat ^ (32 * st)) + buf * S::kTile + blk * 32 * kRow), q[st], s[blk]);
    if (!(kt + kKeys <= wave_all && exists == kAll)) {
      asm volatile("");  // keeps this a branch: most tiles need none of it
      const int left = vis - kt - 4 * (opaque(lane) >> 5);  // of the keys from this lane's first on
      const uint64_t there = exists >> (4 * h);
#pragma unroll
      for (int blk = 0; blk < kKeyBlocks; ++blk)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = 32 * blk + 8 * (r >> 2) + (r & 3);
          const uint32_t half = static_cast<uint32_t>(there >> (32 * blk));
          if (key >= left || (kPaged && !(half & (1u << (key & 31))))) s[blk][r] = -INFINITY;
        }
    }
    float m2[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int r = 0; r < 16; ++r)
#pragma unroll
      for (int blk = 0; blk < kKeyBlocks; ++blk) m2[kKeyBlocks == 1 ? r & 1 : blk] = fmaxf(m2[kKeyBlocks == 1 ? r & 1 : blk], s[blk][r]);
    const float t2 = op_over(fmaxf(m2[0], m2[1]), 32, 64, OpMax{}) * p.scale_log2;
    if (__any(t2 > top + Scale<E>::kSlack)) {
      const float up = fmaxf(top, t2), f = exp2_fast(top - finite_max(up));
      top = up;
      sum *= f;
      full *= f;
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) acc[i] *= f;
    }
    const float mm = finite_max(top) - Scale<E>::kUp;
    float part[2] = {0.f, 0.f};
    float part_sum[2] = {sum, 0.f};
    u32x4 prob[2 * kKeyBlocks];
#pragma unroll
    for (int kk = 0; kk < 2 * kKeyBlocks; ++kk)
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const float x = exp2_fast(s[kk >> 1][8 * (kk & 1) + 2 * a] * p.scale_log2 - mm);
        const float y = exp2_fast(s[kk >> 1][8 * (kk & 1) + 2 * a + 1] * p.scale_log2 - mm);
        prob[kk][a] = pack2<E>(x, y);
        part_sum[a & 1] = E::add2(prob[kk][a], part_sum[a & 1]);
        if constexpr (kLse) {
          part[0] += x;
          part[1] += y;
        }
      }
    sum = part_sum[0] + part_sum[1];
    if constexpr (kLse) full += part[0] + part[1];
#pragma unroll
    for (int kk = 0; kk < 2 * kKeyBlocks; ++kk)  // 16 keys
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) {
        const uint32_t at = (vat ^ (64 * i)) + buf * S::kTile + 16 * kk * kRow;
        const u32x2 lo = read_transposed(at), hi = read_transposed(at + 8 * kRow);
        acc[i] = E::mfma32(u32x4{lo[0], lo[1], hi[0], hi[1]}, prob[kk], acc[i]);
      }
    if (part_seen) {  // what was cleared, to the rows that see it
      for (uint64_t bad = sm.bad[buf]; bad; bad &= bad - 1) {
        const int key = kt + __builtin_ctzll(bad);
        int64_t vo;
        if constexpr (kPaged) {
          const uint32_t pg = p.cache.by_page.of(key);
          vo = pages[pg] * p.cache.v_page + (static_cast<uint32_t>(key) - pg * p.cache.page_size) * p.cache.v_row;
        } else {
          vo = key * p.cache.v_row;
        }
#pragma unroll
        for (int i = 0; i < kBlocks; ++i)
#pragma unroll
          for (int rr = 0; rr < 4; ++rr) {
            const int d = 32 * i + 8 * rr + 4 * (opaque(lane) >> 5);
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

  if (begin < stop) {
    if (tid < 2) sm.bad[tid] = 0;
    if (!kPaged && !exact) {
      for (uint32_t i = tid; i < 4 * S::kTile / 16; i += kThreads) lds_st(lds_addr(sm.k[0][0]) + 16 * i, u32x4{0, 0, 0, 0});
      lds_barrier();
    }
    if constexpr (kPaged) {
      page_now = page_of(begin);
      page_next = page_of(begin + kKeys);
    }
    load(begin, 0, page_now);
    for (int kt = begin; kt < stop; kt += 2 * kKeys) {
      step(kt, std::integral_constant<int, 0>{});
      if (kt + kKeys < stop) step(kt + kKeys, std::integral_constant<int, 1>{});
    }
  }

  sum = op_over(sum, 32, 64, OpAdd{});
  if constexpr (kLse) full = op_over(full, 32, 64, OpAdd{});
  const int row = w0 + (opaque(lane) & 31);
  if (row >= all) return;
  if (!whole_unit) {
    const int part = blockIdx.x;  // items in their order, heads within
    if (part >= p.max_parts) return;  // never, by the choice of chunk and of max_parts, but for `starts` that descend
    f32x4* to = p.part_acc + static_cast<int64_t>(part) * (4 * kBlocks * kThreads) + tid;
#pragma unroll
    for (int i = 0; i < kBlocks; ++i)
#pragma unroll
      for (int rr = 0; rr < 4; ++rr)
        to[(4 * i + rr) * kThreads] = f32x4{acc[i][4 * rr], acc[i][4 * rr + 1], acc[i][4 * rr + 2], acc[i][4 * rr + 3]};
    p.part_ml[static_cast<int64_t>(part) * kThreads + tid] = f32x4{top, sum, full, 0.f};
    return;
  }
  const int tok = p.by_group.of(row), head = hk * p.G + row - tok * p.G;
  const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
  char* dst = p.out + (it.s0 + tok) * p.o_token + head * p.o_head;
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
    if (h == 0) p.lse[static_cast<int64_t>(it.s0 + tok) * p.Hq + head] = full == 0.f ? -INFINITY : (top - Scale<E>::kUp + __log2f(full)) * kLn2;
  }
}

// Adds up the parts of a split unit, 32 dimensions a workgroup; threads as in prompt_kernel.
template <typename E, int kDP, bool kPaged, bool kLse>
__global__ void __launch_bounds__(kThreads) join_kernel(PromptParams p) {
  constexpr int kBlocks = kDP / 32;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), h = lane >> 5, i = blockIdx.y, hk = blockIdx.x % p.Hkv;
  // The split units in the order of their items.
  const Line l = line_of<kPaged>(p, lane);
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
  const int2 qs = rows_of(p.starts, b, p.T);
  const int n = qs.y, m = keys_of<kPaged>(p, b).y;
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
  char* dst = p.out + (qs.x + tok) * p.o_token + head * p.o_head;
#pragma unroll
  for (int rr = 0; rr < 4; ++rr) {
    const int d = 32 * i + 8 * rr + 4 * h;
    if (d < p.D)
      *reinterpret_cast<u32x2*>(dst + 2 * d) = u32x2{pack2<E>(x[rr][0] * inv, x[rr][1] * inv), pack2<E>(x[rr][2] * inv, x[rr][3] * inv)};
  }
  if constexpr (kLse) {
    if (i == 0 && h == 0) p.lse[static_cast<int64_t>(qs.x + tok) * p.Hq + head] = full == 0.f ? -INFINITY : (top - Scale<E>::kUp + __log2f(full)) * kLn2;
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

}  // namespace
}  // namespace attend
}  // namespace latent

using namespace latent;
using namespace latent::attend;

extern "C" int latent_attn_prompt_workspace_size(const latent_attn_prompt_args* args, size_t* bytes) {
  if (!args || !bytes) return LATENT_E_INVALID;
  const int st = validate(*args);
  if (st != LATENT_OK) return st;
  const Plan pl = plan_for(*args);
  *bytes = pl.acc_bytes + pl.ml_bytes;
  return LATENT_OK;
}

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
    if (a.n_keys || !a.lengths) return LATENT_E_INVALID;
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
  p.by_group = divisor(p.G);
  p.D = static_cast<int32_t>(a.head_dim);
  p.causal = a.causal != 0;
  p.scale_log2 = a.scale * kLog2e;
  const Plan pl = plan_for(a);
  if (pl.split && a.workspace && a.workspace_bytes >= pl.acc_bytes + pl.ml_bytes) {
    if (!aligned16(a.workspace)) return LATENT_E_UNSUPPORTED;
    p.max_parts = pl.parts;
    p.items = static_cast<float>(pl.items);
    p.least = static_cast<int32_t>(pl.least);
    p.part_acc = static_cast<f32x4*>(a.workspace);
    p.part_ml = reinterpret_cast<f32x4*>(static_cast<char*>(a.workspace) + pl.acc_bytes);
  }
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  (void)hipGetLastError();
  auto launch = [&](auto e, auto dp) {
    constexpr int kDP = decltype(dp)::value;
    using E = decltype(e);
    // Split units have less than pl.items parts beyond their first.
    const int64_t more = (pl.items / p.Hkv + 1) * p.Hkv, units = std::max<int64_t>(pl.units, p.Hkv);
    auto go = [&](auto paged_c, auto lse_c) {
      constexpr bool kPaged = decltype(paged_c)::value, kLse = decltype(lse_c)::value;
      const dim3 grid(static_cast<unsigned>(units + (p.max_parts ? more : 0)));
      hipLaunchKernelGGL((prompt_kernel<E, kDP, kDP == 256 ? 32 : 64, kPaged, kLse>), grid, dim3(kThreads), 0, s, p);
      if (p.max_parts)
        hipLaunchKernelGGL((join_kernel<E, kDP, kPaged, kLse>), dim3(static_cast<unsigned>(std::min(units, more)), kDP / 32),
                           dim3(kThreads), 0, s, p);
    };
    auto with_lse = [&](auto paged_c) { p.lse ? go(paged_c, std::true_type{}) : go(paged_c, std::false_type{}); };
    paged ? with_lse(std::true_type{}) : with_lse(std::false_type{});
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
