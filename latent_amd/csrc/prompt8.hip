// Attention of prompts over an 8-bit paged cache: the 16-bit kernel's items, rows and products (prompt.hip), its tiles made from
// codes on their way to LDS.
//
//   score[j] = scale ks[j] (q . kcode[j]),   out = sum_j (p[j] vs[j]) vcode[j] / sum_j p[j]
//
// Codes are loaded a tile ahead into registers (a tile's keys and values are 64 bytes a thread at D = 128), made exact
// elements of the queries' type there and written to the LDS buffer that the waves do not read: each code is
// converted once for the four waves, and the operands' reads are the 16-bit kernel's.  The scales of a tile's keys lie in LDS beside
// it.  A value's scale is a power of two, which its elements take exactly, times a rest, which its weight takes: as the
// logarithm added to the score (the product with the key's scale becomes a multiply-add), so that one exponential gives p[j] rest[j].
//
// Measured (heads of 128, 32 over 8): two prompts of 4099 behind 8 and 5701 916 us in bf16 over e4m3, 960 over int8, 782 over a 16-bit cache; four
// chunks of 287 to 517 29, 31 and 25 us.  Bound by vector and matrix instructions, which the SIMDs' two waves take in turn (85 % of the
// cycles together): the products are the 16-bit kernel's, the rest is conversions, two operations more a score and the sums.
#include "prompt.hpp"

namespace latent {
namespace attend {
namespace {

// A value row of scale s: its codes times `power`, of two, are the elements; the probability takes `rest`.  s = power rest.  f16: rest
// is from 1 to 2, so that a weight has the bits of its probability, whatever the values' size; the elements are exact but for those
// below the type's normal numbers, which are as near as it has them.  bf16 has fp32's range: the weight takes all of a scale that is
// neither tiny nor huge, beside which the others' weights would be nothing.
template <typename E, typename Q>
struct Split {
  static __device__ __forceinline__ float power(float s) {
    const uint32_t e = __float_as_uint(s) & 0x7F800000u;
    if (!held<E, Q>(s) || (E::kLift == 0.f && e - 0x21800000u < 0x32000000u)) return 1.f;  // from 2^-60 to 2^40
    return __uint_as_float(e);  // 0 for 0
  }
  static __device__ __forceinline__ float rest(float s) {  // of one that is held
    const float p = power(s);
    return p == 0.f ? 1.f : s * __uint_as_float(0x7F000000u - __float_as_uint(p));
  }
};

// Eight codes as 16 bytes of elements, and times a power of two.
template <typename E, typename Q>
__device__ __forceinline__ u32x4 convert8(uint32_t a, uint32_t b) {
  return {Q::template pair<E, false>(a), Q::template pair<E, true>(a), Q::template pair<E, false>(b), Q::template pair<E, true>(b)};
}
template <typename E, typename Q, bool kSmall>
__device__ __forceinline__ u32x4 convert8(uint32_t a, uint32_t b, float power) {
  return {Q::template scaled_pair<E, false, kSmall>(a, power), Q::template scaled_pair<E, true, kSmall>(a, power),
          Q::template scaled_pair<E, false, kSmall>(b, power), Q::template scaled_pair<E, true, kSmall>(b, power)};
}
template <typename E, typename Q>
__device__ __forceinline__ u32x4 convert_value8(uint32_t a, uint32_t b, float power) {
  if constexpr (__is_same(Q, E4M3)) return convert8<E, Q, true>(a, b, power);
  if constexpr (E::kLift == 0.f) {
    if (__all(power == 1.f)) return convert8<E, Q>(a, b);
  } else {
    if (__all(power >= 0x1p-14f)) return convert8<E, Q, false>(a, b, power);
  }
  return convert8<E, Q, true>(a, b, power);
}

template <int kDP, int kKeys>
struct Shared8 {
  static constexpr int kC = kDP / 8;
  static constexpr uint32_t kTile = kKeys * kDP * 2;
  alignas(512) u32x4 k[2][kKeys * kC];
  u32x4 v[2][kKeys * kC];
  float ks[2][kKeys], add[2][kKeys];  // a score's factor, base 2, and what is added: the log2 of its value's rest
  float whole[2][kKeys];              // one over the rest; the log-sum-exp takes it unrounded
  u32x4 over[2][kKeys / 4];           // one over the rests of four keys as two summands of the element type: (0, 1), (2, 3), then the smaller
  int bad[2];                         // the first key whose value row is not held, INT32_MAX: none
  static __device__ __forceinline__ int k_turn(int key) { return kC >= 16 ? key & 15 : (key >> 1) & 7; }
  static __device__ __forceinline__ int v_turn(int key) { return kC >= 16 ? 4 * (key & 3) : 4 * ((key >> 1) & 1); }
};

template <typename T>
__device__ __forceinline__ T load_global(uint64_t at) {  // which a pointer that may be the zeros' would not be seen to be
  return *reinterpret_cast<const __attribute__((address_space(1))) T*>(at);
}

template <typename E, typename Q, int kDP, int kKeys, bool kLse, bool kPrefix>
__global__ void __launch_bounds__(kThreads, kDP == 256 ? 1 : 2) prompt8_kernel(PromptParams p) {
  typedef Shared8<kDP, kKeys> S;
  constexpr int kKeyBlocks = kKeys / 32, kSteps = kDP / 16, kBlocks = kDP / 32;
  constexpr int kPieces = kDP / 16, kLoads = kKeys * kPieces / kThreads, kRowsLoad = kThreads / kPieces;  // 16 codes a piece
  constexpr uint32_t kRow = kDP * 2;
  __shared__ S sm;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid >> 6), l32 = lane & 31, h = lane >> 5;
  const int hk = blockIdx.x % p.Hkv;
  const Item it = find_item<true, kPrefix>(p, blockIdx.x / p.Hkv, lane);
  if (it.b < 0) return;
  const int tile = it.tile, n = it.n, m = it.m;
  const int32_t* pages = p.cache.pages + it.b * p.cache.pages_stride;

  // This lane's row, and how many keys it sees.
  const int all = n * p.G, row0 = tile * kRowsTile, w0 = row0 + wave * kRowsWave;
  int vis, end, wave_all, wave_any;
  if constexpr (kPrefix) {
    vis = prefix_seen(p, m, w0 + l32);
    end = m;
    wave_all = least_of(vis);
    wave_any = w0 < all ? -least_of(-vis) : 0;
  } else {
    vis = keys_seen(p, n, m, w0 + l32);
    end = uniform(keys_seen(p, n, m, row0 + kRowsTile - 1));  // keys that some row sees
    wave_all = uniform(keys_seen(p, n, m, w0));               // that every row of the wave sees
    wave_any = uniform(w0 < all ? keys_seen(p, n, m, w0 + kRowsWave - 1) : 0);
  }
  // This item's keys, and whether they are all of the unit's.
  const int begin = it.part ? it.part * it.chunk : 0;
  if (begin > 0 && begin >= end) return;
  const int stop = begin + min(end - begin, it.chunk);
  const bool whole_unit = !kPrefix && begin == 0 && stop == end;

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

  // Loading: load i of a thread is piece tid % kPieces of row tid / kPieces + i kRowsLoad.  Eight rows from a multiple of eight share a page, so
  // a wave's rows of a load lie behind one wave-uniform address (two at D = 64), and what a lane adds to it never changes; every lane's
  // address worked out by itself was a third of the vector instructions that this kernel had beyond the 16-bit one's.  Lane g holds the
  // page of rows 8 g .. and where in it they are, looked up a tile before; lane l of the first wave takes the scales of row l.
  constexpr int kRowsHere = kWave / kPieces, kGroups = kRowsHere > 8 ? 2 : 1;
  const int piece = tid % kPieces, lrow = tid / kPieces, in_group = lrow & 7;
  const int64_t lane_k = in_group * p.cache.k_row + 16 * piece, lane_v = in_group * p.cache.v_row + 16 * piece;
  const uint64_t kbase = reinterpret_cast<uint64_t>(p.cache.k + hk * p.cache.k_head), vbase = reinterpret_cast<uint64_t>(p.cache.v + hk * p.cache.v_head);
  const uint64_t kscale = reinterpret_cast<uint64_t>(p.scales.k + hk * p.scales.k_head), vscale = reinterpret_cast<uint64_t>(p.scales.v + hk * p.scales.v_head);
  const bool exact = p.D == kDP;
  u32x4 raw_k[kLoads], raw_v[kLoads];
  float scale_v[kLoads], raw_ks = 0.f, raw_vs = 0.f;
  uint32_t group_page, group_off;
  uint64_t exists_next = 0;
  auto find_pages = [&](int kt) {
    const int key = kt + 8 * lane;
    const uint32_t slot = p.cache.by_page.of(key);
    group_page = lane < kKeys / 8 && key < stop ? static_cast<uint32_t>(pages[slot]) : 0xFFFFFFFFu;
    group_off = key - slot * p.cache.page_size;
  };
  auto load = [&](int kt) {
    const uint64_t zero = reinterpret_cast<uint64_t>(kZeroRow);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      uint64_t k[kGroups], v[kGroups], sc[kGroups];
      bool there[kGroups];
#pragma unroll
      for (int j = 0; j < kGroups; ++j) {
        const int g = (wave * kRowsHere + i * kRowsLoad) / 8 + j;
        const uint32_t page = __builtin_amdgcn_readlane(group_page, g), off = __builtin_amdgcn_readlane(group_off, g);
        k[j] = kbase + page * p.cache.k_page + off * p.cache.k_row;
        v[j] = vbase + page * p.cache.v_page + off * p.cache.v_row;
        sc[j] = vscale + page * p.scales.v_page + 4 * off;
        there[j] = page < p.cache.n_pages;
      }
      const bool second = kGroups > 1 && lane >= 32;
      uint64_t ka = (second ? k[kGroups - 1] : k[0]) + lane_k, va = (second ? v[kGroups - 1] : v[0]) + lane_v;
      uint64_t sa = (second ? sc[kGroups - 1] : sc[0]) + 4 * in_group;
      if (!(exact && there[0] && there[kGroups - 1] && kt + kKeys <= stop)) {
        const bool ok = (second ? there[kGroups - 1] : there[0]) && 16 * piece < p.D && kt + lrow + i * kRowsLoad < stop;
        ka = ok ? ka : zero;
        va = ok ? va : zero;
        sa = ok ? sa : zero;
      }
      raw_k[i] = load_global<u32x4>(ka);
      raw_v[i] = load_global<u32x4>(va);
      scale_v[i] = load_global<float>(sa);
    }
    const uint32_t page = __builtin_amdgcn_ds_bpermute(4 * (lane >> 3), group_page);
    const bool there = page < p.cache.n_pages && lane < kKeys && kt + lane < stop;
    exists_next = __ballot(there);
    if (wave == 0) {
      const uint32_t off = __builtin_amdgcn_ds_bpermute(4 * (lane >> 3), group_off) + (lane & 7);
      raw_ks = load_global<float>(there ? kscale + page * p.scales.k_page + 4 * off : zero);
      raw_vs = load_global<float>(there ? vscale + page * p.scales.v_page + 4 * off : zero);
    }
  };
  const uint32_t lds_k = lds_addr(sm.k[0][0]), lds_v = lds_addr(sm.v[0][0]);
  // What was loaded into buffer buf, a half of a piece at a time: keys' halves, then values'.
  constexpr int kHalves = 4 * kLoads;
  auto store_half = [&](int buf, int half) {
    const int i = half / 2 % kLoads, j = half % 2, row = lrow + i * kRowsLoad;
    if (half < kHalves / 2)
      lds_st(lds_k + buf * S::kTile + row * kRow + 16 * ((2 * piece + j) ^ S::k_turn(row)), convert8<E, Q>(raw_k[i][2 * j], raw_k[i][2 * j + 1]));
    else
      lds_st(lds_v + buf * S::kTile + row * kRow + 16 * ((2 * piece + j) ^ S::v_turn(row)),
             convert_value8<E, Q>(raw_v[i][2 * j], raw_v[i][2 * j + 1], Split<E, Q>::power(scale_v[i])));
  };
  auto store_scales = [&](int buf) {
    if (wave == 0 && lane < kKeys) {
      // The key of a value row that is not held counts in the sums as any other; the rows that see it, and no others, are divided by a NaN.
      const bool is = held<E, Q>(raw_vs);
      const int bad = __ffsll(__ballot(!is)) - 1;
      if (lane == 0) sm.bad[buf] = bad < 0 ? INT32_MAX : bad;
      const float f = is ? Split<E, Q>::rest(raw_vs) : 1.f, over = 1.f / f;
      sm.ks[buf][lane] = raw_ks * p.scale_log2;
      sm.add[buf][lane] = __log2f(f);
      if constexpr (kLse) sm.whole[buf][lane] = over;
      const uint32_t hi = pack2<E>(over, 0.f);
      const uint32_t lo = pack2<E>(over - unpack_lo<E>(hi), 0.f);
      uint16_t* to = reinterpret_cast<uint16_t*>(&sm.over[buf][lane >> 2]) + (lane & 3);
      to[0] = static_cast<uint16_t>(hi);
      to[4] = static_cast<uint16_t>(lo);
    }
  };

  // Lane parts of the operands' LDS addresses, as in the 16-bit kernel.
  const uint32_t kat = lds_k + l32 * kRow + 16 * (h ^ S::k_turn(l32));
  const int i16 = lane & 15, vrow = 4 * h + (i16 >> 2);
  const uint32_t vat = lds_v + vrow * kRow + 16 * ((2 * ((lane >> 4) & 1) + ((i16 & 3) >> 1)) ^ S::v_turn(vrow)) + 8 * (i16 & 1);

  f32x16 acc[kBlocks];
#pragma unroll
  for (int i = 0; i < kBlocks; ++i) acc[i] = f32x16{};
  // top: what the exponentials are taken against, within kSlack of the largest weight.  The row is divided by the sum of the probabilities that the
  // rounded weights of its values stand for, so that their roundings cancel as far as they agree (a row of one key is that key's
  // value); the log-sum-exp, where it is asked for, takes the sum of the unrounded ones.
  float top = -INFINITY, sum = 0.f, full = 0.f;
  uint64_t exists_now = 0;

  auto step = [&](int kt, auto bufc) {
    constexpr int buf = decltype(bufc)::value;
    constexpr uint64_t kAll = ~uint64_t{0} >> (64 - kKeys);
    lds_barrier();  // this tile is there, the other buffer read
    const uint64_t exists = exists_now & kAll;
    const bool more = kt + kKeys < stop, busy = kt < wave_any;
    auto follow = [&] {  // what the stores left free takes the tile after the next
      store_scales(buf ^ 1);
      exists_now = exists_next;
      if (kt + 2 * kKeys < stop) {
        load(kt + 2 * kKeys);
        find_pages(kt + 3 * kKeys);
      }
    };
    if (!busy) {  // the other waves' rows see this tile
      if (more) {
#pragma unroll
        for (int half = 0; half < kHalves; ++half) store_half(buf ^ 1, half);
        follow();
      }
      return;
    }
    if (uniform(sm.bad[buf]) < vis - kt) sum = __uint_as_float(0x7FC00000u);  // for the rows that see a value row that is not held
    // Scores; the next tile's codes are converted in the products' shadow (two prompts of 4099 behind 8 and 5701: 1005 us, 1031 before them).
    f32x16 s[kKeyBlocks] = {};
    auto scores = [&](auto converting) {
#pragma unroll
      for (int st = 0; st < kSteps; ++st) {
#pragma unroll
        for (int blk = 0; blk < kKeyBlocks; ++blk) s[blk] = E::mfma32(lds_ld<u32x4>((kat ^ (32 * st)) + buf * S::kTile + blk * 32 * kRow), q[st], s[blk]);
        if constexpr (decltype(converting)::value) {
          if (st < kHalves) store_half(buf ^ 1, st);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if constexpr (decltype(converting)::value) {
#pragma unroll
        for (int half = kSteps; half < kHalves; ++half) store_half(buf ^ 1, half);
        follow();
      }
    };
    more ? scores(std::true_type{}) : scores(std::false_type{});
    __builtin_amdgcn_sched_barrier(0);
    const uint32_t ks_at = lds_addr(sm.ks[buf][0]) + 16 * h, add_at = lds_addr(sm.add[buf][0]) + 16 * h, over_at = lds_addr(sm.over[buf][0]) + 16 * h;
#pragma unroll
    for (int blk = 0; blk < kKeyBlocks; ++blk)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 f = lds_ld<f32x4>(ks_at + 4 * (32 * blk + 8 * g)), add = lds_ld<f32x4>(add_at + 4 * (32 * blk + 8 * g));
#pragma unroll
        for (int r = 0; r < 4; ++r) s[blk][4 * g + r] = __builtin_fmaf(s[blk][4 * g + r], f[r], add[r]);
      }
    if (!(kt + kKeys <= wave_all && exists == kAll)) {
      asm volatile("");  // keeps this a branch: most tiles need none of it
      const int left = vis - kt - 4 * h;  // of the keys from this lane's first on
      const uint64_t there = exists >> (4 * h);
#pragma unroll
      for (int blk = 0; blk < kKeyBlocks; ++blk)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = 32 * blk + 8 * (r >> 2) + (r & 3);
          const uint32_t half = static_cast<uint32_t>(there >> (32 * blk));
          if (key >= left || !(half & (1u << (key & 31)))) s[blk][r] = -INFINITY;
        }
    }
    float m2[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int r = 0; r < 16; ++r)
#pragma unroll
      for (int blk = 0; blk < kKeyBlocks; ++blk) m2[kKeyBlocks == 1 ? r & 1 : blk] = fmaxf(m2[kKeyBlocks == 1 ? r & 1 : blk], s[blk][r]);
    const float t2 = op_over(fmaxf(m2[0], m2[1]), 32, 64, OpMax{});
    if (__any(t2 > top + Scale<E>::kSlack)) {
      const float up = fmaxf(top, t2), f = exp2_fast(top - finite_max(up));
      top = up;
      sum *= f;
      full *= f;
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) acc[i] *= f;
    }
    const float mm = finite_max(top) - Scale<E>::kUp;
    float part[2] = {sum, 0.f}, part_full[2] = {full, 0.f};
    u32x4 prob[2 * kKeyBlocks];
#pragma unroll
    for (int kk = 0; kk < 2 * kKeyBlocks; ++kk)
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const u32x4 over = lds_ld<u32x4>(over_at + 4 * (16 * kk + 8 * g));
        f32x4 whole{};
        if constexpr (kLse) whole = lds_ld<f32x4>(lds_addr(sm.whole[buf][0]) + 16 * h + 4 * (16 * kk + 8 * g));
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          const float x = exp2_fast(s[kk >> 1][8 * (kk & 1) + 4 * g + 2 * a] - mm), y = exp2_fast(s[kk >> 1][8 * (kk & 1) + 4 * g + 2 * a + 1] - mm);
          const uint32_t w = pack2<E>(x, y);
          prob[kk][2 * g + a] = w;
          part[a] = E::dot2(w, over[2 + a], E::dot2(w, over[a], part[a]));
          if constexpr (kLse) {
            part_full[0] += x * whole[2 * a];
            part_full[1] += y * whole[2 * a + 1];
          }
        }
      }
    sum = part[0] + part[1];
    if constexpr (kLse) full = part_full[0] + part_full[1];
#pragma unroll
    for (int kk = 0; kk < 2 * kKeyBlocks; ++kk)  // 16 keys
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) {
        const uint32_t at = (vat ^ (64 * i)) + buf * S::kTile + 16 * kk * kRow;
        const u32x2 lo = read_transposed(at), hi = read_transposed(at + 8 * kRow);
        acc[i] = E::mfma32(u32x4{lo[0], lo[1], hi[0], hi[1]}, prob[kk], acc[i]);
      }
  };

  if (begin < stop) {
    find_pages(begin);
    load(begin);
    find_pages(begin + kKeys);
#pragma unroll
    for (int half = 0; half < kHalves; ++half) store_half(0, half);
    store_scales(0);
    exists_now = exists_next;
    if (begin + kKeys < stop) {
      load(begin + kKeys);
      find_pages(begin + 2 * kKeys);
    }
    for (int kt = begin; kt < stop; kt += 2 * kKeys) {
      step(kt, std::integral_constant<int, 0>{});
      if (kt + kKeys < stop) step(kt + kKeys, std::integral_constant<int, 1>{});
    }
  }

  sum = op_over(sum, 32, 64, OpAdd{});
  if constexpr (kLse) full = op_over(full, 32, 64, OpAdd{});
  const int row = w0 + l32;
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
#pragma unroll
  for (int i = 0; i < kBlocks; ++i)
#pragma unroll
    for (int rr = 0; rr < 4; ++rr) {
      const int d = 32 * i + 8 * rr + 4 * h;
      if (d < p.D)
        store4<E>(p, it.s0 + tok, head, d, acc[i][4 * rr] * inv, acc[i][4 * rr + 1] * inv, acc[i][4 * rr + 2] * inv, acc[i][4 * rr + 3] * inv);
    }
  if constexpr (kLse) {
    if (h == 0) store_lse<E>(p, it.s0 + tok, head, top, full);
  }
}

template <bool kPrefix>
int launch8(const latent_attn_prompt_args& a, int32_t code, const Plan& pl, const PromptParams& p, hipStream_t s) {
  (void)hipGetLastError();
  auto go = [&](auto e, auto q, auto dp) {
    constexpr int kDP = decltype(dp)::value;
    using E = decltype(e);
    // Split units have less than pl.items parts beyond their first.
    const int64_t more = (pl.items / p.Hkv + 1) * p.Hkv, units = std::max<int64_t>(pl.units, p.Hkv);
    auto with_lse = [&](auto lse) {
      constexpr bool kLse = decltype(lse)::value;
      hipLaunchKernelGGL((prompt8_kernel<E, decltype(q), kDP, kDP == 256 ? 32 : 64, kLse, kPrefix>),
                         dim3(static_cast<unsigned>(kPrefix ? p.max_parts : units + (p.max_parts ? more : 0))), dim3(kThreads), 0, s, p);
      if (!kPrefix && p.max_parts)
        hipLaunchKernelGGL((join_kernel<E, kDP, true, kLse>), dim3(static_cast<unsigned>(std::min(units, more)), kDP / 32), dim3(kThreads), 0, s, p);
    };
    if constexpr (kPrefix)
      with_lse(std::true_type{});
    else
      p.lse ? with_lse(std::true_type{}) : with_lse(std::false_type{});
  };
  using std::integral_constant;
  auto dims = [&](auto e, auto q) {
    p.D <= 64 ? go(e, q, integral_constant<int, 64>{}) : p.D <= 128 ? go(e, q, integral_constant<int, 128>{}) : go(e, q, integral_constant<int, 256>{});
  };
  auto codes = [&](auto e) { code == LATENT_CODE_INT8 ? dims(e, Int8{}) : dims(e, E4M3{}); };
  a.dtype == LATENT_F16 ? codes(F16{}) : codes(BF16{});
  return hipGetLastError() == hipSuccess ? LATENT_OK : LATENT_E_HIP;
}

}  // namespace

int launch_prefix8(const latent_attn_decode_args& a, const latent_kv_scales& scales, const int32_t* prefix, int64_t n_prefix, const Prior& prior, hipStream_t s) {
  const latent_attn_prompt_args r = prefix_args(a, prefix, n_prefix);
  PromptParams p{};
  const int st = prefix_params(r, 1, prior, &p);
  if (st != LATENT_OK) return st;
  p.scales = device_scales(scales);
  return launch8<true>(r, scales.code, Plan{}, p, s);
}

}  // namespace attend
}  // namespace latent

using namespace latent;
using namespace latent::attend;

extern "C" int latent_attn_prompt_q8(const latent_attn_prompt_args* args, const latent_kv_scales* scales, latent_stream_t stream) {
  if (!args || !scales) return LATENT_E_INVALID;
  const latent_attn_prompt_args& a = *args;
  if (a.k || a.n_keys) return LATENT_E_INVALID;  // keys are in the cache
  int st = validate(a);
  if (st == LATENT_OK) st = check_codes(a.cache, *scales, a.head_dim);
  if (st != LATENT_OK || a.n_tokens == 0 || a.cache.n_seq == 0) return st;
  const Plan pl = plan_for(a);
  PromptParams p{};
  st = prompt_params(a, 1, pl, &p);
  if (st != LATENT_OK) return st;
  if (p.cache.max_len && (!scales->k || !scales->v)) return LATENT_E_INVALID;
  p.scales = device_scales(*scales);
  return launch8<false>(a, scales->code, pl, p, reinterpret_cast<hipStream_t>(stream));
}
