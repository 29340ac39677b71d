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
#include "prompt.hpp"

namespace latent {
namespace attend {
namespace {

// 0xFFFF in the places of a dword's infinities and NaN.
template <typename E>
__device__ __forceinline__ uint32_t nonfinite(uint32_t w) {
  constexpr uint32_t kExp = __is_same(E, F16) ? 0x7C00u : 0x7F80u;
  return ((w & kExp) == kExp ? 0xFFFFu : 0u) | ((w >> 16 & kExp) == kExp ? 0xFFFF0000u : 0u);
}

template <typename E, int kDP, int kKeys, bool kPaged, bool kLse, bool kPrefix>
__global__ void __launch_bounds__(kThreads, kDP == 256 ? 1 : 2) prompt_kernel(PromptParams p) {
  typedef Shared<kDP, kKeys> S;
  constexpr int kKeyBlocks = kKeys / 32, kC = S::kC, kSteps = kDP / 16, kBlocks = kDP / 32;
  constexpr int kRowsLoad = kWave / kC, kLoads = kKeys / kWaves / kRowsLoad;  // rows of a direct load; loads of a wave and tile
  constexpr uint32_t kRow = kDP * 2;
  __shared__ S sm;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid >> 6), l32 = lane & 31, h = lane >> 5;
  const int hk = blockIdx.x % p.Hkv;
  const Item it = find_item<kPaged, kPrefix>(p, blockIdx.x / p.Hkv, lane);
  if (it.b < 0) return;
  const int b = it.b, tile = it.tile, n = it.n, m = it.m;
  const int32_t* pages = kPaged ? p.cache.pages + b * p.cache.pages_stride : nullptr;
  const char* kbase = p.cache.k + hk * p.cache.k_head + it.k0 * p.cache.k_row;
  const char* vbase = p.cache.v + hk * p.cache.v_head + it.k0 * p.cache.v_row;

  // This lane's row, and how many keys it sees.
  const int all = n * p.G, row0 = tile * kRowsTile, w0 = row0 + wave * kRowsWave;
  int vis, all_see, end, wave_all, wave_any;
  if constexpr (kPrefix) {
    vis = prefix_seen(p, m, w0 + l32);
    all_see = least_of(min(prefix_seen(p, m, row0 + lane), prefix_seen(p, m, row0 + kWave + lane)));
    end = m;
    wave_all = least_of(vis);
    wave_any = w0 < all ? -least_of(-vis) : 0;
  } else {
    vis = keys_seen(p, n, m, w0 + l32);
    all_see = uniform(keys_seen(p, n, m, row0));              // keys that every row of the workgroup sees
    end = uniform(keys_seen(p, n, m, row0 + kRowsTile - 1));  // keys that some row sees
    wave_all = uniform(keys_seen(p, n, m, w0));               // of the wave
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
int launch16(const latent_attn_prompt_args& a, const Plan& pl, const PromptParams& p, hipStream_t s) {
  (void)hipGetLastError();
  auto launch = [&](auto e, auto dp) {
    constexpr int kDP = decltype(dp)::value;
    using E = decltype(e);
    // Split units have less than pl.items parts beyond their first.
    const int64_t more = (pl.items / p.Hkv + 1) * p.Hkv, units = std::max<int64_t>(pl.units, p.Hkv);
    auto go = [&](auto paged_c, auto lse_c) {
      constexpr bool kPaged = decltype(paged_c)::value, kLse = decltype(lse_c)::value;
      const dim3 grid(static_cast<unsigned>(kPrefix ? p.max_parts : units + (p.max_parts ? more : 0)));
      hipLaunchKernelGGL((prompt_kernel<E, kDP, kDP == 256 ? 32 : 64, kPaged, kLse, kPrefix>), grid, dim3(kThreads), 0, s, p);
      if (!kPrefix && p.max_parts)
        hipLaunchKernelGGL((join_kernel<E, kDP, kPaged, kLse>), dim3(static_cast<unsigned>(std::min(units, more)), kDP / 32),
                           dim3(kThreads), 0, s, p);
    };
    if constexpr (kPrefix) {
      go(std::true_type{}, std::true_type{});
    } else {
      auto with_lse = [&](auto paged_c) { p.lse ? go(paged_c, std::true_type{}) : go(paged_c, std::false_type{}); };
      !a.k ? with_lse(std::true_type{}) : with_lse(std::false_type{});
    }
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

}  // namespace

// As many items of a row tile and key/value head as the chip holds at once (one workgroup a CU above D = 128), of 256 keys at least.
PriorBytes plan_prior(const latent_attn_decode_args& a, int64_t n_prefix, Prior* prior) {
  const int64_t rows = a.cache.n_seq * (a.n_head / a.n_kv_head), keys = n_prefix * a.cache.page_size;
  const int64_t tiles = (rows + kRowsTile - 1) / kRowsTile, units = std::max<int64_t>(1, tiles * a.n_kv_head);
  const int64_t most = std::max<int64_t>(1, (a.head_dim > 128 ? 256 : 512) / units), least = (keys + most - 1) / most;
  const int64_t chunk = std::max<int64_t>(kChunk, (least + kChunkStep - 1) / kChunkStep * kChunkStep);
  prior->parts = static_cast<int32_t>(std::max<int64_t>(1, a.cache.n_pages ? (keys + chunk - 1) / chunk : 0));
  prior->chunk = static_cast<int32_t>(chunk);
  prior->tiles = static_cast<int32_t>(tiles);
  prior->up = a.dtype == LATENT_F16 ? Scale<F16>::kUp : Scale<BF16>::kUp;
  const size_t parts = static_cast<size_t>(prior->parts) * units, blocks = a.head_dim <= 64 ? 2 : a.head_dim <= 128 ? 4 : 8;
  return {parts * 4 * blocks * kThreads * sizeof(f32x4), parts * kThreads * sizeof(f32x4)};
}

int launch_prefix16(const latent_attn_decode_args& a, const int32_t* prefix, int64_t n_prefix, const Prior& prior, hipStream_t s) {
  const latent_attn_prompt_args r = prefix_args(a, prefix, n_prefix);
  PromptParams p{};
  const int st = prefix_params(r, 2, prior, &p);
  return st == LATENT_OK ? launch16<true>(r, Plan{}, p, s) : st;
}

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
  int st = validate(a);
  if (st != LATENT_OK || a.n_tokens == 0 || a.cache.n_seq == 0) return st;
  const Plan pl = plan_for(a);
  PromptParams p{};
  st = prompt_params(a, 2, pl, &p);
  if (st != LATENT_OK) return st;
  return launch16<false>(a, pl, p, reinterpret_cast<hipStream_t>(stream));
}
