// Attention of prompts over an 8-bit paged cache: the 16-bit kernel's items, rows and products (prompt.hip), its tiles made from
// codes on their way to LDS.
//
//   score[j] = scale ks[j] (q . kcode[j]),   out = sum_j (p[j] vs[j]) vcode[j] / sum_j p[j]
//
// Codes are loaded a tile ahead into registers (a tile's keys and values are 64 bytes a thread at D = 128), made exact
// elements of the queries' type there and written to the LDS buffer that the waves do not read: each code is
// converted once for the four waves, and the operands' reads are the 16-bit kernel's.  The scales of a tile's keys lie in LDS beside
// it, in fp32: a key's multiplies its score; of a value's the power of two goes into the elements, exactly, and the rest multiplies
// the probability, which is rounded to the element type after it.
#include "prompt.hpp"

namespace latent {
namespace attend {
namespace {

// A value row of scale s: its codes times `power`, of two, are the elements; the probability takes `rest`, from 1 to 2.  s = power
// rest.  The elements are exact but for f16's below its normal numbers, which are as near as f16 has them.
struct Split {
  static __device__ __forceinline__ float power(float s) {
    const uint32_t e = __float_as_uint(s) & 0x7F800000u;
    return e >= 0x7F000000u ? 1.f : __uint_as_float(e);  // a NaN's codes are zeros; 0 for 0
  }
  static __device__ __forceinline__ float rest(float s) {
    const float p = power(s);
    return p == 0.f ? 1.f : s * __uint_as_float(0x7F000000u - __float_as_uint(p));
  }
};

// Sixteen codes as 32 bytes of elements, times a power of two (kScaled).
template <typename E, typename Q, bool kScaled>
__device__ __forceinline__ void convert16(const u32x4& w, float power, u32x4 (&out)[2]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    out[i >> 1][2 * (i & 1)] = kScaled ? Q::template scaled_pair<E, false>(w[i], power) : Q::template pair<E, false>(w[i]);
    out[i >> 1][2 * (i & 1) + 1] = kScaled ? Q::template scaled_pair<E, true>(w[i], power) : Q::template pair<E, true>(w[i]);
  }
}

template <int kDP, int kKeys>
struct Shared8 {
  static constexpr int kC = kDP / 8;
  static constexpr uint32_t kTile = kKeys * kDP * 2;
  alignas(512) u32x4 k[2][kKeys * kC];
  u32x4 v[2][kKeys * kC];
  float ks[2][kKeys], vs[2][kKeys], over[2][kKeys];  // a score's factor, base 2; a probability's, and one over it
  static __device__ __forceinline__ int k_turn(int key) { return kC >= 16 ? key & 15 : (key >> 1) & 7; }
  static __device__ __forceinline__ int v_turn(int key) { return kC >= 16 ? 4 * (key & 3) : 4 * ((key >> 1) & 1); }
};

template <typename E, typename Q, int kDP, int kKeys, bool kLse, bool kPrefix>
__global__ void __launch_bounds__(kThreads, kDP == 256 ? 1 : 2) prompt8_kernel(PromptParams p) {
  typedef Shared8<kDP, kKeys> S;
  constexpr int kKeyBlocks = kKeys / 32, kSteps = kDP / 16, kBlocks = kDP / 32;
  constexpr int kPieces = kDP / 16, kLoads = kKeys * kPieces / kThreads, kRowsLoad = kThreads / kPieces;  // 16 codes a piece
  constexpr uint32_t kRow = kDP * 2;
  constexpr float kRoom = E::kLift != 0.f ? 1.f : 0.f;  // for Split's rest, below two: probabilities are taken so much (log2) lower
  __shared__ S sm;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid >> 6), l32 = lane & 31, h = lane >> 5;
  const int hk = blockIdx.x % p.Hkv;
  const Item it = find_item<true, kPrefix>(p, blockIdx.x / p.Hkv, lane);
  if (it.b < 0) return;
  const int tile = it.tile, n = it.n, m = it.m;
  const int32_t* pages = p.cache.pages + it.b * p.cache.pages_stride;
  const char* kbase = p.cache.k + hk * p.cache.k_head;
  const char* vbase = p.cache.v + hk * p.cache.v_head;
  const char* kscale = p.scales.k + hk * p.scales.k_head;
  const char* vscale = p.scales.v + hk * p.scales.v_head;

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

  // Loading: load i of a thread is piece tid % kPieces of row tid / kPieces + i kRowsLoad, and lane l of the first two waves has the
  // key's and the value's scale of row l.  Pages are looked up a tile before.
  const int piece = tid % kPieces, lrow = tid / kPieces;
  u32x4 raw_k[kLoads], raw_v[kLoads];
  float scale_v[kLoads], raw_scale = 0.f;
  uint32_t piece_page[kLoads], lane_page;
  uint64_t exists_next = 0;
  auto find_pages = [&](int kt) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int key = kt + lrow + i * kRowsLoad;
      piece_page[i] = key < stop ? static_cast<uint32_t>(pages[p.cache.by_page.of(key)]) : 0xFFFFFFFFu;
    }
    const int key = kt + lane;
    lane_page = lane < kKeys && key < stop ? static_cast<uint32_t>(pages[p.cache.by_page.of(key)]) : 0xFFFFFFFFu;
  };
  auto load = [&](int kt) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const uint32_t key = kt + lrow + i * kRowsLoad, off = key - p.cache.by_page.of(key) * p.cache.page_size, page = piece_page[i];
      const bool ok = page < p.cache.n_pages && 16 * piece < p.D;
      const char* zero = reinterpret_cast<const char*>(kZeroRow);
      raw_k[i] = *reinterpret_cast<const u32x4*>(ok ? kbase + page * p.cache.k_page + off * p.cache.k_row + 16 * piece : zero);
      raw_v[i] = *reinterpret_cast<const u32x4*>(ok ? vbase + page * p.cache.v_page + off * p.cache.v_row + 16 * piece : zero);
      scale_v[i] = *reinterpret_cast<const float*>(ok ? vscale + page * p.scales.v_page + 4 * off : zero);
    }
    const bool there = lane_page < p.cache.n_pages;
    exists_next = __ballot(there);
    if (wave < 2) {
      const uint32_t key = kt + lane, off = key - p.cache.by_page.of(key) * p.cache.page_size;
      const char* at = wave == 0 ? kscale + lane_page * p.scales.k_page : vscale + lane_page * p.scales.v_page;
      raw_scale = *reinterpret_cast<const float*>(there ? at + 4 * off : reinterpret_cast<const char*>(kZeroRow));
    }
  };
  const uint32_t lds_k = lds_addr(sm.k[0][0]), lds_v = lds_addr(sm.v[0][0]);
  auto store = [&](int buf) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int row = lrow + i * kRowsLoad;
      u32x4 x[2];
      convert16<E, Q, false>(raw_k[i], 1.f, x);
#pragma unroll
      for (int j = 0; j < 2; ++j) lds_st(lds_k + buf * S::kTile + row * kRow + 16 * ((2 * piece + j) ^ S::k_turn(row)), x[j]);
      convert16<E, Q, true>(raw_v[i], Split::power(scale_v[i]), x);
#pragma unroll
      for (int j = 0; j < 2; ++j) lds_st(lds_v + buf * S::kTile + row * kRow + 16 * ((2 * piece + j) ^ S::v_turn(row)), x[j]);
    }
    if (lane < kKeys && wave < 2) {
      if (wave == 0) {
        sm.ks[buf][lane] = raw_scale * p.scale_log2;
      } else {
        const float f = Split::rest(raw_scale);
        sm.vs[buf][lane] = f;
        sm.over[buf][lane] = f > 0.f ? 1.f / f : 0.f;
      }
    }
  };

  // Lane parts of the operands' LDS addresses, as in the 16-bit kernel.
  const uint32_t kat = lds_k + l32 * kRow + 16 * (h ^ S::k_turn(l32));
  const int i16 = lane & 15, vrow = 4 * h + (i16 >> 2);
  const uint32_t vat = lds_v + vrow * kRow + 16 * ((2 * ((lane >> 4) & 1) + ((i16 & 3) >> 1)) ^ S::v_turn(vrow)) + 8 * (i16 & 1);

  f32x16 acc[kBlocks];
#pragma unroll
  for (int i = 0; i < kBlocks; ++i) acc[i] = f32x16{};
  // top: what the exponentials are taken against, within kSlack of the maximum.  The row is divided by the sum of the probabilities that the
  // rounded weights of its values stand for, so that their roundings cancel as far as they agree (a row of one key is that key's
  // value); the log-sum-exp, where it is asked for, takes the sum of the unrounded ones.
  float top = -INFINITY, sum = 0.f, full = 0.f;
  uint64_t exists_now = 0;

  auto step = [&](int kt, auto bufc) {
    constexpr int buf = decltype(bufc)::value;
    constexpr uint64_t kAll = ~uint64_t{0} >> (64 - kKeys);
    lds_barrier();  // this tile is there, the other buffer read
    const uint64_t exists = exists_now & kAll;
    if (kt + kKeys < stop) {
      store(buf ^ 1);
      exists_now = exists_next;
      if (kt + 2 * kKeys < stop) {
        load(kt + 2 * kKeys);
        find_pages(kt + 3 * kKeys);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if (kt >= wave_any) return;  // the other waves' rows see this tile
    f32x16 s[kKeyBlocks] = {};
#pragma unroll
    for (int st = 0; st < kSteps; ++st)
#pragma unroll
      for (int blk = 0; blk < kKeyBlocks; ++blk) s[blk] = E::mfma32(lds_ld<u32x4>((kat ^ (32 * st)) + buf * S::kTile + blk * 32 * kRow), q[st], s[blk]);
    const uint32_t ks_at = lds_addr(sm.ks[buf][0]) + 16 * h, vs_at = lds_addr(sm.vs[buf][0]) + 16 * h, over_at = lds_addr(sm.over[buf][0]) + 16 * h;
#pragma unroll
    for (int blk = 0; blk < kKeyBlocks; ++blk)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 f = lds_ld<f32x4>(ks_at + 4 * (32 * blk + 8 * g));
#pragma unroll
        for (int r = 0; r < 4; ++r) s[blk][4 * g + r] *= f[r];
      }
    const bool part_seen = !(kt + kKeys <= wave_all && exists == kAll);
    if (part_seen) {
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
    const float mm = finite_max(top) - Scale<E>::kUp + kRoom;
    float part[2] = {sum, 0.f}, part_full[2] = {full, 0.f};
    u32x4 prob[2 * kKeyBlocks];
#pragma unroll
    for (int kk = 0; kk < 2 * kKeyBlocks; ++kk)
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const f32x4 f = lds_ld<f32x4>(vs_at + 4 * (16 * kk + 8 * g)), over = lds_ld<f32x4>(over_at + 4 * (16 * kk + 8 * g));
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          float x[2];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            x[r] = exp2_fast(s[kk >> 1][8 * (kk & 1) + 4 * g + 2 * a + r] - mm);
            if constexpr (kLse) part_full[r] += x[r];
            // A row that does not see a key takes nothing of it, whatever its scale (a NaN, for a row that held one).
            x[r] = part_seen && x[r] == 0.f ? 0.f : x[r] * f[2 * a + r];
          }
          const uint32_t w = pack2<E>(x[0], x[1]);
          prob[kk][2 * g + a] = w;
          part[0] += unpack_lo<E>(w) * over[2 * a];
          part[1] += unpack_hi<E>(w) * over[2 * a + 1];
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
    store(0);
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
  top += kRoom;  // as if taken against that, with the 16-bit kernel's factor
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
        store4<E, kPrefix>(p, it.s0 + tok, head, d, acc[i][4 * rr] * inv, acc[i][4 * rr + 1] * inv, acc[i][4 * rr + 2] * inv, acc[i][4 * rr + 3] * inv);
    }
  if constexpr (kLse) {
    if (h == 0) store_lse<E, kPrefix>(p, it.s0 + tok, head, top, full);
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
                         dim3(static_cast<unsigned>(units + (p.max_parts ? more : 0))), dim3(kThreads), 0, s, p);
      if (p.max_parts)
        hipLaunchKernelGGL((join_kernel<E, kDP, true, kLse, kPrefix>), dim3(static_cast<unsigned>(std::min(units, more)), kDP / 32), dim3(kThreads), 0, s, p);
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

int launch_prefix8(const latent_attn_decode_args& a, const latent_kv_scales& scales, const int32_t* prefix, int64_t n_prefix, const Prior& prior,
                   void* workspace, hipStream_t s) {
  latent_attn_prompt_args r = prefix_args(a, prefix, n_prefix);
  r.workspace = workspace;
  r.workspace_bytes = SIZE_MAX;
  const Plan pl = plan_for(r);
  PromptParams p{};
  const int st = prefix_params(r, 1, pl, prior, &p);
  if (st != LATENT_OK) return st;
  p.scales = device_scales(scales);
  return launch8<true>(r, scales.code, pl, p, s);
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
