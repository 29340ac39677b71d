// Attention of one new token a sequence over the paged cache.
//
//   out[b][h] = sum_j p_j v[j] / sum_j p_j,  p_j = exp(scale q[b][h] . k[j] - max)
//
// Bound by the cache's bytes: each key and value is read once, for all query
// heads of its head (16 of them fill a matrix instruction's columns; fewer leave
// columns idle, which costs nothing here).
//
// Work: a unit is one sequence, key/value head and chunk of its query heads; it
// is cut into tiles of 128 keys.  The launch's workgroups take equal contiguous
// spans of the list of all tiles, so one long sequence, or a batch of very
// different lengths, loads every CU alike.  Each workgroup finds its span from
// the lengths on the device.  A unit inside one span is finished there; others
// leave a part (maximum, sum, unnormalised row) per workgroup, joined by a second
// launch in workgroup order.
//
// Inside a workgroup each wave streams 32-key steps of its own, from the cache
// straight to registers, no LDS and no barrier: scores^T = K Q^T puts a query
// head in every lane column and keys in the rows, and the lane that holds
// query n and keys 8 (lane / 16) .. + 7 of the probabilities is the one whose value
// operand covers those keys.  A value row arrives as VEC = D / 16 neighbours a lane
// for eight keys; eight rows are paired into operand dwords by byte permutes.
//
// A probability is rounded to the element type for its product with the values, at most half a step of its own size; the sum
// that divides takes them unrounded, as the log-sum-exp needs it, so a row may be off by those half steps
// (in bf16 0.0018 of a row's size against 0.0017 with them in 32 bits; the output's own rounding is as much).
//
// Measured (bf16, heads of 128, 8 of them with keys): 131071 tokens 102 us (5.2 TB/s), 35 sequences of 16 to 16000
// tokens, 69502 in all, 60 us (4.8 TB/s), 64 of 10000 to 20000 656 us (5.7 TB/s); 301 tokens 7.0 us, of
// which the launch alone is 5, and 9.4 where the page table is wider than what is taken whole (kWholeTiles).
// Heads of 72 and 96: 3.8 and 4.8 TB/s (16 sequences of 12000), padded to 128 and with the usual loads.
#include "decode.hpp"

namespace latent {
namespace attend {
namespace {

template <bool kAfter, bool kTable = false>
int launch16(const latent_attn_decode_args& a, const Plan& pl, const Params<kAfter || kTable>& p, hipStream_t s) {
  (void)hipGetLastError();
  auto launch = [&](auto e, auto dp, auto exact, auto mt, auto page8) {
    auto go = [&](auto once) {
      typedef Stream<decltype(e), decltype(dp)::value, decltype(exact)::value, decltype(mt)::value, decltype(page8)::value, decltype(once)::value, kTable> S;
      hipLaunchKernelGGL((decode_kernel<S, kAfter>), dim3(pl.groups), dim3(kThreads), 0, s, p);
    };
    if constexpr (decltype(exact)::value && decltype(page8)::value)
      pl.once ? go(std::true_type{}) : go(std::false_type{});
    else
      go(std::false_type{});
  };
  using std::integral_constant;
  auto with_dim = [&](auto e, auto dp) {
    const bool exact = p.D == static_cast<uint32_t>(decltype(dp)::value);
    auto with_mt = [&](auto mt) {
      if (a.cache.page_size % 8)
        launch(e, dp, std::false_type{}, mt, std::false_type{});
      else if (exact)
        launch(e, dp, std::true_type{}, mt, std::true_type{});
      else
        launch(e, dp, std::false_type{}, mt, std::true_type{});
    };
    pl.mt == 1 ? with_mt(integral_constant<int, 1>{}) : with_mt(integral_constant<int, 2>{});
  };
  auto with_type = [&](auto e) {
    if (p.D <= 64)
      with_dim(e, integral_constant<int, 64>{});
    else if (p.D <= 128)
      with_dim(e, integral_constant<int, 128>{});
    else
      with_dim(e, integral_constant<int, 256>{});
  };
  const bool f16 = a.dtype == LATENT_F16;
  f16 ? with_type(F16{}) : with_type(BF16{});
  if (hipGetLastError() != hipSuccess) return LATENT_E_HIP;
  launch_join<kAfter>(pl, p, f16, s);
  return hipGetLastError() == hipSuccess ? LATENT_OK : LATENT_E_HIP;
}

}  // namespace

size_t after_workspace(const latent_attn_decode_args& a, int64_t n_prefix, bool codes) {
  return plan_after(behind(a, n_prefix), codes ? 1 : 2, codes ? kMaxGroups8 : kMaxGroups).all();
}

int launch_after16(const latent_attn_decode_args& a, int64_t n_prefix, const Prior& prior, void* workspace, hipStream_t s) {
  const After w = plan_after(behind(a, n_prefix), 2, kMaxGroups);
  MoreParams p{};
  const int st = after_params(a, n_prefix, 2, w, prior, workspace, &p);
  return st == LATENT_OK ? launch16<true>(a, w.plan, p, s) : st;
}

int launch_together16(const latent_attn_decode_args& a, const int32_t* prefix, int64_t n_prefix, hipStream_t s) {
  const Plan pl = plan_for(a);
  MoreParams p{};
  const int st = decode_params(a, 2, pl, &p);
  if (st != LATENT_OK) return st;
  p.prefix = prefix;
  p.prefix_pages = static_cast<uint32_t>(n_prefix);
  return launch16<false, true>(a, pl, p, s);
}

}  // namespace attend
}  // namespace latent

using namespace latent;
using namespace latent::attend;

extern "C" int latent_attn_decode_workspace_size(const latent_attn_decode_args* args, size_t* bytes) {
  if (!args || !bytes) return LATENT_E_INVALID;
  const int st = validate(*args);
  if (st != LATENT_OK) return st;
  const Plan pl = plan_for(*args);
  *bytes = pl.ml_bytes + pl.acc_bytes + pl.unit_bytes;
  return LATENT_OK;
}

extern "C" int latent_attn_decode(const latent_attn_decode_args* args, latent_stream_t stream) {
  if (!args) return LATENT_E_INVALID;
  const latent_attn_decode_args& a = *args;
  int st = validate(a);
  if (st != LATENT_OK || a.cache.n_seq == 0) return st;
  const Plan pl = plan_for(a);
  DecodeParams p{};
  st = decode_params(a, 2, pl, &p);
  if (st != LATENT_OK) return st;
  return launch16<false>(a, pl, p, reinterpret_cast<hipStream_t>(stream));
}
