// Attention of one new token a sequence over an 8-bit paged cache: the 16-bit kernel's units, spans and joins (decode.hip) over
// a stream of codes (decode8.hpp).
#include "decode8.hpp"

namespace latent {
namespace attend {
namespace {

template <bool kAfter, bool kTable = false>
int launch8(const latent_attn_decode_args& a, int32_t code, const Plan& pl, const MoreParams& p, hipStream_t s) {
  (void)hipGetLastError();
  with_stream8<kTable>(a, code, pl, [&](auto t) {
    hipLaunchKernelGGL((decode_kernel<typename decltype(t)::type, kAfter>), dim3(pl.groups), dim3(kThreads), 0, s, p);
  });
  if (hipGetLastError() != hipSuccess) return LATENT_E_HIP;
  launch_join<kAfter>(pl, p, a.dtype == LATENT_F16, s);
  return hipGetLastError() == hipSuccess ? LATENT_OK : LATENT_E_HIP;
}

}  // namespace

int launch_after8(const latent_attn_decode_args& a, const latent_kv_scales& scales, int64_t n_prefix, const Prior& prior, void* workspace, hipStream_t s) {
  const After w = plan_after(behind(a, n_prefix), 1, kMaxGroups8);
  MoreParams p{};
  const int st = after_params(a, n_prefix, 1, w, prior, workspace, &p);
  if (st != LATENT_OK) return st;
  p.scales = device_scales(scales);
  return launch8<true>(a, scales.code, w.plan, p, s);
}

int launch_together8(const latent_attn_decode_args& a, const latent_kv_scales& scales, const int32_t* prefix, int64_t n_prefix, hipStream_t s) {
  const Plan pl = plan_for(a, 1, kMaxGroups8);
  MoreParams p{};
  const int st = decode_params(a, 1, pl, &p);
  if (st != LATENT_OK) return st;
  p.scales = device_scales(scales);
  p.prefix = prefix;
  p.prefix_pages = static_cast<uint32_t>(n_prefix);
  return launch8<false, true>(a, scales.code, pl, p, s);
}

}  // namespace attend
}  // namespace latent

using namespace latent;
using namespace latent::attend;

extern "C" int latent_attn_decode_q8_workspace_size(const latent_attn_decode_args* args, size_t* bytes) {
  if (!args || !bytes) return LATENT_E_INVALID;
  const int st = validate(*args);
  if (st != LATENT_OK) return st;
  const Plan pl = plan_for(*args, 1, kMaxGroups8);
  *bytes = pl.ml_bytes + pl.acc_bytes + pl.unit_bytes;
  return LATENT_OK;
}

extern "C" int latent_attn_decode_q8(const latent_attn_decode_args* args, const latent_kv_scales* scales, latent_stream_t stream) {
  if (!args || !scales) return LATENT_E_INVALID;
  const latent_attn_decode_args& a = *args;
  int st = validate(a);
  if (st == LATENT_OK) st = check_codes(a.cache, *scales, a.head_dim);
  if (st != LATENT_OK || a.cache.n_seq == 0) return st;
  const Plan pl = plan_for(a, 1, kMaxGroups8);
  MoreParams p{};
  st = decode_params(a, 1, pl, &p);
  if (st != LATENT_OK) return st;
  if (p.cache.max_len && (!scales->k || !scales->v)) return LATENT_E_INVALID;
  p.scales = device_scales(*scales);
  return launch8<false>(a, scales->code, pl, p, reinterpret_cast<hipStream_t>(stream));
}
