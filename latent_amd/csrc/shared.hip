// Attention of one new token for each of a batch of sequences whose first positions are the same.
//
//   out[b][h] = sum_j p_j v[j] / sum_j p_j over the prefix's keys and the sequence's own
//
// The rows of all sequences against the prefix's keys are the products of a prompt without a mask (B G rows of a key/value head
// over one sequence of keys: each key is read once for 128 rows, split over the chip); the sequences' own keys are a decode that
// begins behind the prefix.  Both leave parts in fp32, and a third launch joins a row's.  (Rows joined where the decode finishes
// them, without that launch, took longer: few lanes read all of the prior's parts one after the other, 64 sequences behind 16000 126 us.)
#include "shared.hpp"

using namespace latent;
using namespace latent::attend;

namespace {

struct Layout {
  Prior prior;
  PriorBytes bytes;
  size_t after;
  size_t all() const { return bytes.acc + bytes.ml + after; }
};

int layout_of(const latent_attn_shared_args& a, Layout* l) {
  const latent_attn_decode_args& d = a.decode;
  size_t n;
  // The decode's own checks: the call is one, to its caller.
  int st = a.scales ? latent_attn_decode_q8_workspace_size(&d, &n) : latent_attn_decode_workspace_size(&d, &n);
  if (st == LATENT_OK && a.scales) st = check_codes(d.cache, *a.scales, d.head_dim);
  if (st != LATENT_OK) return st;
  if (a.n_prefix < 0 || a.n_prefix > d.cache.max_pages) return LATENT_E_INVALID;
  const int64_t rows = d.cache.n_seq * d.n_head;
  // Row tiles of the prefix's launch are counted in 32 bits, rows with their elements in 31.
  if (rows * d.head_dim > INT32_MAX || (rows / 128 + d.n_kv_head) > 1 << 20) return LATENT_E_UNSUPPORTED;
  if (a.n_prefix) l->bytes = plan_prior(d, a.n_prefix, &l->prior);
  l->after = a.n_prefix ? after_workspace(d, a.n_prefix, a.scales != nullptr) : n;
  return LATENT_OK;
}

}  // namespace

extern "C" int latent_attn_decode_shared_workspace_size(const latent_attn_shared_args* args, size_t* bytes) {
  if (!args || !bytes) return LATENT_E_INVALID;
  Layout l{};
  const int st = layout_of(*args, &l);
  if (st == LATENT_OK) *bytes = l.all();
  return st;
}

extern "C" int latent_attn_decode_shared(const latent_attn_shared_args* args, latent_stream_t stream) {
  if (!args) return LATENT_E_INVALID;
  const latent_attn_decode_args& a = args->decode;
  Layout l{};
  int st = layout_of(*args, &l);
  if (st != LATENT_OK || a.cache.n_seq == 0) return st;
  if (args->n_prefix == 0) return args->scales ? latent_attn_decode_q8(&a, args->scales, stream) : latent_attn_decode(&a, stream);
  if (!args->prefix || !a.q || !a.out || !a.lengths) return LATENT_E_INVALID;
  if (a.cache.n_pages > 0 && (!a.cache.k || !a.cache.v || !a.cache.pages || (args->scales && (!args->scales->k || !args->scales->v))))
    return LATENT_E_INVALID;
  if (!aligned16(a.q) || !aligned16(a.out) || !aligned16(a.workspace)) return LATENT_E_UNSUPPORTED;
  for (int64_t s : {a.q_token_stride, a.q_head_stride, a.out_token_stride, a.out_head_stride})
    if (!stride_ok(s)) return LATENT_E_UNSUPPORTED;
  if ((a.n_head > 1 && !a.out_head_stride) || (a.cache.n_seq > 1 && !a.out_token_stride)) return LATENT_E_INVALID;
  if (!a.workspace || a.workspace_bytes < l.all()) return LATENT_E_WORKSPACE;
  char* ws = static_cast<char*>(a.workspace);
  Prior& prior = l.prior;
  prior.acc = reinterpret_cast<float*>(ws);
  prior.ml = reinterpret_cast<float*>(ws + l.bytes.acc);
  void* scratch = ws + l.bytes.acc + l.bytes.ml;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  st = args->scales ? launch_prefix8(a, *args->scales, args->prefix, args->n_prefix, prior, s)
                    : launch_prefix16(a, args->prefix, args->n_prefix, prior, s);
  if (st != LATENT_OK) return st;
  return args->scales ? launch_after8(a, *args->scales, args->n_prefix, prior, scratch, s) : launch_after16(a, args->n_prefix, prior, scratch, s);
}
