// Attention of one new token for each of a batch of sequences whose first positions are the same.
//
//   out[b][h] = sum_j p_j v[j] / sum_j p_j over the prefix's keys and the sequence's own
//
// The rows of all sequences against the prefix's keys are the products of a prompt without a mask (B G rows of a key/value head
// over one sequence of keys: each key is read once for 128 rows, split over the chip); the sequences' own keys are a decode that
// begins behind the prefix.  Both leave parts in fp32, and a third launch joins a row's.  (Rows joined where the decode finishes
// them, without that launch, took longer: few lanes read all of the prior's parts one after the other, 64 sequences behind 16000 126 us.)
// Few sequences, or a short prefix, are a decode that looks the first pages up in the prefix instead (kTogether).
//
// Measured: 5 sequences behind 4096 shared positions, up to 700 of their own, 32 over 8 heads, 16-bit, 18.7 us, as a decode; 64 behind
// 16000, up to 2000 of their own, 64 over 8 heads, 106 us (16-bit) to 109 (int8): the prefix 69, bound by its products as prompts are
// (490 TFLOP/s), own keys 31, the join 10.  A decode that reads all positions of each sequence takes 460 us there (int8 306).
#include "shared.hpp"

using namespace latent;
using namespace latent::attend;

namespace {

// Numbers that all sequences together would read of the prefix's keys and values up to which they do, each for itself, in the one or two
// launches of a decode: what the last-level cache gives them costs less than the third launch and the parts.  One number for caches of all types and any
// batch, near where the two cross over 16 bits; over codes, and for a sequence or two, which read little or nothing again, together would be the shorter
// a while longer (int8 at 67M below; one sequence 27.6 us behind 28672 positions, together, and 43.8 behind 32768, split).  32 over 8 heads of 128, up to 300
// positions of their own, together and split: 5 sequences behind 4096 (42M) 19.8 and 23.9 us (int8 23.4 and 27.5), 8 (67M) 27.8 and 23.4 (26.2
// and 27.6), 16 (134M) 42.9 and 25.6 (40.2 and 29.6); 16 over one head of 64, 64 behind 4096 (34M) 18.7 and 22.6.
constexpr int64_t kTogether = 56 << 20;

struct Layout {
  bool together;
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
  const int64_t row = 2 * d.n_kv_head * d.head_dim, keys = a.n_prefix * d.cache.page_size;  // below 2^20 and 2^31
  l->together = keys == 0 || d.cache.n_seq <= kTogether / (row * keys);
  if (!l->together) l->bytes = plan_prior(d, a.n_prefix, &l->prior);
  l->after = l->together ? n : after_workspace(d, a.n_prefix, a.scales != nullptr);
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
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (l.together)
    return args->scales ? launch_together8(a, *args->scales, args->prefix, args->n_prefix, s) : launch_together16(a, args->prefix, args->n_prefix, s);
  if (!a.workspace || a.workspace_bytes < l.all()) return LATENT_E_WORKSPACE;
  char* ws = static_cast<char*>(a.workspace);
  Prior& prior = l.prior;
  prior.acc = reinterpret_cast<float*>(ws);
  prior.ml = reinterpret_cast<float*>(ws + l.bytes.acc);
  void* scratch = ws + l.bytes.acc + l.bytes.ml;
  st = args->scales ? launch_prefix8(a, *args->scales, args->prefix, args->n_prefix, prior, s)
                    : launch_prefix16(a, args->prefix, args->n_prefix, prior, s);
  if (st != LATENT_OK) return st;
  return args->scales ? launch_after8(a, *args->scales, args->n_prefix, prior, scratch, s) : launch_after16(a, args->n_prefix, prior, scratch, s);
}
