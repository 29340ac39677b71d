// Host-side argument handling of the 8-bit caches', the shared prefix's and the residual norm's entry points under AddressSanitizer and
// UndefinedBehaviorSanitizer (built by tests/test_host_cache8_sanitizers.py from their host code only).  Every
// call below returns before any kernel launch.  Exit status = number of failed expectations.
#include <cstdint>
#include <cstdio>
#include <initializer_list>
#include <limits>

#include "latent_ffn.h"

static int failures = 0;
#define EXPECT(cond)                                                    \
  do {                                                                  \
    if (!(cond)) {                                                      \
      std::fprintf(stderr, "%s:%d: expectation failed: %s\n", __FILE__, __LINE__, #cond); \
      ++failures;                                                       \
    }                                                                   \
  } while (0)

namespace {

alignas(16) char buf[64];  // stands in for every operand (never read)
const int32_t* ints = reinterpret_cast<const int32_t*>(buf);
const int64_t kEdges[] = {std::numeric_limits<int64_t>::min(), -1, 0, 1, 7, 8, 16, 63, 64, 1 << 20, int64_t{1} << 31, int64_t{1} << 40,
                          std::numeric_limits<int64_t>::max()};

latent_kv_cache cache() {
  latent_kv_cache c{};
  c.k = c.v = buf;
  c.pages = ints;
  c.n_pages = 10, c.page_size = 16, c.n_seq = 4, c.max_pages = 1000, c.pages_stride = 1000;
  c.k_page_stride = c.v_page_stride = 16 * 128;
  c.k_row_stride = c.v_row_stride = 128;
  c.k_head_stride = c.v_head_stride = 64;
  return c;
}
latent_kv_scales scales() {
  latent_kv_scales s{};
  s.k = s.v = reinterpret_cast<float*>(buf);
  s.k_page_stride = s.v_page_stride = 32, s.k_head_stride = s.v_head_stride = 16;
  return s;
}

// Every field at every edge: a status, no overflow that the sanitizers would report.
template <typename Struct, typename Call>
void sweep(Struct& of, int64_t Struct::*const* fields, int n, Call call) {
  for (int64_t edge : kEdges)
    for (int i = 0; i < n; ++i) {
      const int64_t was = of.*fields[i];
      of.*fields[i] = edge;
      EXPECT(call() <= LATENT_OK);
      of.*fields[i] = was;
    }
}
#define COUNT(a) static_cast<int>(sizeof(a) / sizeof(a[0]))

int64_t latent_kv_cache::*const kCache[] = {
    &latent_kv_cache::n_pages,       &latent_kv_cache::page_size,     &latent_kv_cache::n_seq,         &latent_kv_cache::max_pages,
    &latent_kv_cache::pages_stride,  &latent_kv_cache::k_page_stride, &latent_kv_cache::k_row_stride,  &latent_kv_cache::k_head_stride,
    &latent_kv_cache::v_page_stride, &latent_kv_cache::v_row_stride,  &latent_kv_cache::v_head_stride};
int64_t latent_kv_scales::*const kScales[] = {&latent_kv_scales::k_page_stride, &latent_kv_scales::k_head_stride, &latent_kv_scales::v_page_stride,
                                              &latent_kv_scales::v_head_stride};

template <typename Args, typename Call>
void all(Args& a, latent_kv_cache& c, latent_kv_scales& s, int64_t Args::*const* fields, int n, Call call) {
  EXPECT(call() <= LATENT_OK);
  sweep(a, fields, n, call);
  sweep(c, kCache, COUNT(kCache), call);
  sweep(s, kScales, COUNT(kScales), call);
  for (int32_t code : {-1, 1, 2, 1 << 30}) {
    s.code = code;
    EXPECT(call() <= LATENT_OK);
  }
  s.code = 0;
}

void append_and_read() {
  typedef latent_kv_append_args A;
  A a{};
  latent_kv_scales s = scales();
  a.cache = cache();
  a.q = a.k = a.v = buf;  // no q_out: good sizes end at the pointer checks
  a.positions = ints;
  a.rope = reinterpret_cast<const float*>(buf);
  a.q_token_stride = a.q_out_token_stride = 256, a.k_token_stride = a.v_token_stride = 128;
  a.q_head_stride = a.q_out_head_stride = a.k_head_stride = a.v_head_stride = 64;
  a.rope_rows = 100, a.rot_dim = 64, a.n_tokens = 4, a.n_head = 4, a.n_kv_head = 2, a.head_dim = 64, a.dtype = LATENT_BF16;
  int64_t A::*const fields[] = {&A::q_token_stride, &A::k_token_stride, &A::rope_rows, &A::rot_dim, &A::n_tokens, &A::n_kv_head, &A::head_dim};
  all(a, a.cache, s, fields, COUNT(fields), [&] { return latent_kv_append_q8(&a, &s, nullptr); });

  typedef latent_kv_read_args R;
  R r{};
  r.cache = cache();
  r.k = r.v = buf;  // no positions
  r.k_token_stride = r.v_token_stride = 128, r.k_head_stride = r.v_head_stride = 64;
  r.n_tokens = 4, r.n_kv_head = 2, r.head_dim = 64, r.dtype = LATENT_F16;
  int64_t R::*const more[] = {&R::k_token_stride, &R::v_head_stride, &R::n_tokens, &R::n_kv_head, &R::head_dim};
  all(r, r.cache, s, more, COUNT(more), [&] { return latent_kv_read(&r, &s, nullptr); });
  all(r, r.cache, s, more, COUNT(more), [&] { return latent_kv_read(&r, nullptr, nullptr); });
}

void attention() {
  typedef latent_attn_decode_args A;
  latent_attn_shared_args sh{};
  A& a = sh.decode;
  latent_kv_scales s = scales();
  size_t n;
  a.cache = cache();
  a.q = a.out = buf;  // no lengths
  a.q_token_stride = a.out_token_stride = 256, a.q_head_stride = a.out_head_stride = 64;
  a.n_head = 4, a.n_kv_head = 2, a.head_dim = 64, a.dtype = LATENT_F16, a.scale = 0.125f;
  a.workspace = buf;
  a.workspace_bytes = SIZE_MAX;
  int64_t A::*const fields[] = {&A::q_token_stride, &A::out_head_stride, &A::n_head, &A::n_kv_head, &A::head_dim};
  all(a, a.cache, s, fields, COUNT(fields), [&] { return latent_attn_decode_q8_workspace_size(&a, &n); });
  all(a, a.cache, s, fields, COUNT(fields), [&] { return latent_attn_decode_q8(&a, &s, nullptr); });
  sh.prefix = ints;
  sh.n_prefix = 3;
  int64_t latent_attn_shared_args::*const prefix[] = {&latent_attn_shared_args::n_prefix};
  for (const latent_kv_scales* with : {static_cast<const latent_kv_scales*>(nullptr), static_cast<const latent_kv_scales*>(&s)}) {
    sh.scales = with;
    auto size = [&] { return latent_attn_decode_shared_workspace_size(&sh, &n); };
    auto call = [&] { return latent_attn_decode_shared(&sh, nullptr); };
    EXPECT(size() == LATENT_OK);
    all(a, a.cache, s, fields, COUNT(fields), size);
    all(a, a.cache, s, fields, COUNT(fields), call);
    sweep(sh, prefix, COUNT(prefix), size);
    sweep(sh, prefix, COUNT(prefix), call);
  }
  typedef latent_attn_prompt_args P;
  P p{};
  p.cache = cache();
  p.q = p.out = buf;  // no starts
  p.q_token_stride = p.out_token_stride = 256, p.q_head_stride = p.out_head_stride = 64;
  p.n_tokens = 20, p.n_head = 4, p.n_kv_head = 2, p.head_dim = 64, p.dtype = LATENT_F16, p.scale = 0.125f;
  int64_t P::*const more[] = {&P::q_token_stride, &P::out_head_stride, &P::n_tokens, &P::n_keys, &P::n_head, &P::n_kv_head, &P::head_dim};
  all(p, p.cache, s, more, COUNT(more), [&] { return latent_attn_prompt_q8(&p, &s, nullptr); });
}

void norm() {
  typedef latent_residual_norm_args A;
  A a{};  // no x: good sizes end at the pointer check
  a.y = a.gate = buf;
  a.x_out = a.n_out = buf;
  a.x_stride = a.y_stride = a.gate_stride = a.x_out_stride = a.n_out_stride = 64;
  a.n_tokens = 4, a.n_embd = 64, a.scale = 1.f;
  a.pre.kind = LATENT_NORM_RMS;
  auto call = [&] { return latent_residual_norm(&a, nullptr); };
  EXPECT(call() == LATENT_E_INVALID);
  int64_t A::*const fields[] = {&A::x_stride, &A::y_stride, &A::gate_stride, &A::x_out_stride, &A::n_out_stride, &A::n_tokens, &A::n_embd};
  sweep(a, fields, COUNT(fields), call);
}

}  // namespace

int main() {
  append_and_read();
  attention();
  norm();
  std::printf("host 8-bit cache checks: %d failed\n", failures);
  return failures;
}
