// Host-side argument handling of the attention entry points under
// AddressSanitizer and UndefinedBehaviorSanitizer (built by
// tests/test_host_attention_sanitizers.py from their host code only).  Every
// call below returns before any kernel launch.  Exit status = number of failed
// expectations.
#include <cstdint>
#include <cstdio>
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

latent_kv_cache cache() {
  latent_kv_cache c{};
  c.k = c.v = buf;
  c.pages = reinterpret_cast<const int32_t*>(buf);
  c.n_pages = 10, c.page_size = 16, c.n_seq = 4, c.max_pages = 1000, c.pages_stride = 1000;
  c.k_page_stride = c.v_page_stride = 16 * 128;
  c.k_row_stride = c.v_row_stride = 128;
  c.k_head_stride = c.v_head_stride = 64;
  return c;
}

const int64_t kEdges[] = {std::numeric_limits<int64_t>::min(), -1, 0, 1, 7, 8, 63, 64, 1 << 20, int64_t{1} << 31, int64_t{1} << 40,
                          std::numeric_limits<int64_t>::max()};

// Every size field at every edge: a status, no overflow that the sanitizers would report.
template <typename Args, typename Call>
void sweep(const Args& good, int64_t latent_kv_cache::*const* cf, int nc, int64_t Args::*const* fields, int n, Call call) {
  for (int64_t edge : kEdges) {
    for (int i = 0; i < nc; ++i) {
      Args a = good;
      a.cache.*cf[i] = edge;
      EXPECT(call(a) <= LATENT_OK);
    }
    for (int i = 0; i < n; ++i) {
      Args a = good;
      a.*fields[i] = edge;
      EXPECT(call(a) <= LATENT_OK);
    }
  }
}

int64_t latent_kv_cache::*const kCache[] = {
    &latent_kv_cache::n_pages,       &latent_kv_cache::page_size,     &latent_kv_cache::n_seq,         &latent_kv_cache::max_pages,
    &latent_kv_cache::pages_stride,  &latent_kv_cache::k_page_stride, &latent_kv_cache::k_row_stride,  &latent_kv_cache::k_head_stride,
    &latent_kv_cache::v_page_stride, &latent_kv_cache::v_row_stride,  &latent_kv_cache::v_head_stride};
constexpr int kNCache = sizeof(kCache) / sizeof(kCache[0]);

void append() {
  typedef latent_kv_append_args A;
  A a{};
  a.cache = cache();
  a.q = a.k = a.v = buf;
  // a.q_out stays NULL: a call with good sizes ends at the pointer checks.
  a.positions = reinterpret_cast<const int32_t*>(buf);
  a.rope = reinterpret_cast<const float*>(buf);
  a.q_token_stride = a.q_out_token_stride = 256, a.k_token_stride = a.v_token_stride = 128;
  a.q_head_stride = a.q_out_head_stride = a.k_head_stride = a.v_head_stride = 64;
  a.rope_rows = 100, a.rot_dim = 64, a.n_tokens = 4, a.n_head = 4, a.n_kv_head = 2, a.head_dim = 64, a.dtype = LATENT_BF16;
  auto call = [](const A& x) { return latent_kv_append(&x, nullptr); };
  EXPECT(call(a) == LATENT_E_INVALID);
  int64_t A::*const fields[] = {&A::q_token_stride, &A::q_head_stride, &A::k_token_stride, &A::rope_rows, &A::rot_dim,
                                &A::n_tokens,       &A::n_kv_head,     &A::head_dim};
  sweep(a, kCache, kNCache, fields, sizeof(fields) / sizeof(fields[0]), call);
}

void decode() {
  typedef latent_attn_decode_args A;
  A a{};
  a.cache = cache();
  a.q = buf;
  a.out = buf;
  a.lengths = reinterpret_cast<const int32_t*>(buf);
  a.q_token_stride = a.out_token_stride = 256, a.q_head_stride = a.out_head_stride = 64;
  a.n_head = 4, a.n_kv_head = 2, a.head_dim = 64, a.dtype = LATENT_F16, a.scale = 0.125f;
  int64_t A::*const fields[] = {&A::q_token_stride, &A::out_head_stride, &A::n_head, &A::n_kv_head, &A::head_dim};
  auto size = [](const A& x) {
    size_t n = 0;
    return latent_attn_decode_workspace_size(&x, &n);
  };
  EXPECT(size(a) == LATENT_OK);
  sweep(a, kCache, kNCache, fields, sizeof(fields) / sizeof(fields[0]), size);
  a.lengths = nullptr;  // good sizes end at the pointer checks
  sweep(a, kCache, kNCache, fields, sizeof(fields) / sizeof(fields[0]), [](const A& x) { return latent_attn_decode(&x, nullptr); });
}

void prompt() {
  typedef latent_attn_prompt_args A;
  A a{};
  a.cache = cache();
  a.q = a.k = a.v = buf;  // no starts: good sizes end at the pointer checks
  a.out = buf;
  a.q_token_stride = a.out_token_stride = 256, a.k_token_stride = a.v_token_stride = 128;
  a.q_head_stride = a.out_head_stride = a.k_head_stride = a.v_head_stride = 64;
  a.n_tokens = 20, a.n_keys = 20, a.n_head = 4, a.n_kv_head = 2, a.head_dim = 64, a.dtype = LATENT_F16, a.scale = 0.125f;
  int64_t A::*const fields[] = {&A::q_token_stride, &A::out_head_stride, &A::k_token_stride, &A::n_tokens, &A::n_keys,
                                &A::n_head,         &A::n_kv_head,       &A::head_dim};
  auto call = [](const A& x) { return latent_attn_prompt(&x, nullptr); };
  EXPECT(call(a) == LATENT_E_INVALID);
  sweep(a, kCache, kNCache, fields, sizeof(fields) / sizeof(fields[0]), call);
  auto size = [](const A& x) {
    size_t n = 0;
    return latent_attn_prompt_workspace_size(&x, &n);
  };
  EXPECT(size(a) == LATENT_OK);
  sweep(a, kCache, kNCache, fields, sizeof(fields) / sizeof(fields[0]), size);
  a.k = nullptr;
  a.n_keys = 0;
  sweep(a, kCache, kNCache, fields, sizeof(fields) / sizeof(fields[0]), call);
}

}  // namespace

int main() {
  append();
  decode();
  prompt();
  std::printf("host attention checks: %d failed\n", failures);
  return failures;
}
