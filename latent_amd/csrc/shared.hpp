// The two halves of attention over a shared prefix, each launched by the file that has its kernels (shared.hip tells the whole).
#pragma once

#include "attend.hpp"

namespace latent {
namespace attend {

// What the first half leaves for the second: parts of `chunk` of the prefix's keys.  Row r = sequence G + head of the group is row r % 128 of
// row tile r / 128; a part has a reference, a sum and unnormalised rows, as the prompt kernels' threads hold them.
struct Prior {
  int32_t parts, chunk, tiles;
  float up;    // log2 of what the sums are times
  float* acc;  // [parts][tiles][n_kv_head][D padded / 8][256][4]
  float* ml;   // [parts][tiles][n_kv_head][256][4]: reference, sum, full sum
};
struct PriorBytes {
  size_t acc, ml;
};

// The prefix: queries of all sequences as one sequence's over the n_prefix pages of `prefix`.  plan_prior fills in all but the pointers.
PriorBytes plan_prior(const latent_attn_decode_args& a, int64_t n_prefix, Prior* prior);
int launch_prefix16(const latent_attn_decode_args& a, const int32_t* prefix, int64_t n_prefix, const Prior& prior, hipStream_t s);
int launch_prefix8(const latent_attn_decode_args& a, const latent_kv_scales& scales, const int32_t* prefix, int64_t n_prefix, const Prior& prior, hipStream_t s);

// The sequences' own positions, from n_prefix pages on, in parts too, and the join of both.
size_t after_workspace(const latent_attn_decode_args& a, int64_t n_prefix, bool codes);
int launch_after16(const latent_attn_decode_args& a, int64_t n_prefix, const Prior& prior, void* workspace, hipStream_t s);
int launch_after8(const latent_attn_decode_args& a, const latent_kv_scales& scales, int64_t n_prefix, const Prior& prior, void* workspace, hipStream_t s);

// Both at once, as a decode that looks the first pages up in `prefix`.
int launch_together16(const latent_attn_decode_args& a, const int32_t* prefix, int64_t n_prefix, hipStream_t s);
int launch_together8(const latent_attn_decode_args& a, const latent_kv_scales& scales, const int32_t* prefix, int64_t n_prefix, hipStream_t s);

}  // namespace attend
}  // namespace latent
