// The two halves of attention over a shared prefix, each launched by the file that has its kernels (shared.hip tells the whole).
#pragma once

#include "attend.hpp"

namespace latent {
namespace attend {

// Where the rows' outputs over the prefix lie between the halves: fp32, normalised, and the log2 of their sums of exponentials.
struct Prior {
  float* out;  // [n_seq][n_head][D]
  float* lse;  // [n_seq][n_head]
};

// The prefix: queries of all sequences as one sequence's over the n_prefix pages of `prefix`.
size_t prefix_workspace(const latent_attn_decode_args& a, int64_t n_prefix);
int launch_prefix16(const latent_attn_decode_args& a, const int32_t* prefix, int64_t n_prefix, const Prior& prior, void* workspace, hipStream_t s);
int launch_prefix8(const latent_attn_decode_args& a, const latent_kv_scales& scales, const int32_t* prefix, int64_t n_prefix, const Prior& prior,
                   void* workspace, hipStream_t s);

// The sequences' own positions, from n_prefix pages on, joined with the prior.
size_t after_workspace(const latent_attn_decode_args& a, int64_t n_prefix, bool codes);
int launch_after16(const latent_attn_decode_args& a, int64_t n_prefix, const Prior& prior, void* workspace, hipStream_t s);
int launch_after8(const latent_attn_decode_args& a, const latent_kv_scales& scales, int64_t n_prefix, const Prior& prior, void* workspace, hipStream_t s);

}  // namespace attend
}  // namespace latent
