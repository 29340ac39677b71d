// Between two blocks of a layer: the residual stream after the one, and what the next reads.
//
//   x' = x + scale gate post(y),   n = pre(x')
//   post, pre: v / sqrt(mean(v^2) + eps) w + b, or of v - mean(v), or v itself
//
// Bound by memory: x, y and the gate are read once and x' and n written once.  A row stays in the registers of its waves from the
// first read to the last write, in fp32; each mean is a lane exchange and, where several waves have a row, one through
// LDS.  A layer norm takes the mean first and the squares of what is left after it, as the difference of two large sums
// would lose what a small variance is.
//
// Measured: 8190 rows of 7168, f32 stream, block and gate by token, n in bf16, 212 us (5.0 TB/s, a copy's rate); one row of 4096 4.0 us of GPU, a
// launch's time, 7.0 a call from Python.
#include "common.hpp"

#include <type_traits>

namespace latent {
namespace {

struct NormParams {
  const void *x, *y, *gate;
  void *x_out, *n_out;
  int64_t x_stride, y_stride, gate_stride, xo_stride, no_stride;  // elements
  const void *post_w, *post_b, *pre_w, *pre_b;
  uint32_t T, d;
  int32_t x_dtype, y_dtype, gate_dtype, n_dtype, post_dtype, pre_dtype;
  int32_t post, pre;
  float post_eps, pre_eps, scale;
};

// Elements i, i + kStep, .. i + 7 kStep of an array of any of the three types, those below d; kVec: neighbours, 16 bytes at a time.
template <bool kVec, int kStep>
__device__ __forceinline__ void load8(const void* p, int dtype, int64_t base, uint32_t i, uint32_t d, float fill, float (&v)[8]) {
  if constexpr (kVec) {
    if (i < d) {
      load_act8(p, dtype, base + i, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = fill;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = i + e * kStep < d ? load_act(p, dtype, base + i + e * kStep) : fill;
  }
}

__device__ __forceinline__ uint16_t to_half_bits(float v, int dtype) {
  if (dtype == LATENT_F16) return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
  return __builtin_bit_cast(uint16_t, static_cast<__bf16>(v));
}

template <bool kVec, int kStep>
__device__ __forceinline__ void store8(void* p, int dtype, int64_t base, uint32_t i, uint32_t d, const float (&v)[8]) {
  if constexpr (kVec) {
    if (i >= d) return;
    if (dtype == LATENT_F32) {
      float4* to = reinterpret_cast<float4*>(static_cast<float*>(p) + base + i);
      to[0] = float4{v[0], v[1], v[2], v[3]};
      to[1] = float4{v[4], v[5], v[6], v[7]};
      return;
    }
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = to_half_bits(v[2 * e], dtype) | static_cast<uint32_t>(to_half_bits(v[2 * e + 1], dtype)) << 16;
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + base + i) = uint4{w[0], w[1], w[2], w[3]};
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (i + e * kStep >= d) return;
      if (dtype == LATENT_F32)
        static_cast<float*>(p)[base + i + e * kStep] = v[e];
      else
        static_cast<uint16_t*>(p)[base + i + e * kStep] = to_half_bits(v[e], dtype);
    }
  }
}

// kRowWaves waves a row, kV pieces of eight elements a lane.
template <int kRowWaves, int kV, bool kVec>
__global__ void __launch_bounds__(kRowWaves > 4 ? kRowWaves * kWave : 4 * kWave) residual_norm_kernel(NormParams p) {
  constexpr int kRows = kRowWaves > 4 ? 1 : 4 / kRowWaves;  // of a workgroup
  constexpr int kLanes = kRowWaves * kWave;
  constexpr int kStep = kVec ? 1 : kLanes;  // rows that no 16 bytes divide go by elements, neighbouring lanes' neighbours
  __shared__ float sums[4][kRowWaves];
  const int tid = threadIdx.x, wave = tid / kWave % kRowWaves;
  const uint32_t t = blockIdx.x * kRows + tid / kLanes, lane = tid % kLanes;
  if (t >= p.T) return;  // rows of one wave only: none waits for another
  int round = 0;
  // The sum over the row's lanes.
  auto total = [&](float v) {
    v = op_over(v, 1, 64, OpAdd{});
    if constexpr (kRowWaves > 1) {
      float(&s)[kRowWaves] = sums[round++];
      if (tid % kWave == 0) s[wave] = v;
      __syncthreads();
      v = 0.f;
#pragma unroll
      for (int w = 0; w < kRowWaves; ++w) v += s[w];
    }
    return v;
  };
  const uint32_t d = p.d;
  const float count = static_cast<float>(d);
  auto at = [&](int j) { return kVec ? 8 * (lane + j * kLanes) : lane + 8 * j * kLanes; };
  float x[kV][8];
#pragma unroll
  for (int j = 0; j < kV; ++j) load8<kVec, kStep>(p.x, p.x_dtype, t * p.x_stride, at(j), d, 0.f, x[j]);
  float y[kV][8];
  if (p.y) {
#pragma unroll
    for (int j = 0; j < kV; ++j) load8<kVec, kStep>(p.y, p.y_dtype, t * p.y_stride, at(j), d, 0.f, y[j]);
  }
  // Where a lane has one piece, weights, biases and the gate are fetched with the row: their latency would follow each sum's.
  constexpr bool kAhead = kV == 1;
  struct Fetched {
    float v[kAhead ? 5 : 1][8];
  } ahead;
  if constexpr (kAhead) {
    if (p.post_w) load8<kVec, kStep>(p.post_w, p.post_dtype, 0, at(0), p.d, 0.f, ahead.v[0]);
    if (p.post_b) load8<kVec, kStep>(p.post_b, p.post_dtype, 0, at(0), p.d, 0.f, ahead.v[1]);
    if (p.gate) load8<kVec, kStep>(p.gate, p.gate_dtype, t * p.gate_stride, at(0), p.d, 0.f, ahead.v[2]);
    if (p.pre_w) load8<kVec, kStep>(p.pre_w, p.pre_dtype, 0, at(0), p.d, 0.f, ahead.v[3]);
    if (p.pre_b) load8<kVec, kStep>(p.pre_b, p.pre_dtype, 0, at(0), p.d, 0.f, ahead.v[4]);
  }
  auto operand = [&](const void* from, int dtype, int64_t base, int j, int which, float (&f)[8]) {
    if constexpr (kAhead) {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = ahead.v[which][e];
    } else {
      load8<kVec, kStep>(from, dtype, base, at(j), p.d, 0.f, f);
    }
  };
  auto norm = [&](float (&v)[kV][8], int kind, float eps, const void* w, const void* b, int dtype, int which) {
    float mean = 0.f;
    if (kind == LATENT_NORM_LAYER) {
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < kV; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) s += v[j][e];
      mean = total(s) / count;
    }
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < kV; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        // What is behind the row's end stays zero.
        if (kind == LATENT_NORM_LAYER) v[j][e] = at(j) + e * kStep < d ? v[j][e] - mean : 0.f;
        s += v[j][e] * v[j][e];
      }
    const float r = 1.f / sqrtf(total(s) / count + eps);
#pragma unroll
    for (int j = 0; j < kV; ++j) {
      float f[8];
      if (w) operand(w, dtype, 0, j, which, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[j][e] = w ? v[j][e] * r * f[e] : v[j][e] * r;
      if (b) {
        operand(b, dtype, 0, j, which + 1, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] += f[e];
      }
    }
  };
  if (p.y) {
    if (p.post != LATENT_NORM_NONE) norm(y, p.post, p.post_eps, p.post_w, p.post_b, p.post_dtype, 0);
#pragma unroll
    for (int j = 0; j < kV; ++j) {
      if (p.gate) {
        float g[8];
        operand(p.gate, p.gate_dtype, t * p.gate_stride, j, 2, g);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[j][e] *= g[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) x[j][e] += p.scale * y[j][e];
    }
  }
  if (p.x_out) {
#pragma unroll
    for (int j = 0; j < kV; ++j) store8<kVec, kStep>(p.x_out, p.x_dtype, t * p.xo_stride, at(j), d, x[j]);
  }
  if (!p.n_out) return;
  if (p.pre != LATENT_NORM_NONE) norm(x, p.pre, p.pre_eps, p.pre_w, p.pre_b, p.pre_dtype, 3);
#pragma unroll
  for (int j = 0; j < kV; ++j) store8<kVec, kStep>(p.n_out, p.n_dtype, t * p.no_stride, at(j), d, x[j]);
}

constexpr int64_t kMaxNormDim = 32768;

bool dtype_ok(int32_t t) { return t == LATENT_F32 || t == LATENT_F16 || t == LATENT_BF16; }

int check_norm(const latent_norm& n) {
  if (n.kind != LATENT_NORM_NONE && n.kind != LATENT_NORM_RMS && n.kind != LATENT_NORM_LAYER) return LATENT_E_INVALID;
  if (n.kind == LATENT_NORM_NONE) return n.weight || n.bias ? LATENT_E_INVALID : LATENT_OK;
  if (!(n.eps >= 0.f) || !(n.eps < INFINITY)) return LATENT_E_INVALID;
  return (n.weight || n.bias) && !dtype_ok(n.dtype) ? LATENT_E_INVALID : LATENT_OK;
}

}  // namespace
}  // namespace latent

using namespace latent;

extern "C" int latent_residual_norm(const latent_residual_norm_args* args, latent_stream_t stream) {
  if (!args) return LATENT_E_INVALID;
  const latent_residual_norm_args& a = *args;
  if (a.n_tokens < 0 || a.n_embd < 0) return LATENT_E_INVALID;
  for (const latent_norm* n : {&a.post, &a.pre})
    if (check_norm(*n) != LATENT_OK) return LATENT_E_INVALID;
  if (!dtype_ok(a.x_dtype) || (a.y && !dtype_ok(a.y_dtype)) || (a.gate && !dtype_ok(a.gate_dtype)) || (a.n_out && !dtype_ok(a.n_dtype)))
    return LATENT_E_INVALID;
  if (!(a.scale > -INFINITY) || !(a.scale < INFINITY)) return LATENT_E_INVALID;
  if (!a.y && (a.gate || a.post.kind != LATENT_NORM_NONE)) return LATENT_E_INVALID;
  if (!a.n_out && a.pre.kind != LATENT_NORM_NONE) return LATENT_E_INVALID;
  // A launch's threads are counted in 32 bits: a wave, four or sixteen a row.
  if (a.n_embd > kMaxNormDim || a.n_tokens > (int64_t{1} << 32) / (a.n_embd <= 1024 ? 64 : a.n_embd <= 8192 ? 256 : 1024) - 8) return LATENT_E_UNSUPPORTED;
  constexpr int64_t kFar = int64_t{1} << 40;
  for (int64_t s : {a.x_stride, a.y_stride, a.gate_stride, a.x_out_stride, a.n_out_stride})
    if (s < 0 || s > kFar) return LATENT_E_UNSUPPORTED;
  if (a.n_tokens == 0 || a.n_embd == 0) return LATENT_OK;
  if (!a.x) return LATENT_E_INVALID;
  if (!a.x_out && !a.n_out) return LATENT_OK;
  // Rows that are written may not overlap.
  if (a.n_tokens > 1 && ((a.x_out && a.x_out_stride < a.n_embd) || (a.n_out && a.n_out_stride < a.n_embd))) return LATENT_E_INVALID;
  NormParams p{};
  p.x = a.x, p.y = a.y, p.gate = a.gate, p.x_out = a.x_out, p.n_out = a.n_out;
  p.x_stride = a.x_stride, p.y_stride = a.y_stride, p.gate_stride = a.gate_stride, p.xo_stride = a.x_out_stride, p.no_stride = a.n_out_stride;
  p.post_w = a.post.weight, p.post_b = a.post.bias, p.pre_w = a.pre.weight, p.pre_b = a.pre.bias;
  p.T = static_cast<uint32_t>(a.n_tokens);
  p.d = static_cast<uint32_t>(a.n_embd);
  p.x_dtype = a.x_dtype, p.y_dtype = a.y_dtype, p.gate_dtype = a.gate_dtype, p.n_dtype = a.n_dtype;
  p.post_dtype = a.post.dtype, p.pre_dtype = a.pre.dtype;
  p.post = a.post.kind, p.pre = a.pre.kind;
  p.post_eps = a.post.eps, p.pre_eps = a.pre.eps;
  p.scale = a.scale;
  // Sixteen bytes at a time where every row and array allows it.
  bool vec = a.n_embd % 8 == 0;
  for (const void* ptr : {a.x, a.y, a.gate, static_cast<const void*>(a.x_out), static_cast<const void*>(a.n_out), a.post.weight, a.post.bias, a.pre.weight, a.pre.bias})
    vec = vec && (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0;
  for (int64_t s : {a.x_stride, a.y_stride, a.gate_stride, a.x_out_stride, a.n_out_stride}) vec = vec && s % 8 == 0;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  (void)hipGetLastError();
  auto launch = [&](auto waves, auto v) {
    constexpr int kRowWaves = decltype(waves)::value, kV = decltype(v)::value, kRows = kRowWaves > 4 ? 1 : 4 / kRowWaves;
    const dim3 grid((p.T + kRows - 1) / kRows), block(kRowWaves > 4 ? kRowWaves * kWave : 4 * kWave);
    if (vec)
      hipLaunchKernelGGL((residual_norm_kernel<kRowWaves, kV, true>), grid, block, 0, s, p);
    else
      hipLaunchKernelGGL((residual_norm_kernel<kRowWaves, kV, false>), grid, block, 0, s, p);
  };
  using std::integral_constant;
  typedef integral_constant<int, 1> One;
  typedef integral_constant<int, 2> Two;
  typedef integral_constant<int, 4> Four;
  typedef integral_constant<int, 16> Sixteen;
  // Few rows: as many waves as leave a lane one piece.  Many: fewer waves, which exchange less.  f32 stream, bf16 block, both norms and a
  // gate, as a part of a graph: 1 row of 7168 4.6 us, 7.2 by four waves, 256 rows 8.3 and 11.4, 1024 rows 24.7 and 20.2; 1 row of 4096 4.0 and
  // 4.7, 512 rows 11.0 and 9.4; 512 rows of 1024 4.2 by four waves and 5.2 by one, 2048 rows 10.1 and 9.2.
  const uint32_t d = p.d;
  const bool few = p.T <= (d <= 2048 ? 1024 : 256);
  if (d <= 512) launch(One{}, One{});
  else if (d <= 1024 && !few) launch(One{}, Two{});
  else if (d <= 2048) launch(Four{}, One{});
  else if (d <= 8192 && few) launch(Sixteen{}, One{});
  else if (d <= 4096) launch(Four{}, Two{});
  else if (d <= 8192) launch(Four{}, Four{});
  else if (d <= 16384) launch(Sixteen{}, Two{});
  else launch(Sixteen{}, Four{});
  return hipGetLastError() == hipSuccess ? LATENT_OK : LATENT_E_HIP;
}
