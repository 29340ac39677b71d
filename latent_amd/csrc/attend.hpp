// What the attention kernels share: element types and their matrix products,
// the paged cache's addressing, the pairing of rows that turns loaded value rows
// into matrix operands, and the host's checks.
#pragma once

#include "common.hpp"

namespace latent {
namespace attend {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kMaxDim = 256;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

// The two element types: conversions and the fp32-accumulating products.  Eight
// elements of an operand travel as four dwords.
//
// Probabilities that are to be rounded to f16 are held times 2^kLift, so that the largest come near the type's
// largest: unlifted, those below 2^-14 of the largest would lose their bits, and a hundred thousand of them are not little.
// bf16 has fp32's range and needs none.
struct F16 {
  static constexpr float kLift = 15.f;
  typedef _Float16 T;
  typedef _Float16 T2 __attribute__((ext_vector_type(2)));
  typedef _Float16 T8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(T8, a), __builtin_bit_cast(T8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(T8, a), __builtin_bit_cast(T8, b), c, 0, 0, 0);
  }
  // c plus the dword's two elements.
  static __device__ __forceinline__ float add2(uint32_t w, float c) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(T2, w), __builtin_bit_cast(T2, 0x3C003C00u), c, false);
  }
};
struct BF16 {
  static constexpr float kLift = 0.f;
  typedef __bf16 T;
  typedef __bf16 T2 __attribute__((ext_vector_type(2)));
  typedef __bf16 T8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(T8, a), __builtin_bit_cast(T8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(T8, a), __builtin_bit_cast(T8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float add2(uint32_t w, float c) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(T2, w), __builtin_bit_cast(T2, 0x3F803F80u), c, false);
  }
};

// Two fp32 values rounded to nearest even, the first in the low half.
template <typename E>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), typename E::T2));
}
template <typename E>
__device__ __forceinline__ float unpack_lo(uint32_t w) {
  if constexpr (sizeof(E) && __is_same(E, F16)) return half_bits_to_float(static_cast<uint16_t>(w));
  return __uint_as_float(w << 16);
}
template <typename E>
__device__ __forceinline__ float unpack_hi(uint32_t w) {
  if constexpr (sizeof(E) && __is_same(E, F16)) return half_bits_to_float(static_cast<uint16_t>(w >> 16));
  return __uint_as_float(w & 0xFFFF0000u);
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// A running maximum of -inf (nothing seen yet) would make -inf - -inf: its
// exponentials are taken against 0 instead, where they are 0 too.
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.f : m; }

// What a masked key reads: 0 * p stays 0 whatever the cache's unused rows hold.
__device__ const u32x4 kZeroRow[kMaxDim * 2 / 16] = {};

// Direct global -> LDS loads: lane l's 16 bytes land at LDS byte address lds + 16 l; lds is wave-uniform.  Inline
// assembly, so that the compiler does not make every later LDS read wait for them; whoever issues them waits
// (pipeline_barrier).  They write memory, so no access of the program's own moves across them.  The second form takes a wave-uniform base and a 32-bit lane offset.
__device__ __forceinline__ void dma16(const void* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(__builtin_amdgcn_readfirstlane(lds)) : "m0", "memory");
}
__device__ __forceinline__ void dma16s(const void* base, uint32_t off, uint32_t lds) {
  const uint64_t v = reinterpret_cast<uintptr_t>(base);
  const uint64_t u = static_cast<uint64_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32))) << 32 |
                     static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v)));
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(u),
               "s"(__builtin_amdgcn_readfirstlane(lds))
               : "m0", "memory");
}

template <typename T>
__device__ __forceinline__ uint32_t lds_addr(T& obj) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)(&obj)));
}
template <typename T>
__device__ __forceinline__ T lds_ld(uint32_t addr) {
  return *reinterpret_cast<const __attribute__((address_space(3))) T*>(static_cast<uintptr_t>(addr));
}
template <typename T>
__device__ __forceinline__ void lds_st(uint32_t addr, T v) {
  *reinterpret_cast<__attribute__((address_space(3))) T*>(static_cast<uintptr_t>(addr)) = v;
}

// Workgroup barriers: every wave's direct loads have landed and its LDS accesses are done; or the latter alone.
__device__ __forceinline__ void pipeline_barrier() {
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}
__device__ __forceinline__ void lds_barrier() {
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

// x / d for x < 2^31 as x * mul >> shift: mul = ceil(2^(31 + s) / d) with 2^s >= d.  mul d exceeds 2^(31 + s) by less than d <= 2^s,
// so x mul / 2^(31 + s) exceeds x / d by less than x / (2^31 d) < 1 / d, and its whole part is the quotient.
struct Divisor {
  uint32_t mul, shift;
  __device__ __forceinline__ uint32_t of(uint32_t x) const { return static_cast<uint32_t>(static_cast<uint64_t>(x) * mul >> shift); }
};
inline Divisor divisor(int64_t d) {
  uint32_t s = 0;
  while ((int64_t{1} << s) < d) ++s;
  return {static_cast<uint32_t>(((uint64_t{1} << (31 + s)) + d - 1) / d), 31 + s};
}

// The cache as the kernels address it (byte strides).
struct Cache {
  const char* k;
  const char* v;
  const int32_t* pages;
  int64_t pages_stride;
  int64_t k_page, k_row, k_head;
  int64_t v_page, v_row, v_head;
  uint32_t n_pages, page_size, max_len;  // max_len: positions a page table row has room for
  Divisor by_page;  // key / page_size
};

// ---- host ---------------------------------------------------------------------
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool stride_ok(int64_t s) { return s >= 0 && s % 8 == 0 && s <= int64_t{1} << 40; }

// Sizes every call shares.
inline int check_heads(int64_t n_head, int64_t n_kv_head, int64_t head_dim, int32_t dtype) {
  if (n_kv_head <= 0 || n_head < 0 || head_dim <= 0) return LATENT_E_INVALID;
  if (n_head % n_kv_head) return LATENT_E_INVALID;
  if (dtype != LATENT_F16 && dtype != LATENT_BF16) return LATENT_E_INVALID;
  if (head_dim % 8 || head_dim > kMaxDim || n_head > 1024 || n_kv_head > 1024) return LATENT_E_UNSUPPORTED;
  return LATENT_OK;
}

inline int check_cache(const latent_kv_cache& c) {
  if (c.n_pages < 0 || c.page_size <= 0 || c.max_pages < 0 || c.n_seq < 0) return LATENT_E_INVALID;
  if (c.n_pages > INT32_MAX || c.page_size > INT32_MAX || c.n_seq > (1 << 20)) return LATENT_E_UNSUPPORTED;
  if (c.max_pages > INT32_MAX || c.max_pages * c.page_size > INT32_MAX - 1024) return LATENT_E_UNSUPPORTED;
  if (c.n_seq > 1 && c.pages_stride < c.max_pages) return LATENT_E_INVALID;
  for (int64_t s : {c.k_page_stride, c.k_row_stride, c.k_head_stride, c.v_page_stride, c.v_row_stride, c.v_head_stride})
    if (!stride_ok(s)) return LATENT_E_UNSUPPORTED;
  if (!aligned16(c.k) || !aligned16(c.v)) return LATENT_E_UNSUPPORTED;
  return LATENT_OK;
}

inline Cache device_cache(const latent_kv_cache& c) {
  Cache d{};
  d.k = static_cast<const char*>(c.k);
  d.v = static_cast<const char*>(c.v);
  d.pages = c.pages;
  d.pages_stride = c.pages_stride;
  d.k_page = c.k_page_stride * 2;
  d.k_row = c.k_row_stride * 2;
  d.k_head = c.k_head_stride * 2;
  d.v_page = c.v_page_stride * 2;
  d.v_row = c.v_row_stride * 2;
  d.v_head = c.v_head_stride * 2;
  d.n_pages = static_cast<uint32_t>(c.n_pages);
  d.page_size = static_cast<uint32_t>(c.page_size);
  d.max_len = static_cast<uint32_t>(c.max_pages * c.page_size);
  d.by_page = divisor(c.page_size);
  return d;
}

}  // namespace attend
}  // namespace latent
