// kv8.h — what the 8-bit paged cache's kernels share: codes, scales, the pool
// layout and the host checks.
//
// Pools: K [n_pages, n_kv_heads, page_size, Dp] and V [n_pages, n_kv_heads, Dp,
// page_size] codes (one byte), Dp = d_head rounded up to 16; scales [n_pages,
// n_kv_heads] fp32. value = code * scale.
#pragma once

#include "dfattn.h"
#include "dfattn_internal.h"
#include "dfattn_status.h"

#include <initializer_list>
#include <string>

namespace dfattn {
namespace kv8 {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

inline __host__ __device__ int padded(int d) { return (d + 15) & ~15; }

// Largest code magnitude: 127 = 127/128 * 2^7 (int8), 448 = 7/8 * 2^9 (e4m3).
template <bool E4M3>
__device__ __forceinline__ float pow2_scale(float amax) {
  // The smallest 2^e >= 2^-126 with amax <= limit * 2^e: with amax = m 2^x,
  // m in [1/2, 1), that is e = x - bits, one more where m is above limit / 2^bits.
  int x;
  const float m = frexpf(amax, &x);
  const int e = E4M3 ? x - 9 + (m > 0.875f) : x - 7 + (m > 0.9921875f);
  return __uint_as_float((unsigned)(max(amax > 0.f ? e : -126, -126) + 127) << 23);
}

// Four values of four codes.
template <bool E4M3>
__device__ __forceinline__ float4 decode4(unsigned c) {
  if constexpr (E4M3) {
    return make_float4(__builtin_amdgcn_cvt_f32_fp8(c, 0), __builtin_amdgcn_cvt_f32_fp8(c, 1),
                       __builtin_amdgcn_cvt_f32_fp8(c, 2), __builtin_amdgcn_cvt_f32_fp8(c, 3));
  } else {
    const int i = (int)c;
    return make_float4((float)(i << 24 >> 24), (float)(i << 16 >> 24), (float)(i << 8 >> 24), (float)(i >> 24));
  }
}
// Four codes of four values already divided by their scale (|x| at most the
// largest code), to the nearest, ties to even.
template <bool E4M3>
__device__ __forceinline__ unsigned encode4(float4 v) {
  if constexpr (E4M3) {
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(v.x, v.y, 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v.z, v.w, c, true);
  } else {
    auto r = [](float x) { return (unsigned)(int)__builtin_rintf(x) & 0xffu; };
    return r(v.x) | r(v.y) << 8 | r(v.z) << 16 | r(v.w) << 24;
  }
}

// bf16 bits of a float, to the nearest, ties to even; a NaN stays one.
__device__ __forceinline__ unsigned bf16_bits(float f) {
  const unsigned u = __float_as_uint(f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return (u >> 16) | 0x40u;
  return (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
}
__device__ __forceinline__ float load_act(const void *p, size_t i, bool bf16) {
  return bf16 ? __uint_as_float((unsigned)static_cast<const unsigned short *>(p)[i] << 16)
              : static_cast<const float *>(p)[i];
}

// ---- host ----
inline bool aligned_to(const void *p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

inline int check_types(const char *fn, uint32_t act_dtype, uint32_t kv_dtype) {
  if (act_dtype != DFATTN_KV_F32 && act_dtype != DFATTN_KV_BF16)
    return record_error(DFATTN_ERR_FLAGS, std::string(fn) + ": act_dtype must be DFATTN_KV_F32 or DFATTN_KV_BF16");
  if (kv_dtype != DFATTN_KV_I8 && kv_dtype != DFATTN_KV_E4M3)
    return record_error(DFATTN_ERR_FLAGS, std::string(fn) + ": kv_dtype must be DFATTN_KV_I8 or DFATTN_KV_E4M3");
  return DFATTN_OK;
}

// The pool's shape; *row_bytes = n_kv_heads * Dp, a position's bytes in one pool.
inline int check_pool_shape(const char *fn, uint32_t n_pages, uint32_t n_kv_heads, uint32_t page_size, uint32_t d_head) {
  if (n_pages == 0 || n_kv_heads == 0)
    return record_error(DFATTN_ERR_SHAPE, std::string(fn) + ": n_pages and n_kv_heads must be >= 1");
  if (page_size == 0 || page_size % 16 != 0 || page_size > 256)
    return record_error(DFATTN_ERR_SHAPE, std::string(fn) + ": page_size must be a multiple of 16 up to 256");
  if (d_head == 0 || d_head > 128)
    return record_error(DFATTN_ERR_HEAD_DIM, std::string(fn) + ": d_head must be in the range 1..=128");
  if (n_kv_heads > 65535u || (uint64_t)n_pages * page_size > (1ull << 31))
    return record_error(DFATTN_ERR_OVERFLOW, std::string(fn) + ": cache shape is too large");
  return DFATTN_OK;
}

inline int check_all(const char *fn, std::initializer_list<const void *> ptrs, size_t align) {
  for (const void *p : ptrs)
    if (p == nullptr) return record_error(DFATTN_ERR_NULL_POINTER, std::string(fn) + ": null pointer");
  for (const void *p : ptrs)
    if (!aligned_to(p, align)) return record_error(DFATTN_ERR_MISALIGNED, std::string(fn) + ": misaligned pointer");
  return DFATTN_OK;
}

inline int launched(const char *fn) {
  const hipError_t err = hipGetLastError();
  if (err == hipSuccess) return DFATTN_OK;
  return record_error(DFATTN_ERR_HIP, std::string(fn) + ": " + hipGetErrorString(err));
}

}  // namespace kv8
}  // namespace dfattn
