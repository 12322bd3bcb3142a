// gpt2_w4.hip — linear layers with 4-bit weights and a scale for each group of
// inputs: quantising, the values back, and the entry points (gfx950).
#include "gpt2_w4.h"
#include "dfattn_status.h"

#include <initializer_list>
#include <string>
#include <type_traits>

namespace dfattn {
namespace {

using namespace w4;

constexpr uint32_t kMaxFeatures = 1u << 24;

// The value of code c (0..15) before its scale.
template <Format F>
__device__ __forceinline__ float code_value(unsigned c, float zero) {
  if constexpr (F == kE2M1) {
    // 0 1/2 1 3/2 2 3 4 6: from 2 on an exponent and one bit, below multiples of 1/2.
    const unsigned m = c & 7;
    const float v = m < 2 ? 0.5f * m : __uint_as_float((126 + (m >> 1)) << 23 | (m & 1) << 22);
    return c & 8 ? -v : v;
  } else {
    return (float)c - zero;
  }
}

// ---------------------------------------------------------------- quantise
struct QuantArgs {
  const void *w;
  unsigned *codes;
  unsigned short *scales;
  unsigned char *zeros;
  void *out;
  size_t stride;
  uint32_t N, K, log_group, row_dwords, column_blocks;
};

// The nearest bf16 to q >= 0, ties to even: by way of the float below it with the rest in its
// last bit, so that the second rounding sees what the first left out.
__device__ __forceinline__ unsigned short nearest_bf16(double q) {
  float f = __double2float_rz(q);
  if ((double)f != q) f = __uint_as_float(__float_as_uint(f) | 1u);
  return bf16_bits(f);
}

// x / s to the nearest whole number, ties to even, for a bf16 s > 0 and |x| up to some 16 s: x times the
// hardware's 1 / s (one unit in the last place off) is at most one off after rounding, and the remainder
// x - c s is exact (c s has at most 13 bits, and where c is not 0 it is within a factor of two of x).
struct Divider {
  float f, s, inv, half;
  __device__ __forceinline__ explicit Divider(float scale) {
    f = scale < 0x1p-100f ? 0x1p64f : 1.f;  // (1 / s would be infinite)
    s = scale * f;
    inv = __builtin_amdgcn_rcpf(s);
    half = 0.5f * s;
  }
  __device__ __forceinline__ float nearest(float x) const {
    x *= f;
    float c = __builtin_rintf(x * inv);
    const float r = fmaf(-c, s, x);
    const bool odd = ((int)c & 1) != 0;
    if (fabsf(r) > half || (fabsf(r) == half && odd)) c += r > 0.f ? 1.f : -1.f;
    return c;
  }
  // The same without the correction; *far grows to the largest remainder. Right for all x where that stays below near().
  __device__ __forceinline__ float first(float x, float *far) const {
    const float c = __builtin_rintf(x * inv);
    *far = fmaxf(*far, fabsf(fmaf(-c, s, x)));
    return c;
  }
  __device__ __forceinline__ float near() const { return f == 1.f ? half * (1.f - 0x1p-20f) : 0.f; }
};

// A workgroup takes 32 outputs and 256 inputs: a lane 8 inputs of four outputs, 4 to 16 neighbours a
// group. Each of four neighbours divides for one of the four outputs. The scales go through LDS, so that neighbouring
// outputs' are written together.
// Bound: from fp32 memory (16384 x 4096 to u4 55 us, 5.5 TB/s, VALU busy 53 % of the time), from bf16 VALU (u4 46 to 54 us, 3.1 to 3.7
// TB/s, i4 41; busy 95 % of the time in both): extremes, one double division a group and four neighbours, the product, its
// check and clamp for each value, and the correction, which three of five rows of a wave take where values have bf16's 8 bits (0.2 % of
// them are half way; from fp32 hardly any). 768 x 768 4 to 6 us, a launch's latency. Workgroups of several blocks with the next one's loads ahead were slower (63 us, then 54 without).
constexpr int kQuantRows = 32, kQuantCols = 256;
template <Format F, bool BF16>
__global__ __launch_bounds__(kThreads) void quantize_kernel(QuantArgs a) {
  __shared__ unsigned short scale_lds[kQuantCols / 32][kQuantRows];
  __shared__ unsigned char zero_lds[kQuantCols / 32][kQuantRows];
  const uint32_t block = linear_block(), n0 = block / a.column_blocks * kQuantRows, k0 = block % a.column_blocks * kQuantCols;
  if (n0 >= a.N) return;
  const uint32_t lane = threadIdx.x & 31, d = k0 / 8 + lane, lanes = 1u << (a.log_group - 3);
  float x[4][8];
  const char *w = static_cast<const char *>(a.w) + ((n0 + (threadIdx.x >> 5)) * a.stride + d * 8) * (BF16 ? 2 : 4);
  const size_t rows8 = 8 * a.stride * (BF16 ? 2 : 4);
  if (n0 + kQuantRows <= a.N && k0 + kQuantCols <= a.K) {
    if constexpr (BF16) {  // (all loads before the first use)
      unsigned v[4][4];
#pragma unroll
      for (int r = 0; r < 4; ++r) __builtin_memcpy(v[r], w + r * rows8, 16);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < 8; ++j) x[r][j] = __uint_as_float(j & 1 ? v[r][j / 2] & 0xffff0000u : v[r][j / 2] << 16);
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) __builtin_memcpy(x[r], w + r * rows8, 32);
    }
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        x[r][j] = n0 + 8 * r + (threadIdx.x >> 5) < a.N && d * 8 + j < a.K ? load_value<BF16>(w + r * rows8, j) : 0.f;
  }
  // The groups' extremes over 4, 8 or 16 neighbouring lanes: with zero points the lowest and highest, where a NaN goes on, else
  // the largest magnitude by its bits (an infinity or NaN is above all numbers).
  auto among = [&](auto v, auto better) {
    v = better(v, dpp<0xb1>(v));
    v = better(v, dpp<0x4e>(v));
    if (lanes > 4) v = better(v, dpp<0x141>(v));
    if (lanes > 8) v = better(v, dpp<0x140>(v));
    return v;
  };
  auto lower = [](float x, float y) { return __builtin_elementwise_minimum(x, y); };
  auto higher = [](float x, float y) { return __builtin_elementwise_maximum(x, y); };
  float lo[4], hi[4];
  unsigned most[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    lo[r] = hi[r] = 0.f;
    most[r] = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (F == kU4) {
        lo[r] = lower(lo[r], x[r][j]);
        hi[r] = higher(hi[r], x[r][j]);
      } else {
        most[r] = max(most[r], __float_as_uint(x[r][j]) & 0x7fffffffu);
      }
    }
    if (F == kU4) {
      lo[r] = among(lo[r], lower);
      hi[r] = among(hi[r], higher);
      most[r] = max(__float_as_uint(lo[r]) & 0x7fffffffu, __float_as_uint(hi[r]) & 0x7fffffffu);
    } else {
      most[r] = among(most[r], [](unsigned a, unsigned b) { return max(a, b); });
    }
  }
  const uint32_t which = lane & 3;
  float low = lo[0], high = F == kU4 ? hi[0] : __uint_as_float(most[0]);
#pragma unroll
  for (uint32_t r = 1; r < 4; ++r) {
    low = which == r ? lo[r] : low;
    high = which == r ? F == kU4 ? hi[r] : __uint_as_float(most[r]) : high;
  }
  const double top = F == kU4 ? ((double)high - (double)low) / 15.0 : (double)high / (F == kI4 ? 7.0 : 6.0);
  unsigned near = nearest_bf16(top);
  if (F == kU4 && near != 0) near |= (unsigned)fminf(fmaxf(Divider(bf16_value((unsigned short)near)).nearest(-low), 0.f), 15.f) << 16;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const uint32_t row = 8 * r + (threadIdx.x >> 5), n = n0 + row;
    const unsigned theirs = (unsigned)__shfl((int)near, (int)((threadIdx.x & 63 & ~3u) + r), 64);  // scale, and zero point above
    const unsigned short bits = most[r] >= 0x7f800000u ? 0x7fc0u : (unsigned short)theirs;
    const float s = bf16_value(bits);
    const bool some = s > 0.f;  // (neither 0 nor NaN)
    const Divider by(some ? s : 1.f);
    float zero = F == kI4 ? 8.f : 0.f;
    if (F == kU4 && some) zero = (float)(theirs >> 16);
    float v[8], far = 0.f;
    if constexpr (F != kE2M1) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = by.first(x[r][j], &far);
      // (Few fp32 values are next to a border: with the correction always 3 of 70 us more.)
      if (__any(some && !(far < by.near()))) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = by.nearest(x[r][j]);
      }
    }
    unsigned c = 0;
    if constexpr (F == kE2M1) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float y = fabsf(x[r][j]);
        const unsigned q = (y > 0.25f * s) + (y >= 0.75f * s) + (y > 1.25f * s) + (y >= 1.75f * s) + (y > 2.5f * s) +
                           (y >= 3.5f * s) + (y > 5.f * s);
        c |= (some ? q | (__float_as_uint(x[r][j]) >> 31 << 3) : 0u) << (4 * j);
      }
    } else {  // (four codes are a float's 16 bits)
      float low = 0.f, high = 0.f;
#pragma unroll
      for (int j = 3; j >= 0; --j) {
        low = fmaf(low, 16.f, fminf(fmaxf((some ? v[j] : 0.f) + zero, 0.f), 15.f));
        high = fmaf(high, 16.f, fminf(fmaxf((some ? v[j + 4] : 0.f) + zero, 0.f), 15.f));
      }
      c = (unsigned)low | (unsigned)high << 16;
    }
    if (n < a.N && d < a.row_dwords) a.codes[(size_t)n * a.row_dwords + d] = c;
    if ((lane & (lanes - 1)) == 0) {
      scale_lds[lane / lanes][row] = bits;
      if (F == kU4) zero_lds[lane / lanes][row] = (unsigned char)zero;
    }
  }
  __syncthreads();
  const uint32_t g = threadIdx.x >> 5, n = n0 + lane, at = (k0 >> a.log_group) + g;
  if (g >= (uint32_t)kQuantCols >> a.log_group || n >= a.N || (size_t)at << a.log_group >= a.K) return;
  a.scales[(size_t)at * a.N + n] = scale_lds[g][lane];
  if (F == kU4) a.zeros[(size_t)at * a.N + n] = zero_lds[g][lane];
}

// ---------------------------------------------------------------- values
// A lane writes 16 bytes at a time, neighbours next to each other: 4 fp32 or 8 bf16 values of a row; kValueSteps
// times 256 lanes a workgroup. Bound: to fp32 the stores (16384 x 4096 47 us into the same memory each time, part of which stays in the
// Infinity Cache, 70 us into four in turn, 4.3 TB/s); to bf16 neither memory nor VALU (46 us, 3.7 TB/s, 56 %): each wave loads,
// computes and stores in turn. 768 x 768 to fp32 3.8 us, to bf16, with half the workgroups, 5.7.
constexpr uint32_t kValueSteps = 8;
template <Format F, bool BF16>
__global__ __launch_bounds__(kThreads) void dequantize_kernel(QuantArgs a) {
  constexpr uint32_t V = BF16 ? 8 : 4;
  const uint32_t per_row = (a.K + V - 1) / V;
  const size_t base = (size_t)linear_block() * (kThreads * kValueSteps), row0 = base / per_row;
  const uint32_t at0 = (uint32_t)(base % per_row);
  const unsigned char *codes = reinterpret_cast<const unsigned char *>(a.codes);
  size_t n[kValueSteps];
  uint32_t k[kValueSteps];
  unsigned c[kValueSteps];
  float scale[kValueSteps], zero[kValueSteps];
#pragma unroll
  for (uint32_t i = 0; i < kValueSteps; ++i) {  // (all loads before the first use)
    const uint32_t at = at0 + i * kThreads + threadIdx.x;
    k[i] = at % per_row * V;
    n[i] = row0 + at / per_row;
    const size_t row = min(n[i], (size_t)a.N - 1), group = (size_t)(k[i] >> a.log_group) * a.N + row;
    if constexpr (BF16)
      c[i] = *reinterpret_cast<const unsigned *>(codes + row * a.row_dwords * 4 + k[i] / 2);
    else
      c[i] = *reinterpret_cast<const unsigned short *>(codes + row * a.row_dwords * 4 + k[i] / 2);
    scale[i] = bf16_value(a.scales[group]);
    zero[i] = F == kU4 ? (float)a.zeros[group] : 8.f;
  }
#pragma unroll
  for (uint32_t i = 0; i < kValueSteps; ++i) {
    if (n[i] >= a.N) break;
    float v[V];
#pragma unroll
    for (uint32_t j = 0; j < V; ++j) v[j] = code_value<F>(c[i] >> (4 * j) & 15u, zero[i]) * scale[i];
    if (k[i] + V <= a.K) {
      u32x4 o;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        o[j] = BF16 ? (unsigned)bf16_bits(v[2 * j % V]) | (unsigned)bf16_bits(v[(2 * j + 1) % V]) << 16 : __float_as_uint(v[j]);
      __builtin_memcpy(static_cast<char *>(a.out) + (n[i] * a.K + k[i]) * (BF16 ? 2 : 4), &o, 16);
    } else {
#pragma unroll
      for (uint32_t j = 0; j < V; ++j)
        if (k[i] + j < a.K) store_value<BF16>(a.out, n[i] * a.K + k[i] + j, v[j]);
    }
  }
}

// ---------------------------------------------------------------- host
template <typename G>
void by_format(uint32_t format, uint32_t dtype, G go) {
  auto with = [&](auto f) {
    if (dtype == DFATTN_KV_BF16)
      go(f, std::true_type{});
    else
      go(f, std::false_type{});
  };
  if (format == DFGPT2_W4_I4)
    with(std::integral_constant<Format, kI4>{});
  else if (format == DFGPT2_W4_U4)
    with(std::integral_constant<Format, kU4>{});
  else
    with(std::integral_constant<Format, kE2M1>{});
}

int check_weights(const char *fn, const void *codes, const uint16_t *scales, const void *zeros, uint32_t dtype,
                  uint32_t format, uint32_t group, uint32_t out_features, uint32_t in_features) {
  const std::string at = std::string(fn) + ": ";
  if (dtype != DFATTN_KV_F32 && dtype != DFATTN_KV_BF16)
    return record_error(DFATTN_ERR_FLAGS, at + "dtype must be DFATTN_KV_F32 or DFATTN_KV_BF16");
  if (format > DFGPT2_W4_E2M1) return record_error(DFATTN_ERR_FLAGS, at + "format must be one of DFGPT2_W4_*");
  if (group != 32 && group != 64 && group != 128)
    return record_error(DFATTN_ERR_SHAPE, at + "a group has 32, 64 or 128 inputs");
  if (out_features == 0 || in_features == 0)
    return record_error(DFATTN_ERR_SHAPE, at + "out_features and in_features must be >= 1");
  if (out_features > kMaxFeatures || in_features > kMaxFeatures)
    return record_error(DFATTN_ERR_OVERFLOW, at + "shape is too large");
  if (codes == nullptr || scales == nullptr || (format == DFGPT2_W4_U4 && zeros == nullptr))
    return record_error(DFATTN_ERR_NULL_POINTER, at + "null pointer");
  if (reinterpret_cast<uintptr_t>(codes) % 16 != 0 || reinterpret_cast<uintptr_t>(scales) % 2 != 0)
    return record_error(DFATTN_ERR_MISALIGNED, at + "misaligned pointer");
  return DFATTN_OK;
}

int need(const char *fn, std::initializer_list<const void *> ptrs, size_t align) {
  for (const void *p : ptrs)
    if (p == nullptr) return record_error(DFATTN_ERR_NULL_POINTER, std::string(fn) + ": null pointer");
  for (const void *p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) % align != 0)
      return record_error(DFATTN_ERR_MISALIGNED, std::string(fn) + ": misaligned pointer");
  return DFATTN_OK;
}

int launched(const char *fn) {
  const hipError_t err = hipGetLastError();
  if (err == hipSuccess) return DFATTN_OK;
  return record_error(DFATTN_ERR_HIP, std::string(fn) + ": " + hipGetErrorString(err));
}

struct Span {
  const void *p;
  size_t bytes;
};
bool overlap(const Span &x, const Span &y) {
  const char *a = static_cast<const char *>(x.p), *b = static_cast<const char *>(y.p);
  return a != nullptr && b != nullptr && a < b + y.bytes && b < a + x.bytes;
}

uint32_t log2_of(uint32_t group) { return group == 32 ? 5 : group == 64 ? 6 : 7; }
uint32_t dwords_of(uint32_t in_features) { return (in_features + 31) / 32 * 4; }

}  // namespace
}  // namespace dfattn

using namespace dfattn;
using namespace dfattn::w4;

extern "C" {

size_t dfgpt2_w4_row_bytes(uint32_t in_features) { return in_features > kMaxFeatures ? 0 : 4 * (size_t)dwords_of(in_features); }

int dfgpt2_w4_quantize(const void *w, void *codes, uint16_t *scales, void *zeros, uint32_t dtype, uint32_t format,
                       uint32_t group, uint32_t out_features, uint32_t in_features, uint32_t row_stride,
                       hipStream_t stream) {
  const char *fn = "dfgpt2_w4_quantize";
  int st = check_weights(fn, codes, scales, zeros, dtype, format, group, out_features, in_features);
  if (st == DFATTN_OK) st = need(fn, {w}, dtype == DFATTN_KV_F32 ? 4 : 2);
  if (st != DFATTN_OK) return st;
  if (row_stride < in_features)
    return record_error(DFATTN_ERR_SHAPE, std::string(fn) + ": row_stride must be at least in_features");
  const size_t item = dtype == DFATTN_KV_F32 ? 4 : 2, groups = (in_features + group - 1) / group;
  const Span spans[] = {{codes, (size_t)out_features * dwords_of(in_features) * 4}, {scales, 2 * groups * out_features},
                        {format == DFGPT2_W4_U4 ? zeros : nullptr, groups * out_features},
                        {w, ((size_t)(out_features - 1) * row_stride + in_features) * item}};
  for (int i = 0; i < 3; ++i)
    for (int j = i + 1; j < 4; ++j)
      if (overlap(spans[i], spans[j]))
        return record_error(DFATTN_ERR_SHAPE, std::string(fn) + ": outputs must not overlap inputs or each other");
  QuantArgs a{w, static_cast<unsigned *>(codes), scales, static_cast<unsigned char *>(zeros), nullptr, row_stride,
              out_features, in_features, log2_of(group), dwords_of(in_features), (in_features + kQuantCols - 1) / kQuantCols};
  const dim3 grid = linear_grid((size_t)((out_features + kQuantRows - 1) / kQuantRows) * a.column_blocks);
  by_format(format, dtype, [&](auto f, auto bf16) {
    hipLaunchKernelGGL((quantize_kernel<decltype(f)::value, decltype(bf16)::value>), grid, dim3(kThreads), 0, stream, a);
  });
  return launched(fn);
}

int dfgpt2_w4_dequantize(const void *codes, const uint16_t *scales, const void *zeros, void *w, uint32_t dtype,
                         uint32_t format, uint32_t group, uint32_t out_features, uint32_t in_features,
                         hipStream_t stream) {
  const char *fn = "dfgpt2_w4_dequantize";
  int st = check_weights(fn, codes, scales, zeros, dtype, format, group, out_features, in_features);
  if (st == DFATTN_OK) st = need(fn, {w}, dtype == DFATTN_KV_F32 ? 4 : 2);
  if (st != DFATTN_OK) return st;
  const size_t item = dtype == DFATTN_KV_F32 ? 4 : 2, groups = (in_features + group - 1) / group;
  const Span to{w, (size_t)out_features * in_features * item};
  if (overlap(to, {codes, (size_t)out_features * dwords_of(in_features) * 4}) ||
      overlap(to, {scales, 2 * groups * out_features}) || (format == DFGPT2_W4_U4 && overlap(to, {zeros, groups * out_features})))
    return record_error(DFATTN_ERR_SHAPE, std::string(fn) + ": w must not overlap what is read");
  QuantArgs a{nullptr, static_cast<unsigned *>(const_cast<void *>(codes)), const_cast<uint16_t *>(scales),
              static_cast<unsigned char *>(const_cast<void *>(zeros)), w, 0, out_features, in_features, log2_of(group),
              dwords_of(in_features), 0};
  const size_t values = dtype == DFATTN_KV_F32 ? 4 : 8, lanes = (size_t)out_features * ((in_features + values - 1) / values);
  by_format(format, dtype, [&](auto f, auto bf16) {
    hipLaunchKernelGGL((dequantize_kernel<decltype(f)::value, decltype(bf16)::value>),
                       linear_grid((lanes + kThreads * kValueSteps - 1) / (kThreads * kValueSteps)), dim3(kThreads), 0, stream, a);
  });
  return launched(fn);
}

size_t dfgpt2_w4_linear_workspace_bytes(uint32_t rows, uint32_t in_features, uint32_t out_features) {
  if (rows == 0 || rows > (1u << 20) || in_features == 0 || in_features > kMaxFeatures || out_features == 0 ||
      out_features > kMaxFeatures)
    return 0;
  if (path_of(rows, out_features, in_features, false) != kMatrix) return 0;  // (then nor is it with bf16)
  const uint32_t splits = splits_of(rows, out_features, in_features);
  return splits == 1 ? 0 : 4 * (size_t)splits * rows * out_features;
}

int dfgpt2_w4_linear(const void *x, const void *codes, const uint16_t *scales, const void *zeros, const float *bias,
                     const void *residual, void *out, uint32_t dtype, uint32_t format, uint32_t group, uint32_t rows,
                     uint32_t in_features, uint32_t out_features, uint32_t row_stride, uint32_t gelu,
                     void *workspace, size_t workspace_bytes, hipStream_t stream) {
  const char *fn = "dfgpt2_w4_linear";
  int st = check_weights(fn, codes, scales, zeros, dtype, format, group, out_features, in_features);
  if (st != DFATTN_OK) return st;
  if (row_stride < in_features)
    return record_error(DFATTN_ERR_SHAPE, std::string(fn) + ": row_stride must be at least in_features");
  if (rows > (1u << 20) || (uint64_t)rows * out_features > (1ull << 40) || row_stride > (1u << 28))
    return record_error(DFATTN_ERR_OVERFLOW, std::string(fn) + ": shape is too large");
  if (rows == 0) return DFATTN_OK;
  const size_t item = dtype == DFATTN_KV_F32 ? 4 : 2, groups = (in_features + group - 1) / group;
  const size_t need_bytes = dfgpt2_w4_linear_workspace_bytes(rows, in_features, out_features);
  if (workspace != nullptr && workspace_bytes < need_bytes)
    return record_error(DFATTN_ERR_WORKSPACE, std::string(fn) + ": the workspace is too small");
  st = need(fn, {x, out}, item);
  if (st == DFATTN_OK && workspace != nullptr && need_bytes > 0) st = need(fn, {workspace}, 4);
  if (st == DFATTN_OK && bias != nullptr) st = need(fn, {bias}, 4);
  if (st == DFATTN_OK && residual != nullptr) st = need(fn, {residual}, item);
  if (st != DFATTN_OK) return st;
  const Span to{out, (size_t)rows * out_features * item}, sums_to{need_bytes > 0 ? workspace : nullptr, need_bytes};
  const Span read[] = {{x, ((size_t)(rows - 1) * row_stride + in_features) * item}, {codes, (size_t)out_features * dwords_of(in_features) * 4},
                       {scales, 2 * groups * out_features}, {format == DFGPT2_W4_U4 ? zeros : nullptr, groups * out_features},
                       {bias, 4 * (size_t)out_features}, {residual, to.bytes}};
  bool clash = overlap(to, sums_to);
  for (const Span &r : read) clash |= overlap(sums_to, r) || (overlap(to, r) && !(r.p == residual && residual == out));
  if (clash)
    return record_error(DFATTN_ERR_SHAPE, std::string(fn) + ": out must not overlap what is read, or be the residual itself; the workspace neither");
  LinearArgs a{x, static_cast<const unsigned char *>(codes), scales,
               static_cast<const unsigned char *>(zeros), bias, residual, out, nullptr, row_stride,
               rows, out_features, in_features, 4 * dwords_of(in_features), (uint32_t)groups, log2_of(group), 1, 1, (int)gelu};
  float *sums = need_bytes > 0 ? static_cast<float *>(workspace) : nullptr;
  const bool bf16 = dtype == DFATTN_KV_BF16;
  if (format == DFGPT2_W4_I4)
    launch_linear_format<kI4>(a, bf16, group, sums, stream);
  else if (format == DFGPT2_W4_U4)
    launch_linear_format<kU4>(a, bf16, group, sums, stream);
  else
    launch_linear_format<kE2M1>(a, bf16, group, sums, stream);
  return launched(fn);
}

}  // extern "C"
