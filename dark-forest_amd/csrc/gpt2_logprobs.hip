// gpt2_logprobs.hip — log probabilities of given tokens with the row's entropy
// and its largest alternatives, and the logits' gradient (gfx950).
//
// Per row x: m = max x, S = sum exp(x - m), T = sum exp(x - m) (x - m);
// ln p_j = (x_j - m) - ln S, entropy = ln S - T / S.
#include "dfattn_internal.h"
#include "dfattn_status.h"
#include "dfgpt2.h"

#include <initializer_list>
#include <string>
#include <type_traits>

namespace dfattn {
namespace {

constexpr int kThreads = 1024;
constexpr uint32_t kMaxTop = 64;
constexpr uint32_t kMaxRows = 1u << 21;  // a grid of 1024-thread workgroups stays below 2^32 threads

struct LogprobArgs {
  const void *logits;
  const uint32_t *tokens;
  float *logprob, *entropy, *stats;
  uint32_t *top_ids;
  float *top_logprobs;
  size_t stride;
  int cols, k;
};

template <bool BF16>
__device__ __forceinline__ float load_logit(const void *p, size_t i) {
  if (BF16) return __uint_as_float((unsigned)static_cast<const unsigned short *>(p)[i] << 16);
  return static_cast<const float *>(p)[i];
}

// Order of the alternatives as an unsigned number: larger logits larger, both
// zeros alike, NaN above all.
__device__ __forceinline__ unsigned rank_of(float x) {
  if (x != x) return 0xffffffffu;
  const unsigned u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

template <typename T, typename F>
__device__ __forceinline__ T block_reduce(T v, T *scratch, F f) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = f(v, __shfl_xor(v, off, 64));
  __syncthreads();
  if (lane == 0) scratch[wave] = v;
  __syncthreads();
  T r = scratch[0];
#pragma unroll
  for (int w = 1; w < kThreads / 64; ++w) r = f(r, scratch[w]);
  return r;
}

// One workgroup per row: the maximum, the sums, then one alternative after the
// other (the largest (rank, lowest id) below the one before).
template <bool BF16>
__global__ __launch_bounds__(kThreads) void logprob_kernel(LogprobArgs a) {
  __shared__ float scratch[kThreads / 64];
  __shared__ unsigned long long scratch64[kThreads / 64];
  const size_t row = blockIdx.x, at = row * a.stride;
  const int tid = threadIdx.x, n = a.cols;
  auto fmax2 = [](float x, float y) { return x != x ? x : y != y ? y : fmaxf(x, y); };
  auto add = [](float x, float y) { return x + y; };
  float m = -INFINITY;
  for (int i = tid; i < n; i += kThreads) m = fmax2(m, load_logit<BF16>(a.logits, at + i));
  m = block_reduce(m, scratch, fmax2);
  float s = 0.f, t = 0.f;
  for (int i = tid; i < n; i += kThreads) {
    const float d = load_logit<BF16>(a.logits, at + i) - m, e = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(d * kLog2e);
    s += e;
    t += e == 0.f ? 0.f : e * d;
  }
  s = block_reduce(s, scratch, add);
  t = block_reduce(t, scratch, add);
  const float ln_s = m == -INFINITY ? 0.f : logf(s);
  auto logp = [&](float x) { return x == -INFINITY && ln_s == ln_s ? x : (x - m) - ln_s; };
  if (tid == 0) {
    const uint32_t token = a.tokens[row];
    a.logprob[row] = token < (uint32_t)n ? logp(load_logit<BF16>(a.logits, at + token)) : 0.f;
    if (a.entropy) a.entropy[row] = m == -INFINITY ? 0.f : ln_s - t / s;
    if (a.stats) {
      a.stats[2 * row] = m;
      a.stats[2 * row + 1] = ln_s;
    }
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < a.k; ++k) {
    unsigned long long best = 0;
    for (int i = tid; i < n; i += kThreads) {
      const unsigned long long key =
          (unsigned long long)rank_of(load_logit<BF16>(a.logits, at + i)) << 32 | (0xffffffffu - (unsigned)i);
      if (key < last || (k == 0)) best = key > best ? key : best;
    }
    best = block_reduce(best, scratch64, [](unsigned long long x, unsigned long long y) { return x > y ? x : y; });
    last = best;
    if (tid == 0) {
      const uint32_t id = 0xffffffffu - (uint32_t)best;
      a.top_ids[row * a.k + k] = id;
      a.top_logprobs[row * a.k + k] = logp(load_logit<BF16>(a.logits, at + id));
    }
  }
}

struct GradArgs {
  const void *logits;
  const uint32_t *tokens;
  const float *stats, *entropy, *g_logprob, *g_entropy;
  void *grad;
  size_t stride;
  int cols;
};

__device__ __forceinline__ unsigned short to_bf16(float f) {
  const unsigned u = __float_as_uint(f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return (unsigned short)((u >> 16) | 0x40u);
  return (unsigned short)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}

template <bool BF16>
__global__ __launch_bounds__(256) void logprob_grad_kernel(GradArgs a) {
  const size_t row = blockIdx.x;
  const float m = a.stats[2 * row], ln_s = a.stats[2 * row + 1], h = a.entropy[row];
  const float gl = a.g_logprob ? a.g_logprob[row] : 0.f, ge = a.g_entropy ? a.g_entropy[row] : 0.f;
  const uint32_t token = a.tokens[row];
  const bool hit = token < (uint32_t)a.cols;
  for (int i = (int)threadIdx.x; i < a.cols; i += 256) {
    const float x = load_logit<BF16>(a.logits, row * a.stride + i), lp = (x - m) - ln_s;
    const float p = x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(lp * kLog2e);
    float g = hit ? gl * (((uint32_t)i == token ? 1.f : 0.f) - p) : 0.f;
    if (p != 0.f) g -= ge * p * (lp + h);
    if (m == -INFINITY) g = 0.f;
    const size_t o = row * (size_t)a.cols + i;
    if (BF16)
      static_cast<unsigned short *>(a.grad)[o] = to_bf16(g);
    else
      static_cast<float *>(a.grad)[o] = g;
  }
}

int check(const char *fn, uint32_t dtype, uint32_t rows, uint32_t cols, uint32_t row_stride) {
  if (dtype != DFATTN_KV_F32 && dtype != DFATTN_KV_BF16)
    return record_error(DFATTN_ERR_FLAGS, std::string(fn) + ": dtype must be DFATTN_KV_F32 or DFATTN_KV_BF16");
  if (cols == 0) return record_error(DFATTN_ERR_SHAPE, std::string(fn) + ": row length must be >= 1");
  if (row_stride < cols) return record_error(DFATTN_ERR_SHAPE, std::string(fn) + ": row_stride must be at least cols");
  if (rows > kMaxRows || cols > (1u << 30))
    return record_error(DFATTN_ERR_OVERFLOW, std::string(fn) + ": shape is too large");
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

int optional(const char *fn, std::initializer_list<const void *> ptrs) {
  for (const void *p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) % 4 != 0)
      return record_error(DFATTN_ERR_MISALIGNED, std::string(fn) + ": misaligned pointer");
  return DFATTN_OK;
}

int launched(const char *fn) {
  const hipError_t err = hipGetLastError();
  if (err == hipSuccess) return DFATTN_OK;
  return record_error(DFATTN_ERR_HIP, std::string(fn) + ": " + hipGetErrorString(err));
}

}  // namespace
}  // namespace dfattn

using namespace dfattn;

extern "C" {

int dfgpt2_token_logprobs(const void *logits, const uint32_t *tokens, float *logprob, float *entropy, float *stats,
                          uint32_t *top_ids, float *top_logprobs, uint32_t dtype, uint32_t rows, uint32_t cols,
                          uint32_t row_stride, uint32_t top_k, hipStream_t stream) {
  const char *fn = "dfgpt2_token_logprobs";
  int st = check(fn, dtype, rows, cols, row_stride);
  if (st != DFATTN_OK) return st;
  if (top_k > kMaxTop || top_k > cols)
    return record_error(DFATTN_ERR_SHAPE, std::string(fn) + ": top_k must be at most 64 and at most cols");
  if (rows == 0) return DFATTN_OK;
  st = need(fn, {logits}, dtype == DFATTN_KV_F32 ? 4 : 2);
  if (st == DFATTN_OK) st = need(fn, {tokens, logprob}, 4);
  if (st == DFATTN_OK && top_k > 0) st = need(fn, {top_ids, top_logprobs}, 4);
  if (st == DFATTN_OK) st = optional(fn, {entropy, stats});
  if (st != DFATTN_OK) return st;
  LogprobArgs a{logits, tokens, logprob, entropy, stats, top_ids, top_logprobs, row_stride, (int)cols, (int)top_k};
  if (dtype == DFATTN_KV_BF16)
    hipLaunchKernelGGL(logprob_kernel<true>, dim3(rows), dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL(logprob_kernel<false>, dim3(rows), dim3(kThreads), 0, stream, a);
  return launched(fn);
}

int dfgpt2_token_logprobs_backward(const void *logits, const uint32_t *tokens, const float *stats, const float *entropy,
                                   const float *grad_logprob, const float *grad_entropy, void *grad_logits,
                                   uint32_t dtype, uint32_t rows, uint32_t cols, uint32_t row_stride,
                                   hipStream_t stream) {
  const char *fn = "dfgpt2_token_logprobs_backward";
  int st = check(fn, dtype, rows, cols, row_stride);
  if (st != DFATTN_OK) return st;
  if (rows == 0) return DFATTN_OK;
  st = need(fn, {logits, grad_logits}, dtype == DFATTN_KV_F32 ? 4 : 2);
  if (st == DFATTN_OK) st = need(fn, {tokens, stats, entropy}, 4);
  if (st == DFATTN_OK) st = optional(fn, {grad_logprob, grad_entropy});
  if (st != DFATTN_OK) return st;
  if (logits == grad_logits && row_stride != cols)
    return record_error(DFATTN_ERR_SHAPE, std::string(fn) + ": grad_logits may be logits only where row_stride is cols");
  GradArgs a{logits, tokens, stats, entropy, grad_logprob, grad_entropy, grad_logits, row_stride, (int)cols};
  if (dtype == DFATTN_KV_BF16)
    hipLaunchKernelGGL(logprob_grad_kernel<true>, dim3(rows), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL(logprob_grad_kernel<false>, dim3(rows), dim3(256), 0, stream, a);
  return launched(fn);
}

}  // extern "C"
