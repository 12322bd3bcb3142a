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

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr uint32_t kMaxTop = 64;
constexpr uint32_t kMaxRows = 1u << 21;
constexpr int kCandidates = 512;

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
__device__ __forceinline__ float logit_of_rank(unsigned r) {
  return r == 0xffffffffu ? __builtin_nanf("") : __uint_as_float(r & 0x80000000u ? r ^ 0x80000000u : ~r);
}
// One number whose order is that of the alternatives: rank, then the lowest id.
__device__ __forceinline__ unsigned long long key_of(float x, int i) {
  return (unsigned long long)rank_of(x) << 32 | (0xffffffffu - (unsigned)i);
}

// 16 bytes of a row: 4 fp32 or 8 bf16 logits, from any element's address.
typedef unsigned raw4 __attribute__((ext_vector_type(4)));
template <bool BF16>
constexpr int kPer = BF16 ? 8 : 4;
template <bool BF16>
__device__ __forceinline__ float logit_of(raw4 r, int w) {
  if (BF16) return __uint_as_float(w & 1 ? r[w >> 1] & 0xffff0000u : r[w >> 1] << 16);
  return __uint_as_float(r[w & 3]);
}
// Those of ids i0 .., all below n, and the last ones of a row, -infinity from n on.
template <bool BF16>
__device__ __forceinline__ raw4 load_group(const void *row, int i0) {
  raw4 r;
  __builtin_memcpy(&r, static_cast<const char *>(row) + (unsigned)i0 * (BF16 ? 2u : 4u), 16);
  return r;
}
template <bool BF16>
__device__ __forceinline__ raw4 load_end(const void *row, int i0, int n) {
  raw4 r;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if constexpr (BF16) {
      const unsigned lo = i0 + 2 * w < n ? static_cast<const unsigned short *>(row)[i0 + 2 * w] : 0xff80u;
      const unsigned hi = i0 + 2 * w + 1 < n ? static_cast<const unsigned short *>(row)[i0 + 2 * w + 1] : 0xff80u;
      r[w] = lo | hi << 16;
    } else {
      r[w] = i0 + w < n ? static_cast<const unsigned *>(row)[i0 + w] : 0xff800000u;
    }
  }
  return r;
}

// The row's groups of this thread: group j holds ids (j * kThreads + thread) *
// kPer; the last, partial one of the workgroup is apart. Up to G whole ones stay
// in registers; G = 0: read again by each pass.
template <bool BF16, int G>
struct Row {
  const void *row;
  int whole, first;
  raw4 r[G > 0 ? G : 1], end;
  static constexpr int kStep = kThreads * kPer<BF16>;
  __device__ __forceinline__ Row(const void *p, int n, int tid) : row(p), whole(n / kStep), first(tid * kPer<BF16>) {
    if constexpr (G > 0) {
#pragma unroll
      for (int j = 0; j < G; ++j)
        if (j < whole) r[j] = load_group<BF16>(row, j * kStep + first);
    }
    end = load_end<BF16>(row, whole * kStep + first, n);
  }
  // f(logits of a group, its first id); ids from n on are -infinity.
  template <typename F>
  __device__ __forceinline__ void each(F f) {
    if constexpr (G > 0) {
#pragma unroll
      for (int j = 0; j < G; ++j)
        if (j < whole) {
          // Not known to be the values of the pass before: the compiler would keep every widened one.
          asm volatile("" : "+v"(r[j].x), "+v"(r[j].y), "+v"(r[j].z), "+v"(r[j].w));
          f(r[j], j * kStep + first);
        }
    } else {
#pragma unroll 4
      for (int j = 0; j < whole; ++j) f(load_group<BF16>(row, j * kStep + first), j * kStep + first);
    }
    f(end, whole * kStep + first);
  }
};

struct Shared {
  float lane_max[kWaves][64], sum_s[kWaves], sum_t[kWaves], thr;
  unsigned n_cand, wave_equal[kWaves];
  unsigned long long cand[kCandidates], best[kWaves];
};

// One workgroup per row, in one pass over memory where the row fits the
// registers: the threads' maxima, the sums of exponentials, then the
// alternatives. For those, the k-th largest of the 64 lanes' maxima (a lane's
// over all waves) bounds the k-th largest logit from below, so the few logits
// at or above it are the candidates; each one's rank among them is its place.
template <bool BF16, int G>
__global__ __launch_bounds__(kThreads) void logprob_kernel(LogprobArgs a) {
  constexpr int W = kPer<BF16>;
  __shared__ Shared sh;
  const size_t row = blockIdx.x, at = row * a.stride;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = a.cols, k = a.k;
  const void *base = static_cast<const char *>(a.logits) + at * (BF16 ? 2 : 4);
  Row<BF16, G> x(base, n, tid);
  const uint32_t token = a.tokens[row];
  const float chosen = token < (uint32_t)n ? load_logit<BF16>(base, token) : 0.f;
  float mine = -INFINITY;
  x.each([&](raw4 r, int) {
#pragma unroll
    for (int w = 0; w < W; ++w) mine = fmaxf(mine, logit_of<BF16>(r, w));
  });
  sh.lane_max[wave][lane] = mine;
  if (tid == 0) sh.n_cand = 0;
  __syncthreads();
  float top = sh.lane_max[0][lane];
#pragma unroll
  for (int v = 1; v < kWaves; ++v) top = fmaxf(top, sh.lane_max[v][lane]);
  const float m = wave_max(top), m0 = m == -INFINITY ? 0.f : m;
  if (k > 0 && wave == kWaves - 1) {
    int above = 0;
#pragma unroll
    for (int j = 0; j < 64; ++j) {
      const float o = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(top), j));
      above += o > top || (o == top && j < lane);
    }
    if (above == k - 1) sh.thr = top;
  }
  // S = sum e^(x - m) and T = sum e^(x - m) (x - m) log2 e. A masked-out logit
  // adds 0 to T (0 times at least -200), a NaN makes both NaN.
  float s = 0.f, t = 0.f;
  x.each([&](raw4 r, int) {
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float y = (logit_of<BF16>(r, w) - m0) * kLog2e, e = __builtin_amdgcn_exp2f(y);
      s += e;
      t = fmaf(e, fmaxf(y, -200.f), t);
    }
  });
  s = wave_sum(s);
  t = wave_sum(t);
  if (lane == 0) {
    sh.sum_s[wave] = s;
    sh.sum_t[wave] = t;
  }
  __syncthreads();
  s = sh.sum_s[0];
  t = sh.sum_t[0];
#pragma unroll
  for (int v = 1; v < kWaves; ++v) {
    s += sh.sum_s[v];
    t += sh.sum_t[v];
  }
  const bool nan = s != s;
  const float ln_s = m == -INFINITY && !nan ? 0.f : logf(s);
  auto logp = [&](float v) { return v == -INFINITY && !nan ? v : (v - m0) - ln_s; };
  if (tid == 0) {
    a.logprob[row] = token < (uint32_t)n ? logp(chosen) : 0.f;
    if (a.entropy) a.entropy[row] = m == -INFINITY && !nan ? 0.f : ln_s - t * kLn2 / s;
    if (a.stats) {
      a.stats[2 * row] = nan ? ln_s : m;
      a.stats[2 * row + 1] = ln_s;
    }
  }
  if (k == 0) return;

  const float thr = sh.thr;
  auto put = [&](unsigned long long key, int place) {
    a.top_ids[row * k + place] = 0xffffffffu - (uint32_t)key;
    a.top_logprobs[row * k + place] = logp(logit_of_rank((unsigned)(key >> 32)));
  };
  // The candidates: what is at or above the bound, where there is room for it all; else
  // what is above it. A group of a thread's is looked through where its largest is.
  auto collect = [&](bool equal_too) {
    x.each([&](raw4 r, int i0) {
      float g = logit_of<BF16>(r, 0);
#pragma unroll
      for (int w = 1; w < W; ++w) g = fmaxf(g, logit_of<BF16>(r, w));
      if (g >= thr) {
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const float v = logit_of<BF16>(r, w);
          if ((v > thr || (equal_too && v == thr)) && i0 + w < n) {
            const unsigned c = atomicAdd(&sh.n_cand, 1u);
            if (c < kCandidates) sh.cand[c] = key_of(v, i0 + w);
          }
        }
      }
    });
    __syncthreads();
    return sh.n_cand;
  };
  unsigned c = kCandidates + 1;
  bool all = true;
  if (!nan) {
    c = collect(true);
    if (c > kCandidates) {
      all = false;
      __syncthreads();
      if (tid == 0) sh.n_cand = 0;
      __syncthreads();
      c = collect(false);
    }
  }
  if (c <= kCandidates) {
    // Four lanes a candidate, each against a quarter of them.
    for (unsigned i = tid >> 2; i < ((c + 15) & ~15u); i += kThreads / 4) {
      const unsigned long long key = i < c ? sh.cand[i] : 0;
      int place = 0;
      for (unsigned j = tid & 3; j < c; j += 4) place += sh.cand[j] > key;
      place += __shfl_xor(place, 1, 64);
      place += __shfl_xor(place, 2, 64);
      if ((tid & 3) == 0 && i < c && place < k) put(key, place);
    }
    if (all || (int)c >= k) return;
    // The rest equals the bound (a mask's value, say): the lowest ids of those.
    int found = (int)c;
    for (int i0 = 0; i0 < n && found < k; i0 += kThreads) {
      const int i = i0 + tid;
      const float v = i < n ? load_logit<BF16>(base, i) : 0.f;
      const bool eq = i < n && v == thr;
      const unsigned long long hits = __ballot(eq);
      __syncthreads();
      if (lane == 0) sh.wave_equal[wave] = __popcll(hits);
      __syncthreads();
      int place = found + __popcll(hits & ((1ull << lane) - 1));
      for (int v2 = 0; v2 < kWaves; ++v2) {
        if (v2 < wave) place += sh.wave_equal[v2];
        found += sh.wave_equal[v2];
      }
      if (eq && place < k) put(key_of(v, i), place);
    }
    return;
  }
  // NaN, or the large logits crowded into a few lanes: one alternative after the other.
  unsigned long long last = ~0ull;
  for (int j = 0; j < k; ++j) {
    unsigned long long best = 0;
    for (int i = tid; i < n; i += kThreads) {
      const unsigned long long key = key_of(load_logit<BF16>(base, i), i);
      if (key < last || j == 0) best = key > best ? key : best;
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      const unsigned long long o = __shfl_xor(best, off, 64);
      best = o > best ? o : best;
    }
    __syncthreads();
    if (lane == 0) sh.best[wave] = best;
    __syncthreads();
    best = sh.best[0];
#pragma unroll
    for (int v = 1; v < kWaves; ++v) best = sh.best[v] > best ? sh.best[v] : best;
    last = best;
    if (tid == 0) put(best, j);
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

// g_j = g_l 1[j = token] - p_j (g_l + g_h (ln p_j + H)), elementwise: bound by
// memory (a read and a write). 16 bytes a thread and step, from any element's
// address. Everything a workgroup reads of its part of the row is read before it
// is written, so the gradient may lie where the logits do.
constexpr int kGradSteps = 4;
template <bool BF16>
__global__ __launch_bounds__(256) void logprob_grad_kernel(GradArgs a) {
  constexpr int W = kPer<BF16>;
  const size_t row = blockIdx.x;
  const float m = a.stats[2 * row], ln_s = a.stats[2 * row + 1], h = a.entropy[row];
  const uint32_t token = a.tokens[row];
  const bool dead = m == -INFINITY;
  const float gl = a.g_logprob && token < (uint32_t)a.cols && !dead ? a.g_logprob[row] : 0.f;
  const float ge = a.g_entropy ? a.g_entropy[row] : 0.f, c = gl + ge * h, m0 = dead ? 0.f : m;
  const void *base = static_cast<const char *>(a.logits) + row * a.stride * (BF16 ? 2 : 4);
  char *out = static_cast<char *>(a.grad) + row * (size_t)a.cols * (BF16 ? 2 : 4);
  const int i1 = (int)blockIdx.y * (256 * W * kGradSteps) + (int)threadIdx.x * W;
  raw4 r[kGradSteps];
#pragma unroll
  for (int j = 0; j < kGradSteps; ++j)
    if (i1 + j * 256 * W < a.cols)
      r[j] = i1 + j * 256 * W + W <= a.cols ? load_group<BF16>(base, i1 + j * 256 * W)
                                            : load_end<BF16>(base, i1 + j * 256 * W, a.cols);
#pragma unroll
  for (int j = 0; j < kGradSteps; ++j) {
    const int i0 = i1 + j * 256 * W;
    if (i0 >= a.cols) break;
    float g[W];
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float lp = (logit_of<BF16>(r[j], w) - m0) - ln_s, p = __builtin_amdgcn_exp2f(lp * kLog2e);
      g[w] = ((uint32_t)(i0 + w) == token ? gl : 0.f) - p * fmaf(ge, fmaxf(lp, -1000.f), c);
    }
    raw4 o;
#pragma unroll
    for (int w = 0; w < 4; ++w)
      o[w] = BF16 ? (unsigned)to_bf16(g[(2 * w) % W]) | (unsigned)to_bf16(g[(2 * w + 1) % W]) << 16 : __float_as_uint(g[w]);
    if (i0 + W <= a.cols) {
      __builtin_memcpy(out + (size_t)i0 * (BF16 ? 2 : 4), &o, 16);
    } else {
#pragma unroll
      for (int w = 0; w < W; ++w)
        if (i0 + w < a.cols) {
          if constexpr (BF16)
            reinterpret_cast<unsigned short *>(out)[i0 + w] = (unsigned short)(o[w >> 1] >> (16 * (w & 1)));
          else
            reinterpret_cast<unsigned *>(out)[i0 + w] = o[w];
        }
    }
  }
}

// Rows of up to 1, 6, 12 and 24 whole groups a thread (and the partial one) stay in registers.
template <bool BF16>
void launch_logprobs(const LogprobArgs &a, uint32_t rows, hipStream_t s) {
  const int groups = a.cols / (kThreads * kPer<BF16>);
  if (groups <= 1)
    hipLaunchKernelGGL((logprob_kernel<BF16, 1>), dim3(rows), dim3(kThreads), 0, s, a);
  else if (groups <= 6)
    hipLaunchKernelGGL((logprob_kernel<BF16, 6>), dim3(rows), dim3(kThreads), 0, s, a);
  else if (groups <= 12)
    hipLaunchKernelGGL((logprob_kernel<BF16, 12>), dim3(rows), dim3(kThreads), 0, s, a);
  else if (groups <= 24)
    hipLaunchKernelGGL((logprob_kernel<BF16, 24>), dim3(rows), dim3(kThreads), 0, s, a);
  else
    hipLaunchKernelGGL((logprob_kernel<BF16, 0>), dim3(rows), dim3(kThreads), 0, s, a);
}

int check(const char *fn, uint32_t dtype, uint32_t rows, uint32_t cols, uint32_t row_stride) {
  if (dtype != DFATTN_KV_F32 && dtype != DFATTN_KV_BF16)
    return record_error(DFATTN_ERR_FLAGS, std::string(fn) + ": dtype must be DFATTN_KV_F32 or DFATTN_KV_BF16");
  if (cols == 0) return record_error(DFATTN_ERR_SHAPE, std::string(fn) + ": row length must be >= 1");
  if (row_stride < cols) return record_error(DFATTN_ERR_SHAPE, std::string(fn) + ": row_stride must be at least cols");
  if (rows > kMaxRows || cols > (1u << 27))
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
    launch_logprobs<true>(a, rows, stream);
  else
    launch_logprobs<false>(a, rows, stream);
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
  const bool bf16 = dtype == DFATTN_KV_BF16;
  const uint32_t part = 256 * kGradSteps * (bf16 ? kPer<true> : kPer<false>);
  const dim3 grid(rows, (cols + part - 1) / part);
  if (grid.y > 65535u) return record_error(DFATTN_ERR_OVERFLOW, std::string(fn) + ": shape is too large");
  if (bf16)
    hipLaunchKernelGGL(logprob_grad_kernel<true>, grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL(logprob_grad_kernel<false>, grid, dim3(256), 0, stream, a);
  return launched(fn);
}

}  // extern "C"
