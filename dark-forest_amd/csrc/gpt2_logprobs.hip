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

constexpr int kThreads = 512, kFewThreads = 256;  // of a row of more than kLong logits, of a shorter one
constexpr uint32_t kLong = 16384;
constexpr uint32_t kMaxTop = 64;
constexpr uint32_t kMaxRows = 1u << 21;
constexpr int kCandidates = 512, kSlots = 8;

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

template <int kWaves>
struct Shared {
  float lane_max[kWaves][64], sum_s[kWaves], sum_t[kWaves];
  int above[64];
  unsigned n_cand, wave_equal[kWaves];
  unsigned long long cand[kCandidates], best[kWaves];
};

// The next larger number; the smallest one after either zero.
__device__ __forceinline__ float next_above(float x) {
  const unsigned u = __float_as_uint(x);
  return x == 0.f ? __uint_as_float(1u) : __uint_as_float(u & 0x80000000u ? u - 1u : u + 1u);
}

// S = sum e^(x - m) and T = sum e^(x - m) (x - m) log2 e about a maximum m.
struct Sums {
  float m, s, t;
  // The same about m_new >= m. (2^-1000 is 0: sums about -infinity are 0.)
  __device__ __forceinline__ void move(float m_new) {
    const float d = fmaxf((m - (m_new == -INFINITY ? 0.f : m_new)) * kLog2e, -1000.f);
    const float f = __builtin_amdgcn_exp2f(d);
    t = f * fmaf(d, s, t);
    s *= f;
    m = m_new;
  }
};

// The k-th largest of the 64 lanes' maxima (a lane's over all waves): a lower bound
// of the k-th largest of the values so far. `strict`: eight or more lanes hold it,
// a mask's value most likely, so that only what is above it makes a candidate.
template <int kWaves>
__device__ __forceinline__ float lane_bound(Shared<kWaves> &sh, float mine, int k, int lane, int wave, bool &strict) {
  sh.lane_max[wave][lane] = mine;
  if (wave == 0) sh.above[lane] = 0;
  __syncthreads();
  float top = sh.lane_max[0][lane];
#pragma unroll
  for (int v = 1; v < kWaves; ++v) top = fmaxf(top, sh.lane_max[v][lane]);
  int above = 0;
#pragma unroll
  for (int j = 0; j < 64 / kWaves; ++j) {
    const int o_lane = wave * (64 / kWaves) + j;
    const float o = __shfl(top, o_lane, 64);
    above += o > top || (o == top && o_lane < lane);
  }
  atomicAdd(&sh.above[lane], above);
  __syncthreads();
  const int who = __ffsll(__ballot(sh.above[lane] == k - 1)) - 1;
  const float thr = __shfl(top, who, 64);
  strict = __popcll(__ballot(top == thr)) >= 8;
  return thr;
}

// One workgroup per row, one pass over memory: kBatch groups a thread at a time,
// the next ones on their way meanwhile; exponentials about the thread's maximum so
// far. The alternatives: each thread's maxima by slots of batches wait in LDS until
// lane_bound gives a bound that at least k logits reach. The few slots that reach it
// (some 30 of 512 threads hold one) are read again for the candidates, and each
// candidate's rank among them is its place.
// A row that has more than kCandidates of them, or a NaN, is read k times more, an alternative at
// a time. That takes large logits crowded into a few lanes, or k = 64: the bound is then the
// smallest of the 64 maxima, which some 300 ordinary logits reach, but 3 of 100 rows have more than 512
// that do (none of 300 rows at k = 63, 425 the most): 2048 rows of 50257 in bf16 take 1227 us, at
// k = 60 75.
//
// Measured: 1000 rows of 50257 in fp32 38 us by themselves, 5.2 TB/s; 2048 in bf16 49 us, with 20
// alternatives 59, where the rows' ends, two rounds of them, leave memory idle. 8 rows 10.5 us: seven
// batches one after the other.
// 512 threads a row, 256 where it is short: 8192 rows of 1000 28 us for 16, of 8192 52 for 48; of
// 4096 rows of 32768 97 for 102, and of 2048 of 50257 (bf16, 20 alternatives) 59 for 67.
template <bool BF16, bool TOP, int kThreads>
__global__ __launch_bounds__(kThreads) void logprob_kernel(LogprobArgs a) {
  constexpr int W = kPer<BF16>, kBatch = BF16 ? 2 : 4, kStep = kThreads * W, kWaves = kThreads / 64;
  __shared__ Shared<kWaves> sh;
  __shared__ float slot_max[TOP ? kSlots : 1][kThreads];
  const size_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = a.cols, k = a.k;
  const void *base = static_cast<const char *>(a.logits) + row * a.stride * (BF16 ? 2 : 4);
  const uint32_t token = a.tokens[row];
  const float chosen = token < (uint32_t)n ? load_logit<BF16>(base, token) : 0.f;
  // Group j of a thread: ids (j * kThreads + tid) * W ..; `whole` of them are whole in the workgroup.
  const int whole = n / kStep, first = tid * W;
  const raw4 end = load_end<BF16>(base, whole * kStep + first, n);
  const unsigned fill = BF16 ? 0xff80ff80u : 0xff800000u;
  auto load = [&](int j) {
    if (j < whole) return load_group<BF16>(base, j * kStep + first);
    return j == whole ? end : raw4{fill, fill, fill, fill};
  };
  const int per_slot = ((whole + kBatch) / kBatch + kSlots - 1) / kSlots;  // batches
  Sums x = {-INFINITY, 0.f, 0.f};
  auto batch = [&](const raw4 *r) {
    float top = -INFINITY;
#pragma unroll
    for (int q = 0; q < kBatch; ++q)
#pragma unroll
      for (int w = 0; w < W; ++w) top = fmaxf(top, logit_of<BF16>(r[q], w));
    if (top > x.m) x.move(top);
    const float m0 = x.m == -INFINITY ? 0.f : x.m;
#pragma unroll
    for (int q = 0; q < kBatch; ++q)
#pragma unroll
      for (int w = 0; w < W; ++w) {
        // A masked-out logit adds 0 to T (0 times at least -200), a NaN makes both NaN.
        const float y = (logit_of<BF16>(r[q], w) - m0) * kLog2e, e = __builtin_amdgcn_exp2f(y);
        x.s += e;
        x.t = fmaf(e, fmaxf(y, -200.f), x.t);
      }
    return top;
  };
  if (TOP && tid == 0) sh.n_cand = 0;
  raw4 cur[kBatch], next[kBatch];
#pragma unroll
  for (int q = 0; q < kBatch; ++q) cur[q] = load(q);
  int slot = 0, left = per_slot;
  float slot_top = -INFINITY;
  for (int j0 = 0; j0 <= whole; j0 += kBatch) {
#pragma unroll
    for (int q = 0; q < kBatch; ++q) next[q] = load(j0 + kBatch + q);
    const float top = batch(cur);
    if constexpr (TOP) {
      slot_top = fmaxf(slot_top, top);
      slot_max[slot][tid] = slot_top;
      if (--left == 0) {
        ++slot;
        left = per_slot;
        slot_top = -INFINITY;
      }
    }
#pragma unroll
    for (int q = 0; q < kBatch; ++q) cur[q] = next[q];
  }
  const int slots = slot + (left < per_slot);
  const float mine = x.m;
  const float wave_top = wave_max(mine);
  x.move(wave_top);
  x.s = wave_sum(x.s);
  x.t = wave_sum(x.t);
  if (lane == 0) {
    sh.lane_max[0][wave] = wave_top;
    sh.sum_s[wave] = x.s;
    sh.sum_t[wave] = x.t;
  }
  __syncthreads();
  float m = sh.lane_max[0][0];
#pragma unroll
  for (int v = 1; v < kWaves; ++v) m = fmaxf(m, sh.lane_max[0][v]);
  float s = 0.f, t = 0.f;
#pragma unroll
  for (int v = 0; v < kWaves; ++v) {
    Sums y = {sh.lane_max[0][v], sh.sum_s[v], sh.sum_t[v]};
    y.move(m);
    s += y.s;
    t += y.t;
  }
  const bool nan = s != s, none = m == -INFINITY && !nan;
  const float m0 = none ? 0.f : m, ln_s = none ? 0.f : logf(s);
  auto logp = [&](float v) { return v == -INFINITY && !nan ? v : (v - m0) - ln_s; };
  if (tid == 0) {
    a.logprob[row] = token < (uint32_t)n ? logp(chosen) : 0.f;
    if (a.entropy) a.entropy[row] = none ? 0.f : ln_s - t * kLn2 / s;
    if (a.stats) {
      a.stats[2 * row] = nan ? ln_s : m;
      a.stats[2 * row + 1] = ln_s;
    }
  }
  if constexpr (!TOP) return;

  auto put = [&](unsigned long long key, int place) {
    a.top_ids[row * k + place] = 0xffffffffu - (uint32_t)key;
    a.top_logprobs[row * k + place] = logp(logit_of_rank((unsigned)(key >> 32)));
  };
  float thr = INFINITY;
  bool strict = false;
  unsigned c = kCandidates + 1;
  for (int pass = 0; pass < 2 && c > kCandidates && !nan; ++pass) {
    __syncthreads();
    if (pass == 0)
      thr = lane_bound(sh, mine, k, lane, wave, strict);
    else  // too many equal the bound
      strict = true;
    if (pass > 0 && tid == 0) sh.n_cand = 0;
    if (pass > 0) __syncthreads();
    const float least = strict ? next_above(thr) : thr;
    unsigned todo = 0;
    if (mine >= least)
      for (int i = 0; i < slots; ++i) todo |= slot_max[i][tid] >= least ? 1u << i : 0u;
    for (; todo; todo &= todo - 1) {
      const int j1 = (__ffs(todo) - 1) * per_slot * kBatch, j2 = min(j1 + per_slot * kBatch, whole + 1);
#pragma unroll kBatch
      for (int j = j1; j < j2; ++j) {
        const raw4 r = j < whole ? load_group<BF16>(base, j * kStep + first) : end;
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const float v = logit_of<BF16>(r, w);
          if (v >= least && j * kStep + first + w < n) {
            const unsigned at = atomicAdd(&sh.n_cand, 1u);
            if (at < kCandidates) sh.cand[at] = key_of(v, j * kStep + first + w);
          }
        }
      }
    }
    __syncthreads();
    c = sh.n_cand;
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
    if (!strict || (int)c >= k) return;
    // The rest equals the bound: the lowest ids of those.
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
  // NaN, or too many candidates: one alternative after the other.
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
// is written, so the gradient may lie where the logits do. 1000 rows of 50257 in fp32 67 us,
// 6.0 TB/s (after the forward, with part of the logits still in the Infinity Cache), in bf16 39, 5.2.
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

template <bool BF16, int THREADS>
void launch_logprobs(const LogprobArgs &a, uint32_t rows, hipStream_t s) {
  if (a.k > 0)
    hipLaunchKernelGGL((logprob_kernel<BF16, true, THREADS>), dim3(rows), dim3(THREADS), 0, s, a);
  else
    hipLaunchKernelGGL((logprob_kernel<BF16, false, THREADS>), dim3(rows), dim3(THREADS), 0, s, a);
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
  const bool bf16 = dtype == DFATTN_KV_BF16, few = cols <= kLong;
  if (bf16 && few)
    launch_logprobs<true, kFewThreads>(a, rows, stream);
  else if (bf16)
    launch_logprobs<true, kThreads>(a, rows, stream);
  else if (few)
    launch_logprobs<false, kFewThreads>(a, rows, stream);
  else
    launch_logprobs<false, kThreads>(a, rows, stream);
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
  const size_t item = dtype == DFATTN_KV_F32 ? 4 : 2;
  const char *x = static_cast<const char *>(logits), *g = static_cast<const char *>(grad_logits);
  const bool overlap = x < g + (size_t)rows * cols * item && g < x + ((size_t)(rows - 1) * row_stride + cols) * item;
  if (overlap && (x != g || row_stride != cols))
    return record_error(DFATTN_ERR_SHAPE, std::string(fn) + ": grad_logits may overlap logits only as the same rows");
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
