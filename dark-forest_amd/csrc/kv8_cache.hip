// kv8_cache.hip — the paged 8-bit cache of a batch of requests: tables and slot
// maps from lengths, the quantising append and the read-back (gfx950).
#include "kv8.h"

namespace dfattn {
namespace {

using namespace kv8;

// ---------------------------------------------------------------- plan
constexpr int kPlanThreads = 256;
constexpr uint32_t kMaxRequests = 8192;

struct PlanArgs {
  const uint32_t *cached, *fresh, *free_pages, *free_start;
  uint32_t *table, *seq_lens, *query_start, *slots, *counts;
  uint32_t n_free, R, max_pages, capacity, P, n_pages;
};

// The last i in [0, n] with a[i] <= x (a does not fall, a[0] <= x).
__device__ __forceinline__ uint32_t find_last(const uint32_t *a, uint32_t n, uint32_t x) {
  uint32_t lo = 0, hi = n + 1;  // a[lo] <= x, a[hi] > x
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (a[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// Every workgroup sums the lengths by itself (at most 8192 requests: 64 KB from
// L2), so that one launch does it all: tok[i] and pg[i] are the tokens and
// fresh pages of the requests before i, which are both rising, so the
// admitted requests are those before the first that does not fit. Then
// the workgroups share out the tokens and the fresh pages.
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(PlanArgs a) {
  extern __shared__ uint32_t lds[];
  uint32_t *tok = lds, *pg = lds + a.R + 1;
  __shared__ unsigned long long tok_w[kPlanThreads / 64], pg_w[kPlanThreads / 64];
  __shared__ uint32_t first_bad;
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t per = (a.R + kPlanThreads - 1) / kPlanThreads;
  const uint32_t i0 = min(a.R, tid * per), i1 = min(a.R, i0 + per);
  const uint32_t start = min(*a.free_start, a.n_free), avail = a.n_free - start;
  auto need = [&](uint32_t c, uint32_t n) {
    return (uint32_t)(((uint64_t)c + n + a.P - 1) / a.P - ((uint64_t)c + a.P - 1) / a.P);
  };
  unsigned long long t = 0, p = 0;
  for (uint32_t i = i0; i < i1; ++i) {
    t += a.fresh[i];
    p += need(a.cached[i], a.fresh[i]);
  }
  unsigned long long ti = t, pi = p;  // inclusive over the wave's lanes
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const unsigned long long tu = __shfl_up(ti, off, 64), pu = __shfl_up(pi, off, 64);
    if ((int)lane >= off) {
      ti += tu;
      pi += pu;
    }
  }
  if (tid == 0) first_bad = a.R;
  if (lane == 63) {
    tok_w[wave] = ti;
    pg_w[wave] = pi;
  }
  __syncthreads();
  unsigned long long tb = ti - t, pb = pi - p;
  for (uint32_t w = 0; w < wave; ++w) {
    tb += tok_w[w];
    pb += pg_w[w];
  }
  for (uint32_t i = i0; i < i1; ++i) {
    const uint32_t c = a.cached[i], n = a.fresh[i];
    tok[i] = (uint32_t)tb;
    pg[i] = (uint32_t)pb;
    tb += n;
    pb += need(c, n);
    if ((uint64_t)c + n > (uint64_t)a.max_pages * a.P || pb > avail || tb > a.capacity) {
      atomicMin(&first_bad, i);
      break;  // (the sums behind it are not read)
    }
    if (i + 1 == a.R) {
      tok[a.R] = (uint32_t)tb;
      pg[a.R] = (uint32_t)pb;
    }
  }
  __syncthreads();
  const uint32_t in = first_bad, total = tok[in], pages = pg[in];
  const uint32_t id = blockIdx.x * kPlanThreads + tid, step = gridDim.x * kPlanThreads;
  for (uint32_t i = id; i <= a.R; i += step) {
    a.query_start[i] = tok[min(i, in)];
    if (i < a.R) a.seq_lens[i] = a.cached[i] + (i < in ? a.fresh[i] : 0u);
  }
  if (id == 0) {
    a.counts[0] = in;
    a.counts[1] = total;
    a.counts[2] = start + pages;
  }
  for (uint32_t x = id; x < pages; x += step) {
    const uint32_t r = find_last(pg, in, x);
    const uint32_t had = (uint32_t)(((uint64_t)a.cached[r] + a.P - 1) / a.P);
    a.table[(size_t)r * a.max_pages + had + (x - pg[r])] = a.free_pages[start + x];
  }
  for (uint32_t x = id; x < a.capacity; x += step) {
    uint32_t slot = DFATTN_NO_SLOT;
    if (x < total) {
      const uint32_t r = find_last(tok, in, x), c = a.cached[r], pos = c + (x - tok[r]);
      const uint32_t lp = pos / a.P, had = (uint32_t)(((uint64_t)c + a.P - 1) / a.P);
      const uint32_t page =
          lp < had ? a.table[(size_t)r * a.max_pages + lp] : a.free_pages[start + pg[r] + (lp - had)];
      if (page < a.n_pages) slot = page * a.P + pos % a.P;
    }
    a.slots[x] = slot;
  }
}

// ---------------------------------------------------------------- append
struct CacheArgs {
  const void *k, *v;  // rows of activations (append), or the pools (read)
  const uint32_t *slots;
  unsigned char *k_pool, *v_pool;
  float *k_scales, *v_scales;
  void *k_out, *v_out;
  size_t stride;
  uint32_t n;
  int H, D, P, n_pages;
};

constexpr int kAppendThreads = 256;

// One wave takes one run (the consecutive rows of one page), one kv head and K
// or V. It finds the largest magnitude, then the scale, then the codes; the
// rows already there are coded again where the scale grew.
template <bool E4M3, bool BF16>
__global__ __launch_bounds__(kAppendThreads) void append_kernel(CacheArgs a) {
  const uint32_t i = linear_block();
  if (i >= a.n) return;
  const int lane = threadIdx.x & 63;
  const uint32_t n_slots = (uint32_t)a.n_pages * (uint32_t)a.P;
  const uint32_t slot = a.slots[i];
  if (slot >= n_slots) return;
  const int off = (int)(slot % (uint32_t)a.P);
  if (i > 0 && off != 0 && a.slots[i - 1] == slot - 1) return;  // not the first of its run
  int len = 1;
  while (len < a.P - off && i + len < a.n && a.slots[i + len] == slot + len) ++len;
  const size_t page = slot / (uint32_t)a.P;
  const int D = a.D, Dp = padded(D), P = a.P;
  for (int task = (int)(blockIdx.z * 4 + (threadIdx.x >> 6)); task < 2 * a.H; task += 4 * gridDim.z) {
    const int h = task >> 1;
    const bool is_v = task & 1;
    const void *src = is_v ? a.v : a.k;
    auto value = [&](int row, int d) { return load_act(src, (size_t)(i + row) * a.stride + h * D + d, BF16); };
    float amax = 0.f;
    bool bad = false;
    for (int e = lane; e < len * D; e += 64) {
      const float x = fabsf(value(e / D, e % D));
      bad |= !(x <= 3.4028234e38f);
      amax = fmaxf(amax, x);
    }
    amax = wave_max(amax);
    const size_t head = page * a.H + h;
    float *scale = (is_v ? a.v_scales : a.k_scales) + head;
    const float old = off > 0 ? *scale : 0.f;
    float s = fmaxf(old, pow2_scale<E4M3>(amax));
    if (__any(bad) || old != old) s = __builtin_nanf("");
    if (lane == 0) *scale = s;
    // A poisoned page and head holds zeros (times NaN).
    const bool dead = s != s;
    const float inv = dead ? 0.f : 1.f / s, ratio = dead ? 0.f : old * inv;
    auto code = [&](float x) { return encode4<E4M3>(make_float4(dead ? 0.f : x * inv, 0.f, 0.f, 0.f)) & 0xffu; };
    auto recode = [&](unsigned c) { return encode4<E4M3>(make_float4(decode4<E4M3>(c).x * ratio, 0.f, 0.f, 0.f)) & 0xffu; };
    unsigned char *dst = (is_v ? a.v_pool : a.k_pool) + head * (size_t)(P * Dp);
    const bool grew = off > 0 && ratio != 1.f;
    for (int e = lane; e < len * Dp; e += 64) {
      const int row = is_v ? e % len : e / Dp, d = is_v ? e / len : e % Dp;
      if (is_v && d >= D) continue;
      dst[is_v ? d * P + off + row : (off + row) * Dp + d] = (unsigned char)(d < D ? code(value(row, d)) : 0u);
    }
    if (grew)
      for (int e = lane; e < off * Dp; e += 64) {
        unsigned char *c = dst + (is_v ? e / off * P + e % off : e);
        *c = (unsigned char)recode(*c);
      }
  }
}

// ---------------------------------------------------------------- read
template <bool E4M3, bool BF16>
__global__ __launch_bounds__(256) void read_kernel(CacheArgs a) {
  const uint32_t i = linear_block();
  if (i >= a.n) return;
  const uint32_t slot = a.slots[i];
  const bool in = slot < (uint32_t)a.n_pages * (uint32_t)a.P;
  const size_t page = in ? slot / (uint32_t)a.P : 0;
  const int off = in ? (int)(slot % (uint32_t)a.P) : 0, Dp = padded(a.D), dm = a.H * a.D;
  for (int e = (int)threadIdx.x; e < 2 * dm; e += 256) {
    const bool is_v = e >= dm;
    const int x = is_v ? e - dm : e, h = x / a.D, d = x % a.D;
    const size_t head = page * a.H + h;
    float val = 0.f;
    if (in) {
      const unsigned char *base = (is_v ? a.v_pool : a.k_pool) + head * (size_t)(a.P * Dp);
      val = decode4<E4M3>(base[is_v ? d * a.P + off : off * Dp + d]).x * (is_v ? a.v_scales : a.k_scales)[head];
    }
    void *out = is_v ? a.v_out : a.k_out;
    if (BF16)
      static_cast<unsigned short *>(out)[(size_t)i * dm + x] = (unsigned short)bf16_bits(val);
    else
      static_cast<float *>(out)[(size_t)i * dm + x] = val;
  }
}

template <typename F>
void by_types(uint32_t act, uint32_t kv, F f) {
  const bool e4m3 = kv == DFATTN_KV_E4M3, bf16 = act == DFATTN_KV_BF16;
  if (e4m3 && bf16)
    f(std::true_type{}, std::true_type{});
  else if (e4m3)
    f(std::true_type{}, std::false_type{});
  else if (bf16)
    f(std::false_type{}, std::true_type{});
  else
    f(std::false_type{}, std::false_type{});
}

}  // namespace
}  // namespace dfattn

using namespace dfattn;
using namespace dfattn::kv8;

extern "C" {

int dfattn_paged_plan(const uint32_t *cached_lens, const uint32_t *new_lens, const uint32_t *free_pages,
                      const uint32_t *free_start, uint32_t *block_table, uint32_t *seq_lens, uint32_t *query_start,
                      uint32_t *slot_map, uint32_t *counts, uint32_t n_free, uint32_t n_requests, uint32_t max_pages,
                      uint32_t token_capacity, uint32_t page_size, uint32_t n_pages, void *stream) {
  const char *fn = "dfattn_paged_plan";
  if (n_requests == 0 || max_pages == 0 || page_size == 0 || n_pages == 0)
    return record_error(DFATTN_ERR_SHAPE,
                        std::string(fn) + ": n_requests, max_pages, page_size and n_pages must be >= 1");
  if (n_requests > kMaxRequests || (uint64_t)n_pages * page_size > (1ull << 31) ||
      (uint64_t)max_pages * page_size > (1ull << 31) || token_capacity > (1u << 31) || n_free > (1u << 31))
    return record_error(DFATTN_ERR_OVERFLOW, std::string(fn) + ": shape is too large");
  int st = check_all(fn, {cached_lens, new_lens, free_start, block_table, seq_lens, query_start, counts}, 4);
  if (st == DFATTN_OK && n_free > 0) st = check_all(fn, {free_pages}, 4);
  if (st == DFATTN_OK && token_capacity > 0) st = check_all(fn, {slot_map}, 4);
  if (st != DFATTN_OK) return st;
  if (counts <= free_start && free_start < counts + 3)
    return record_error(DFATTN_ERR_SHAPE, std::string(fn) + ": free_start must not lie in counts");
  PlanArgs a{cached_lens, new_lens, free_pages, free_start, block_table, seq_lens, query_start, slot_map, counts,
             n_free, n_requests, max_pages, token_capacity, page_size, n_pages};
  // Four tokens a thread, up to two workgroups a CU.
  const uint32_t work = std::max(token_capacity, n_requests + 1);
  const uint32_t grid = std::min(512u, (work + 4 * kPlanThreads - 1) / (4 * kPlanThreads));
  const size_t lds = 2 * (size_t)(n_requests + 1) * sizeof(uint32_t);
  hipLaunchKernelGGL(plan_kernel, dim3(grid), dim3(kPlanThreads), lds, static_cast<hipStream_t>(stream), a);
  return launched(fn);
}

size_t dfattn_kv8_pool_bytes(uint32_t n_pages, uint32_t n_kv_heads, uint32_t page_size, uint32_t d_head) {
  if (n_pages == 0 || n_kv_heads == 0 || n_kv_heads > 65535u || page_size == 0 || page_size % 16 != 0 ||
      page_size > 256 || d_head == 0 || d_head > 128 || (uint64_t)n_pages * page_size > (1ull << 31))
    return 0;
  return (size_t)n_pages * n_kv_heads * page_size * padded((int)d_head);
}

int dfattn_kv8_append(const void *k, const void *v, const uint32_t *slot_map, void *k_pool, void *v_pool,
                      float *k_scales, float *v_scales, uint32_t act_dtype, uint32_t kv_dtype, uint32_t n_tokens,
                      uint32_t n_kv_heads, uint32_t d_head, uint32_t page_size, uint32_t n_pages, uint32_t row_stride,
                      void *stream) {
  const char *fn = "dfattn_kv8_append";
  int st = check_types(fn, act_dtype, kv_dtype);
  if (st == DFATTN_OK) st = check_pool_shape(fn, n_pages, n_kv_heads, page_size, d_head);
  if (st != DFATTN_OK) return st;
  if (row_stride < (uint64_t)n_kv_heads * d_head)
    return record_error(DFATTN_ERR_SHAPE, std::string(fn) + ": row_stride must be at least n_kv_heads * d_head");
  if (n_tokens > (1u << 31)) return record_error(DFATTN_ERR_OVERFLOW, std::string(fn) + ": too many tokens");
  if (n_tokens == 0) return DFATTN_OK;
  st = check_all(fn, {k, v}, act_dtype == DFATTN_KV_F32 ? 4 : 2);
  if (st == DFATTN_OK) st = check_all(fn, {slot_map, k_scales, v_scales}, 4);
  if (st == DFATTN_OK) st = check_all(fn, {k_pool, v_pool}, 16);
  if (st != DFATTN_OK) return st;
  CacheArgs a{};
  a.k = k;
  a.v = v;
  a.slots = slot_map;
  a.k_pool = static_cast<unsigned char *>(k_pool);
  a.v_pool = static_cast<unsigned char *>(v_pool);
  a.k_scales = k_scales;
  a.v_scales = v_scales;
  a.stride = row_stride;
  a.n = n_tokens;
  a.H = (int)n_kv_heads;
  a.D = (int)d_head;
  a.P = (int)page_size;
  a.n_pages = (int)n_pages;
  dim3 grid = linear_grid(n_tokens);
  grid.z = (2 * n_kv_heads + 3) / 4;
  by_types(act_dtype, kv_dtype, [&](auto e4m3, auto bf16) {
    hipLaunchKernelGGL((append_kernel<decltype(e4m3)::value, decltype(bf16)::value>), grid, dim3(kAppendThreads), 0,
                       static_cast<hipStream_t>(stream), a);
  });
  return launched(fn);
}

int dfattn_kv8_read(const void *k_pool, const void *v_pool, const float *k_scales, const float *v_scales,
                    const uint32_t *slots, void *k_out, void *v_out, uint32_t act_dtype, uint32_t kv_dtype,
                    uint32_t n_rows, uint32_t n_kv_heads, uint32_t d_head, uint32_t page_size, uint32_t n_pages,
                    void *stream) {
  const char *fn = "dfattn_kv8_read";
  int st = check_types(fn, act_dtype, kv_dtype);
  if (st == DFATTN_OK) st = check_pool_shape(fn, n_pages, n_kv_heads, page_size, d_head);
  if (st != DFATTN_OK) return st;
  if (n_rows > (1u << 31)) return record_error(DFATTN_ERR_OVERFLOW, std::string(fn) + ": too many rows");
  if (n_rows == 0) return DFATTN_OK;
  st = check_all(fn, {k_out, v_out}, act_dtype == DFATTN_KV_F32 ? 4 : 2);
  if (st == DFATTN_OK) st = check_all(fn, {slots, k_scales, v_scales}, 4);
  if (st == DFATTN_OK) st = check_all(fn, {k_pool, v_pool}, 16);
  if (st != DFATTN_OK) return st;
  CacheArgs a{};
  a.slots = slots;
  a.k_pool = static_cast<unsigned char *>(const_cast<void *>(k_pool));
  a.v_pool = static_cast<unsigned char *>(const_cast<void *>(v_pool));
  a.k_scales = const_cast<float *>(k_scales);
  a.v_scales = const_cast<float *>(v_scales);
  a.k_out = k_out;
  a.v_out = v_out;
  a.n = n_rows;
  a.H = (int)n_kv_heads;
  a.D = (int)d_head;
  a.P = (int)page_size;
  a.n_pages = (int)n_pages;
  by_types(act_dtype, kv_dtype, [&](auto e4m3, auto bf16) {
    hipLaunchKernelGGL((read_kernel<decltype(e4m3)::value, decltype(bf16)::value>), linear_grid(n_rows), dim3(256), 0,
                       static_cast<hipStream_t>(stream), a);
  });
  return launched(fn);
}

}  // extern "C"
