// kv8_attention.hip — attention of a batch of requests over the paged 8-bit
// cache, queries of one token or many (gfx950).
//
// For query j of the n of request r, at position L - n + j of its L cached
// tokens: out = sum_t p_t v_t / sum_t p_t, p_t = exp(scale q . k_t - m), over
// the positions t it sees, k_t and v_t codes times the scale of their page and
// head.
#include "kv8.h"

#include <algorithm>

namespace dfattn {
namespace {

using namespace kv8;

struct AttnArgs {
  const void *q;
  const unsigned char *k, *v;
  const float *k_scales, *v_scales;
  const uint32_t *table, *query_start, *seq_lens;
  void *out;
  float *lse;
  uint32_t R, n_tokens, max_q, max_pages, n_pages;
  int H, Hk, D, P;
  size_t q_stride;
  float scale;
  int causal;
};

__device__ __forceinline__ void store_act(void *p, size_t i, float x, bool bf16) {
  if (bf16)
    static_cast<unsigned short *>(p)[i] = (unsigned short)bf16_bits(x);
  else
    static_cast<float *>(p)[i] = x;
}

// One wave per query row and head: 64 keys at a time, lane = key for the
// scores, lane = column for the products with V.
template <bool E4M3>
__global__ __launch_bounds__(64) void attention_kernel(AttnArgs a, bool bf16) {
  __shared__ float q_lds[128], p_lds[64];
  __shared__ uint32_t page_lds[64];
  const uint32_t t = linear_block();
  const int h = blockIdx.z, lane = threadIdx.x, D = a.D, Dp = padded(D), P = a.P;
  if (t >= a.n_tokens || t >= a.query_start[a.R]) return;
  uint32_t lo = 0, hi = a.R;  // the last request that starts at or before t
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (a.query_start[mid] <= t)
      lo = mid;
    else
      hi = mid;
  }
  const uint32_t r = lo, j = t - a.query_start[r], nq = a.query_start[r + 1] - a.query_start[r];
  if (j >= a.max_q) return;
  const long long L = min((long long)a.seq_lens[r], (long long)a.max_pages * P);
  const long long n = a.causal ? min(L, (long long)a.seq_lens[r] - nq + j + 1) : L;
  const int hk = h / (a.H / a.Hk);
  for (int d = lane; d < Dp; d += 64)
    q_lds[d] = d < D ? load_act(a.q, (size_t)t * a.q_stride + (size_t)h * D + d, bf16) * (a.scale * kLog2e) : 0.f;
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  for (long long k0 = 0; k0 < n; k0 += 64) {
    const long long key = k0 + lane;
    float s = -INFINITY, vs = 0.f;
    uint32_t page = 0xffffffffu;
    if (key < n) page = a.table[(size_t)r * a.max_pages + (size_t)(key / P)];
    __syncthreads();
    if (page < a.n_pages) {
      const size_t head = (size_t)page * a.Hk + hk;
      const unsigned *row = reinterpret_cast<const unsigned *>(a.k + (head * P + (size_t)(key % P)) * Dp);
      float acc = 0.f;
      for (int d = 0; d < Dp; d += 4) {
        const float4 k4 = decode4<E4M3>(row[d / 4]);
        acc += k4.x * q_lds[d] + k4.y * q_lds[d + 1] + k4.z * q_lds[d + 2] + k4.w * q_lds[d + 3];
      }
      s = acc * a.k_scales[head];
      vs = a.v_scales[head];
    }
    const float m_new = fmaxf(m, wave_max(s));
    const float base = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - base);
    const float p = page < a.n_pages ? __builtin_amdgcn_exp2f(s - base) : 0.f;
    l = l * alpha + p;
    m = m_new;
    p_lds[lane] = page < a.n_pages ? p * vs : 0.f;
    page_lds[lane] = page;
    __syncthreads();
    o0 *= alpha;
    o1 *= alpha;
    for (int i = 0; i < 64; ++i) {
      const uint32_t pi = page_lds[i];
      if (pi >= a.n_pages) continue;
      const size_t head = (size_t)pi * a.Hk + hk;
      const unsigned char *col = a.v + head * (size_t)(P * Dp) + (size_t)((k0 + i) % P);
      if (lane < D) o0 += p_lds[i] * decode4<E4M3>(col[(size_t)lane * P]).x;
      if (lane + 64 < D) o1 += p_lds[i] * decode4<E4M3>(col[(size_t)(lane + 64) * P]).x;
    }
  }
  l = wave_sum(l);
  const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
  const size_t at = (size_t)t * a.H * D + (size_t)h * D;
  if (lane < D) store_act(a.out, at + lane, o0 * inv, bf16);
  if (lane + 64 < D) store_act(a.out, at + lane + 64, o1 * inv, bf16);
  if (lane == 0 && a.lse) a.lse[(size_t)h * a.n_tokens + t] = (m + __builtin_log2f(l)) * kLn2;
}

}  // namespace
}  // namespace dfattn

using namespace dfattn;
using namespace dfattn::kv8;

extern "C" {

size_t dfattn_kv8_attention_workspace_bytes(uint32_t, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t) {
  return 0;
}

int dfattn_kv8_attention(const void *q, const void *k_pool, const void *v_pool, const float *k_scales,
                         const float *v_scales, const uint32_t *block_table, const uint32_t *query_start,
                         const uint32_t *seq_lens, void *out, float *lse, uint32_t act_dtype, uint32_t kv_dtype,
                         uint32_t n_requests, uint32_t n_tokens, uint32_t max_query_len, uint32_t max_seq_len,
                         uint32_t n_heads, uint32_t n_kv_heads, uint32_t d_head, uint32_t page_size, uint32_t n_pages,
                         uint32_t max_pages, uint32_t q_row_stride, float scale, uint32_t causal, void *workspace,
                         size_t workspace_bytes, void *stream) {
  const char *fn = "dfattn_kv8_attention";
  int st = check_types(fn, act_dtype, kv_dtype);
  if (st == DFATTN_OK) st = check_pool_shape(fn, n_pages, n_kv_heads, page_size, d_head);
  if (st != DFATTN_OK) return st;
  if (n_heads == 0 || n_heads % n_kv_heads != 0)
    return record_error(DFATTN_ERR_SHAPE, std::string(fn) + ": n_heads must be a multiple of n_kv_heads");
  if (max_pages == 0) return record_error(DFATTN_ERR_SHAPE, std::string(fn) + ": max_pages must be >= 1");
  if (q_row_stride < (uint64_t)n_heads * d_head)
    return record_error(DFATTN_ERR_SHAPE, std::string(fn) + ": q_row_stride must be at least n_heads * d_head");
  if (n_heads > 65535u || n_requests > 65535u || n_tokens > (1u << 30) || (uint64_t)max_pages * page_size > (1ull << 31))
    return record_error(DFATTN_ERR_OVERFLOW, std::string(fn) + ": shape is too large");
  if (n_requests == 0 || n_tokens == 0 || max_query_len == 0) return DFATTN_OK;
  st = check_all(fn, {q, out}, act_dtype == DFATTN_KV_F32 ? 4 : 2);
  if (st == DFATTN_OK) st = check_all(fn, {k_scales, v_scales, block_table, query_start, seq_lens}, 4);
  if (st == DFATTN_OK) st = check_all(fn, {k_pool, v_pool}, 16);
  if (st != DFATTN_OK) return st;
  if (lse != nullptr && !aligned_to(lse, 4))
    return record_error(DFATTN_ERR_MISALIGNED, std::string(fn) + ": misaligned pointer");
  const size_t need = dfattn_kv8_attention_workspace_bytes(n_requests, n_tokens, max_query_len, max_seq_len, n_heads,
                                                           n_kv_heads, d_head);
  if (workspace != nullptr && (workspace_bytes < need || !aligned_to(workspace, 16)))
    return record_error(DFATTN_ERR_WORKSPACE, std::string(fn) + ": workspace too small or misaligned");
  AttnArgs a{};
  a.q = q;
  a.k = static_cast<const unsigned char *>(k_pool);
  a.v = static_cast<const unsigned char *>(v_pool);
  a.k_scales = k_scales;
  a.v_scales = v_scales;
  a.table = block_table;
  a.query_start = query_start;
  a.seq_lens = seq_lens;
  a.out = out;
  a.lse = lse;
  a.R = n_requests;
  a.n_tokens = n_tokens;
  a.max_q = max_query_len;
  a.max_pages = max_pages;
  a.n_pages = n_pages;
  a.H = (int)n_heads;
  a.Hk = (int)n_kv_heads;
  a.D = (int)d_head;
  a.P = (int)page_size;
  a.q_stride = q_row_stride;
  a.scale = scale;
  a.causal = causal != 0;
  dim3 grid = linear_grid(n_tokens);
  grid.z = n_heads;
  if (kv_dtype == DFATTN_KV_E4M3)
    hipLaunchKernelGGL(attention_kernel<true>, grid, dim3(64), 0, static_cast<hipStream_t>(stream), a,
                       act_dtype == DFATTN_KV_BF16);
  else
    hipLaunchKernelGGL(attention_kernel<false>, grid, dim3(64), 0, static_cast<hipStream_t>(stream), a,
                       act_dtype == DFATTN_KV_BF16);
  return launched(fn);
}

}  // extern "C"
