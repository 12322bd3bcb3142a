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
  float *part_o, *part_ml;  // n_splits > 1: normalised outputs, and (m, l), of each (row, head, split)
  uint32_t n_tokens, max_q, max_pages, n_pages, q_tiles, n_splits, chunk, total;
  int H, Hk, D, P;
  size_t q_stride;
  float scale;
  bool causal, q_vec;
};

__device__ __forceinline__ void store_act(void *p, size_t i, float x, bool bf16) {
  if (bf16)
    static_cast<unsigned short *>(p)[i] = (unsigned short)bf16_bits(x);
  else
    static_cast<float *>(p)[i] = x;
}

// Maximum and sum over the four lanes l, l ^ 16, l ^ 32, l ^ 48 (one column of
// a 16x16 result).
__device__ __forceinline__ float column_max(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return pair_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float column_sum(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return pair_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// 8 codes (two dwords) as 8 fp16 values, exactly. int8: the code plus 128 as
// the low byte of 0x6400 is 1024 + 128 + code, which is exact in fp16.
template <bool E4M3>
__device__ __forceinline__ half8_t widen8(unsigned lo, unsigned hi) {
  half2_t h[4];
  if constexpr (E4M3) {
    h[0] = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false));
    h[1] = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true));
    h[2] = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false));
    h[3] = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true));
  } else {
    const half2_t off = {(half_t)-1152.f, (half_t)-1152.f};
    lo ^= 0x80808080u;
    hi ^= 0x80808080u;
    h[0] = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, lo, 0x07010700u)) + off;
    h[1] = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, lo, 0x07030702u)) + off;
    h[2] = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, hi, 0x07010700u)) + off;
    h[3] = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, hi, 0x07030702u)) + off;
  }
  return half8_t{h[0][0], h[0][1], h[1][0], h[1][1], h[2][0], h[2][1], h[3][0], h[3][1]};
}

__device__ __forceinline__ f32x4 mfma(half8_t a, half8_t b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// The rows a workgroup works on: request r, kv head hk, and the columns (query
// token, head of the group) col0 .. col0+16*QT-1 of its nq * G.
struct Where {
  uint32_t r, split, tile;
  int hk, nq, n_cols, active;
  uint32_t q0;       // first token of the request
  long long first;   // position of its first query
  int length, k_end; // cached positions; those the last column sees
};
__device__ __forceinline__ bool find_rows(const AttnArgs &a, Where &w, int cols_per_tile) {
  const int G = a.H / a.Hk;
  const uint32_t q0 = min(a.query_start[w.r], a.n_tokens), q1 = min(a.query_start[w.r + 1], a.n_tokens);
  const int nq = q1 > q0 ? (int)(q1 - q0) : 0;
  w.q0 = q0;
  w.nq = min((uint32_t)nq, a.max_q);
  w.n_cols = w.nq * G;
  const int col0 = (int)w.tile * cols_per_tile;
  if (col0 >= w.n_cols) return false;
  const uint32_t L = a.seq_lens[w.r];
  w.length = (int)min((unsigned long long)L, (unsigned long long)a.max_pages * a.P);
  w.first = (long long)L - nq;
  const int last = (min(w.n_cols, col0 + cols_per_tile) - 1) / G;
  w.k_end = a.causal ? (int)min((long long)w.length, max(w.first + last + 1, 0ll)) : w.length;
  w.active = max(1, (int)min((long long)a.n_splits, ((long long)w.k_end + a.chunk - 1) / a.chunk));
  return true;
}

constexpr int kWaves = 4;

// One workgroup: 16*QT columns (queries of one kv head) against the keys of one
// split, 64 keys a wave and step, the waves' results merged at the end.
//
// S^T = K Q^T on 16x16x32 tiles: A is K as it lies in memory, lane (m, g) =
// (l % 16, l / 16) reading 16 bytes of one key, B is Q. Row m of tile t is key
// 16 (m / 4) + 4 t + m % 4 of the 64, so that the result's lane (column, g)
// holds the 16 consecutive keys 16 g .. of one page group: their scales are one
// number each, and P goes as it stands into B of O^T += V^T P^T, whose A is V's
// columns as they lie in memory (16 keys of one column are 16 bytes). Nothing
// passes through LDS in the loop.
//
// q and P enter as NT fp16 terms: q times a power of two that brings its
// column's largest value to 2^14 .. 2^15; P times the page's scale and 2^(14 -
// r), where 2^r (r whole) bounds the largest such product so far: m and r move
// together, so weights keep 2^-39 of the largest one whatever the pages'
// scales.
template <bool E4M3, int NT, int NC, int QT>
__global__ __launch_bounds__(64 * kWaves, QT == 1 ? 2 : 1) void attention_kernel(AttnArgs a) {
  constexpr bool BF16 = NT == 1;
  constexpr int NV = 4 * NC;
  constexpr int kCols = 16 * QT;
  __shared__ float m_lds[kWaves][kCols], l_lds[kWaves][kCols];
  __shared__ __attribute__((aligned(16))) float o_lds[kWaves][kCols][20];
  uint32_t id = linear_block();
  if (id >= a.total) return;
  Where w;
  w.split = id % a.n_splits;
  id /= a.n_splits;
  w.hk = (int)(id % (uint32_t)a.Hk);
  id /= (uint32_t)a.Hk;
  w.tile = id % a.q_tiles;
  w.r = id / a.q_tiles;
  if (!find_rows(a, w, kCols)) return;
  if ((int)w.split >= w.active) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, m16 = lane & 15, g = lane >> 4;
  const int G = a.H / a.Hk, D = a.D, Dp = padded(D), P = a.P, col0 = (int)w.tile * kCols;
  const int k0 = (int)w.split * (int)a.chunk;
  const int k1 = (int)w.split + 1 == w.active ? w.k_end : k0 + (int)a.chunk;
  const uint32_t *table = a.table + (size_t)w.r * a.max_pages;
  const size_t head_bytes = (size_t)P * Dp;

  // Q, and where each column's keys end.
  half8_t q[QT][NC][2][NT];
  float col_scale[QT];
  int k_end[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int c = min(col0 + 16 * t + m16, w.n_cols - 1), j = c / G;
    const size_t row = (size_t)(w.q0 + j) * a.q_stride + (size_t)(w.hk * G + c % G) * D;
    k_end[t] = a.causal ? (int)min((long long)w.length, max(w.first + j + 1, 0ll)) : w.length;
    float x[NC][16];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const int d0 = 64 * n + 16 * g;
      if (a.q_vec) {
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
          if (d0 + i < D) {
            if constexpr (BF16) {
              const uint2 u = *reinterpret_cast<const uint2 *>(static_cast<const unsigned short *>(a.q) + row + d0 + i);
              f = make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u),
                              __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u));
            } else {
              f = *reinterpret_cast<const float4 *>(static_cast<const float *>(a.q) + row + d0 + i);
            }
          }
          x[n][i] = f.x;
          x[n][i + 1] = f.y;
          x[n][i + 2] = f.z;
          x[n][i + 3] = f.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[n][i] = d0 + i < D ? load_act(a.q, row + d0 + i, BF16) : 0.f;
      }
    }
    float top = 0.f;
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(x[n][i]));
    top = column_max(top);
    const int e = top > 0.f && top <= 3.4028234e38f ? 15 - __builtin_amdgcn_frexp_expf(top) : 0;
    col_scale[t] = __builtin_amdgcn_ldexpf(a.scale * kLog2e, -e);
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float y = __builtin_amdgcn_ldexpf(x[n][8 * h + i], e);
          const half_t hi = (half_t)y;
          q[t][n][h][0][i] = hi;
          if constexpr (NT == 2) q[t][n][h][1][i] = (half_t)(y - (float)hi);
        }
  }
  int min_end = k_end[0];  // of the workgroup's columns: the first one's
  min_end = __builtin_amdgcn_readfirstlane(min_end);

  float m[QT], l[QT], r[QT];
  f32x4 o[QT][NV];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    m[t] = -INFINITY;
    l[t] = 0.f;
    r[t] = -300.f;
#pragma unroll
    for (int n = 0; n < NV; ++n) o[t][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  struct Pages {
    uint32_t k, v;
  };
  struct Tile {
    u32x4 k[NC][4], v[NV];
    float ks, vs;
    bool ok;
  };
  // The pages of the step at keys t0: of the K rows this lane reads, and of the
  // V columns (and of the scores it gets). Steps past the end read its last page.
  auto load_pages = [&](int t0) {
    const int last = k1 - 1;
    return Pages{table[(unsigned)min(t0 + 16 * (m16 >> 2), last) / (unsigned)P],
                 table[(unsigned)min(t0 + 16 * g, last) / (unsigned)P]};
  };
  auto load_tile = [&](Tile &x, Pages p, int t0) {
    const bool ok_k = p.k < a.n_pages, ok_v = p.v < a.n_pages;
    x.ok = ok_v;
    const size_t hk_at = (size_t)(ok_k ? p.k : 0u) * a.Hk + w.hk, hv_at = (size_t)(ok_v ? p.v : 0u) * a.Hk + w.hk;
    x.ks = a.k_scales[hv_at];
    x.vs = a.v_scales[hv_at];
    const int kr = (int)((unsigned)(t0 + 16 * (m16 >> 2)) % (unsigned)P) + (m16 & 3);
    const unsigned char *kp = a.k + hk_at * head_bytes + (size_t)kr * Dp + 16 * g;
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int t = 0; t < 4; ++t)
        x.k[n][t] = 64 * n + 16 * g < Dp ? *reinterpret_cast<const u32x4 *>(kp + 64 * n + 4 * t * Dp) : u32x4{0, 0, 0, 0};
    const unsigned char *vp = a.v + hv_at * head_bytes + (size_t)m16 * P + (unsigned)(t0 + 16 * g) % (unsigned)P;
#pragma unroll
    for (int n = 0; n < NV; ++n)
      x.v[n] = 16 * n < Dp ? *reinterpret_cast<const u32x4 *>(vp + (size_t)16 * n * P) : u32x4{0, 0, 0, 0};
  };
  auto compute = [&](const Tile &x, int t0) {
    f32x4 s[QT][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int t = 0; t < QT; ++t) s[t][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const half8_t kh = widen8<E4M3>(x.k[n][j][2 * h], x.k[n][j][2 * h + 1]);
#pragma unroll
          for (int t = 0; t < QT; ++t)
#pragma unroll
            for (int e = 0; e < NT; ++e) s[t][j] = mfma(kh, q[t][n][h][e], s[t][j]);
        }
    }
    // Whether every column sees all 64 keys.
    const bool whole = t0 + 64 <= min(k1, min_end) && __all(x.ok);
    half8_t p[QT][2][NT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      const float f = x.ks * col_scale[t];
      float y[16], top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 16; ++i) y[i] = s[t][i >> 2][i & 3] * f;
      if (!whole) {
        const int n = x.ok ? min(k1, k_end[t]) - (t0 + 16 * g) : 0;  // of this lane's 16 keys
#pragma unroll
        for (int i = 0; i < 16; ++i) y[i] = i < n ? y[i] : -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, y[i]);
      const float m_new = fmaxf(m[t], column_max(top));
      const float base = m_new == -INFINITY ? 0.f : m_new;
      const float dm = m[t] - base;  // <= 0, -inf at first
      const float reach = column_max(top - base + __builtin_amdgcn_logf(x.vs));
      const float r_new = fmaxf(fmaxf(r[t] + __builtin_ceilf(fmaxf(dm, -1000.f)), __builtin_ceilf(reach)), -300.f);
      if (__any(m_new != m[t] || r_new != r[t])) {
        const float al = __builtin_amdgcn_exp2f(dm), ao = __builtin_amdgcn_ldexpf(al, (int)(r[t] - r_new));
        l[t] *= al;
#pragma unroll
        for (int n = 0; n < NV; ++n) o[t][n] *= ao;
        m[t] = m_new;
        r[t] = r_new;
      }
      const float pv = __builtin_amdgcn_ldexpf(x.vs, 14 - (int)r_new);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float e = __builtin_amdgcn_exp2f(y[i] - base);
        float u = e * pv;
        if (!whole) u = y[i] == -INFINITY ? 0.f : u;
        l[t] += e;
        const half_t hi = (half_t)u;
        p[t][i >> 3][0][i & 7] = hi;
        if constexpr (NT == 2) p[t][i >> 3][1][i & 7] = (half_t)(u - (float)hi);
      }
    }
    // V: the codes of keys past the end hold anything (e4m3: a NaN).
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      u32x4 c = x.v[n];
      if (!whole) {
        const int left = x.ok ? k1 - (t0 + 16 * g) : 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int b = left - 4 * i;  // bytes of this dword to keep
          c[i] &= b >= 4 ? 0xffffffffu : b <= 0 ? 0u : (1u << (8 * b)) - 1u;
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const half8_t vh = widen8<E4M3>(c[2 * h], c[2 * h + 1]);
#pragma unroll
        for (int t = 0; t < QT; ++t)
#pragma unroll
          for (int e = 0; e < NT; ++e) o[t][n] = mfma(vh, p[t][h][e], o[t][n]);
      }
    }
  };

  constexpr int kStep = 64 * kWaves;
  int t0 = k0 + 64 * wave;
  if (t0 < k1) {
    Tile x, y;
    load_tile(x, load_pages(t0), t0);
    Pages next = load_pages(t0 + kStep);
    while (true) {
      if (t0 + kStep < k1) load_tile(y, next, t0 + kStep);
      next = load_pages(t0 + 2 * kStep);
      compute(x, t0);
      t0 += kStep;
      if (t0 >= k1) break;
      if (t0 + kStep < k1) load_tile(x, next, t0 + kStep);
      next = load_pages(t0 + 2 * kStep);
      compute(y, t0);
      t0 += kStep;
      if (t0 >= k1) break;
    }
  }

  // The waves' results, 16 columns of d at a time. A column's output is
  // normalised here, so that it stays in the values' range.
  const bool direct = w.active == 1;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    l[t] = column_sum(l[t]);
    if (g == 0) {
      m_lds[wave][16 * t + m16] = m[t];
      l_lds[wave][16 * t + m16] = l[t];
    }
  }
  __syncthreads();
  float weight[QT];
  int shift[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int c = 16 * t + m16;
    float mm = m_lds[0][c];
#pragma unroll
    for (int v = 1; v < kWaves; ++v) mm = fmaxf(mm, m_lds[v][c]);
    const float base = mm == -INFINITY ? 0.f : mm;
    float ll = 0.f;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) ll += l_lds[v][c] * __builtin_amdgcn_exp2f(m_lds[v][c] - base);
    weight[t] = ll == 0.f ? 0.f : __builtin_amdgcn_exp2f(m[t] - base) / ll;
    shift[t] = (int)r[t] - 14;
    if (wave == 0 && g == 0 && col0 + c < w.n_cols) {
      const int h = w.hk * G + (col0 + c) % G;
      const size_t row = w.q0 + (col0 + c) / G;
      if (direct) {
        if (a.lse) a.lse[(size_t)h * a.n_tokens + row] = (mm + __builtin_log2f(ll)) * kLn2;
      } else {
        float *ml = a.part_ml + 2 * ((row * a.H + h) * a.n_splits + w.split);
        ml[0] = mm;
        ml[1] = ll;
      }
    }
  }
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    if (16 * n >= D) break;
    if (n > 0) __syncthreads();
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      f32x4 x = o[t][n] * weight[t];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = __builtin_amdgcn_ldexpf(x[i], shift[t]);
      *reinterpret_cast<f32x4 *>(&o_lds[wave][16 * t + m16][4 * g]) = x;
    }
    __syncthreads();
    for (int e = tid; e < 16 * kCols; e += 64 * kWaves) {
      const int c = e >> 4, d = e & 15;
      if (col0 + c >= w.n_cols || 16 * n + d >= D) continue;
      float x = o_lds[0][c][d];
#pragma unroll
      for (int v = 1; v < kWaves; ++v) x += o_lds[v][c][d];
      const int h = w.hk * G + (col0 + c) % G;
      const size_t row = w.q0 + (col0 + c) / G;
      if (direct)
        store_act(a.out, (row * a.H + h) * D + 16 * n + d, x, BF16);
      else
        a.part_o[((row * a.H + h) * a.n_splits + w.split) * D + 16 * n + d] = x;
    }
  }
}

// Rows whose keys were split: out = sum_s (l_s 2^(m_s - m) / l) o_s, one
// workgroup per (query token, head).
constexpr int kReduceThreads = 256;
__global__ __launch_bounds__(kReduceThreads) void attention_reduce_kernel(AttnArgs a, int cols_per_tile, bool bf16) {
  __shared__ float scratch[kReduceThreads / 64], w_lds[kReduceThreads], o_lds[kReduceThreads / 64][128];
  uint32_t id = linear_block();
  const int h = (int)(id % (uint32_t)a.H);
  id /= (uint32_t)a.H;
  const int j = (int)(id % a.max_q);
  Where w;
  w.r = id / a.max_q;
  if (id / a.max_q >= a.total) return;  // (total: the requests here)
  const int G = a.H / a.Hk;
  w.tile = (uint32_t)((j * G + h % G) / cols_per_tile);
  if (!find_rows(a, w, cols_per_tile) || j >= w.nq || w.active == 1) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = w.active, D = a.D;
  const size_t row = (size_t)(w.q0 + j) * a.H + h;
  const float *ml = a.part_ml + 2 * row * a.n_splits, *po = a.part_o + row * a.n_splits * D;
  auto reduce = [&](float v, bool is_max) {
    v = is_max ? wave_max(v) : wave_sum(v);
    __syncthreads();
    if (lane == 0) scratch[wave] = v;
    __syncthreads();
    float x = scratch[0];
    for (int i = 1; i < kReduceThreads / 64; ++i) x = is_max ? fmaxf(x, scratch[i]) : x + scratch[i];
    return x;
  };
  // (n is at most kReduceThreads.)
  const float ms = tid < n ? ml[2 * tid] : -INFINITY, ls = tid < n ? ml[2 * tid + 1] : 0.f;
  const float mm = reduce(ms, true), base = mm == -INFINITY ? 0.f : mm;
  const float ws = ls * __builtin_amdgcn_exp2f(ms - base);
  w_lds[tid] = ws;
  const float ll = reduce(ws, false), inv = ll == 0.f ? 0.f : 1.f / ll;
  float x0 = 0.f, x1 = 0.f;
#pragma unroll 8
  for (int s = wave; s < n; s += kReduceThreads / 64) {
    const float f = w_lds[s] * inv;
    // A split that saw nothing of this row has weight 0 and zeros.
    if (lane < D) x0 += f * po[(size_t)s * D + lane];
    if (lane + 64 < D) x1 += f * po[(size_t)s * D + lane + 64];
  }
  o_lds[wave][lane] = x0;
  o_lds[wave][lane + 64] = x1;
  __syncthreads();
  if (tid < D) {
    float x = 0.f;
    for (int i = 0; i < kReduceThreads / 64; ++i) x += o_lds[i][tid];
    store_act(a.out, row * D + tid, x, bf16);
  }
  if (tid == 0 && a.lse) a.lse[(size_t)h * a.n_tokens + w.q0 + j] = (mm + __builtin_log2f(ll)) * kLn2;
}

// How a call is cut: columns (query tokens times heads of a kv head) by 16, 32
// or 64, keys so that about kTargetGroups workgroups are there to share out.
constexpr uint32_t kTargetGroups = 2048, kMinChunk = 256, kMaxSplits = kReduceThreads;
struct Cut {
  uint32_t qt, q_tiles, n_splits, chunk;
};
Cut cut_of(uint32_t n_requests, uint32_t max_q, uint32_t max_len, uint32_t n_heads, uint32_t n_kv_heads, uint32_t d_head,
           bool split) {
  Cut c;
  const uint64_t cols = (uint64_t)max_q * (n_heads / n_kv_heads);
  c.qt = cols <= 16 ? 1 : cols <= 32 || d_head > 64 ? 2 : 4;
  c.q_tiles = (uint32_t)((cols + 16 * c.qt - 1) / (16 * c.qt));
  c.n_splits = 1;
  c.chunk = 1u << 30;
  if (split && max_len > kMinChunk) {
    const uint64_t groups = (uint64_t)n_requests * n_kv_heads * c.q_tiles;
    const uint64_t want = std::min<uint64_t>(kMaxSplits, (kTargetGroups + groups - 1) / groups);
    const uint32_t per = (uint32_t)((max_len + want - 1) / want);
    c.chunk = std::max(kMinChunk, (per + kMinChunk - 1) / kMinChunk * kMinChunk);
    c.n_splits = (max_len + c.chunk - 1) / c.chunk;
  }
  return c;
}

template <bool E4M3, int NT, int NC>
void launch_qt(const AttnArgs &a, uint32_t qt, dim3 grid, hipStream_t s) {
  if (qt == 1)
    hipLaunchKernelGGL((attention_kernel<E4M3, NT, NC, 1>), grid, dim3(64 * kWaves), 0, s, a);
  else if (qt == 2)
    hipLaunchKernelGGL((attention_kernel<E4M3, NT, NC, 2>), grid, dim3(64 * kWaves), 0, s, a);
  else if constexpr (NC == 1)
    hipLaunchKernelGGL((attention_kernel<E4M3, NT, NC, 4>), grid, dim3(64 * kWaves), 0, s, a);
}
template <bool E4M3, int NT>
void launch_nc(const AttnArgs &a, uint32_t qt, dim3 grid, hipStream_t s) {
  if (a.D <= 64)
    launch_qt<E4M3, NT, 1>(a, qt, grid, s);
  else
    launch_qt<E4M3, NT, 2>(a, qt, grid, s);
}

}  // namespace
}  // namespace dfattn

using namespace dfattn;
using namespace dfattn::kv8;

extern "C" {

size_t dfattn_kv8_attention_workspace_bytes(uint32_t n_requests, uint32_t n_tokens, uint32_t max_query_len,
                                            uint32_t max_seq_len, uint32_t n_heads, uint32_t n_kv_heads,
                                            uint32_t d_head) {
  if (n_requests == 0 || n_tokens == 0 || max_query_len == 0 || n_kv_heads == 0 || n_heads == 0 ||
      n_heads % n_kv_heads != 0 || n_heads > 65535u || n_requests > 65535u || n_tokens > (1u << 30) || d_head == 0 ||
      d_head > 128)
    return 0;
  const Cut c = cut_of(n_requests, std::min(max_query_len, n_tokens), max_seq_len, n_heads, n_kv_heads, d_head, true);
  return c.n_splits == 1 ? 0 : (size_t)n_tokens * n_heads * c.n_splits * (d_head + 2) * sizeof(float);
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
  if (n_heads > 65535u || n_requests > 65535u || n_tokens > (1u << 30) || (uint64_t)max_pages * page_size > (1ull << 30))
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
  max_query_len = std::min(max_query_len, n_tokens);
  const Cut c = cut_of(n_requests, max_query_len, max_seq_len, n_heads, n_kv_heads, d_head, workspace != nullptr);
  const size_t item = act_dtype == DFATTN_KV_F32 ? 4 : 2;
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
  a.part_o = static_cast<float *>(workspace);
  a.part_ml = a.part_o + (size_t)n_tokens * n_heads * c.n_splits * d_head;
  a.n_tokens = n_tokens;
  a.max_q = max_query_len;
  a.max_pages = max_pages;
  a.n_pages = n_pages;
  a.q_tiles = c.q_tiles;
  a.n_splits = c.n_splits;
  a.chunk = c.chunk;
  a.H = (int)n_heads;
  a.Hk = (int)n_kv_heads;
  a.D = (int)d_head;
  a.P = (int)page_size;
  a.q_stride = q_row_stride;
  a.scale = scale;
  a.causal = causal != 0;
  a.q_vec = d_head % 4 == 0 && q_row_stride % 4 == 0 && aligned_to(q, 4 * item);
  const uint64_t total = (uint64_t)n_requests * n_kv_heads * c.q_tiles * c.n_splits;
  const uint64_t rows = (uint64_t)n_requests * max_query_len * n_heads;
  if (total >= (1ull << 31) || (c.n_splits > 1 && rows >= (1ull << 31)))
    return record_error(DFATTN_ERR_OVERFLOW, std::string(fn) + ": shape is too large");
  a.total = (uint32_t)total;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid = linear_grid(total);
  const bool e4m3 = kv_dtype == DFATTN_KV_E4M3, bf16 = act_dtype == DFATTN_KV_BF16;
  if (e4m3 && bf16)
    launch_nc<true, 1>(a, c.qt, grid, s);
  else if (e4m3)
    launch_nc<true, 2>(a, c.qt, grid, s);
  else if (bf16)
    launch_nc<false, 1>(a, c.qt, grid, s);
  else
    launch_nc<false, 2>(a, c.qt, grid, s);
  st = launched(fn);
  if (st != DFATTN_OK || c.n_splits == 1) return st;
  a.total = n_requests;
  hipLaunchKernelGGL(attention_reduce_kernel, linear_grid(rows), dim3(kReduceThreads), 0, s, a, (int)(16 * c.qt), bf16);
  return launched(fn);
}

}  // extern "C"
