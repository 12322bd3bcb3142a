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
  // Shared out (see Share): normalised outputs [parts * Hk][2][cols][Dp] and (m, l) [parts * Hk][2][cols][2]
  // of the pieces, and the steps before each (request, tile) [R * q_tiles + 1].
  float *part_o, *part_ml;
  uint32_t *before;
  uint32_t R, n_tokens, max_q, max_pages, n_pages, q_tiles, parts, cols;
  int H, Hk, D, P;
  size_t q_stride;
  float scale;
  bool causal, q_vec, out_vec;  // q, out: four values at a time
};

// The first `left` of four values, to element i of the output.
__device__ __forceinline__ void store_out(const AttnArgs &a, size_t i, int left, f32x4 x, bool bf16) {
  unsigned short *const p16 = static_cast<unsigned short *>(a.out) + i;
  float *const p32 = static_cast<float *>(a.out) + i;
  if (a.out_vec) {
    if (bf16)
      *reinterpret_cast<uint2 *>(p16) =
          make_uint2(bf16_bits(x[0]) | bf16_bits(x[1]) << 16, bf16_bits(x[2]) | bf16_bits(x[3]) << 16);
    else
      *reinterpret_cast<f32x4 *>(p32) = x;
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (j >= left) break;
    if (bf16)
      p16[j] = (unsigned short)bf16_bits(x[j]);
    else
      p32[j] = x[j];
  }
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

// The product rounded, never fused with what is added to it.
__device__ __forceinline__ float times(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}
// 2^x, x <= 0 or -infinity, as part * 2^whole with part in (1/2, 1] (0 below 2^-1000): a weight too
// small for fp32 may still count, where its values are that much larger.
struct Power {
  float part, whole;
  __device__ __forceinline__ explicit Power(float x)
      : whole(__builtin_ceilf(fmaxf(x, -1000.f))) {
    part = __builtin_amdgcn_exp2f(x - whole);
  }
};

__device__ __forceinline__ f32x4 scaled(f32x4 x, int e) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = __builtin_amdgcn_ldexpf(x[i], e);
  return x;
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

constexpr int kWaves = 4, kStep = 64 * kWaves;  // keys of a workgroup's step
constexpr int kResident = 2, kCus = 256;  // workgroups on a CU (256 registers a wave)

// The rows a workgroup works on: request r, kv head hk, and the columns (query
// token, head of the group) col0 .. of its nq * G.
struct Where {
  uint32_t r, tile, q0;  // q0: first token of the request
  int hk, n_cols, col0;
  int length, k_end, first;  // cached positions, those the last column sees, that of the first query
  // The positions that query j sees.
  __device__ __forceinline__ int end_of(const AttnArgs &a, int j) const {
    return a.causal ? min(length, max(first + j + 1, 0)) : length;
  }
};
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }
// UNIFORM: r and tile are the same in all lanes, and so is what is read for them.
template <bool UNIFORM>
__device__ __forceinline__ bool find_rows(const AttnArgs &a, Where &w, int cols_per_tile) {
  const int G = a.H / a.Hk;
  uint32_t q0 = min(a.query_start[w.r], a.n_tokens), q1 = min(a.query_start[w.r + 1], a.n_tokens);
  uint32_t L = min(a.seq_lens[w.r], a.max_pages * (uint32_t)a.P);
  if constexpr (UNIFORM) {
    q0 = uniform(q0);
    q1 = uniform(q1);
    L = uniform(L);
  }
  const uint32_t nq = q1 > q0 ? q1 - q0 : 0;
  w.q0 = q0;
  w.n_cols = (int)min(nq, a.max_q) * G;
  w.col0 = (int)w.tile * cols_per_tile;
  w.length = (int)L;
  w.first = (int)L - (int)nq;
  const int last = (min(w.n_cols, w.col0 + cols_per_tile) - 1) / G;
  w.k_end = w.end_of(a, last);
  return w.col0 < w.n_cols;
}

// How the work of a call is shared out: the steps (kStep keys of one tile) of one kv
// head, request by request and tile by tile (a tile that sees nothing has one
// step, which writes its zeros), are cut into equal parts of `per`, one to a
// workgroup, and alike for each head. So every workgroup has the same work whatever
// the lengths are, and the heads of a page, which lie together, are read at the
// same time (by parts of one head after the other the call of 2 x 131072 keys took
// 79 us, so 65). A tile cut between workgroups is merged by
// attention_reduce_kernel; a workgroup has at most two such pieces, the tile that
// its part begins in (slot 0) and the one that goes on behind it (slot 1).
constexpr uint32_t kMinSteps = 2;
struct Share {
  uint32_t total, per;
  // before: the steps before each (request, tile)
  __device__ __forceinline__ Share(const uint32_t *before, const AttnArgs &a)
      : total(uniform(before[a.R * a.q_tiles])), per(max((total + a.parts - 1) / a.parts, kMinSteps)) {}
};

// One workgroup: 16*QT columns (queries of one kv head) against the keys of one
// part, 64 keys a wave and step, the waves' results merged at the end.
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
// together, so products keep 2^-39 of the largest one whatever the pages'
// scales. Powers of two that fp32 has no room for (a weight of 2^-200 before values of
// 2^120) are kept apart as exponents, here and in the merges. bf16 takes one term: q fits it, and P's
// rounding of at most 2^-11 is an eighth of the output's (against float64 1.6e-3 as for fp32 sums
// rounded once; 6 outputs in 100 are the neighbouring bf16 value).
//
// Measured (12 heads of 64): one query on 2 x 131072 keys 61 us, 4.9 TB/s, on 64 requests of up to
// 4096 (e4m3, bf16) 47 us, 4.4 TB/s: memory, of which two workgroups a CU keep enough on its
// way (three took 69 us for 67, with the merge). Chunks of 3 x 500 queries of up to 4096 keys 53-61
// us: VALU instructions take 60 % of a SIMD's time (ten for each product), the matrix pipe 20 %, and the
// waves wait 30 % of theirs: two waves a SIMD, in each of which the barriers keep products and
// exponentials apart, overlap no better. fp32 with 48 columns, and 32 of more than 64 values, spill 2 to 19
// registers, none of them in the loop.
template <bool E4M3, int NT, int NC, int QT, bool SHARED>
__global__ __launch_bounds__(64 * kWaves, kResident) void attention_kernel(AttnArgs a) {
  constexpr bool BF16 = NT == 1;
  constexpr int NV = 4 * NC;
  constexpr int kCols = 16 * QT;
  extern __shared__ uint32_t before[];  // SHARED: R * q_tiles + 1
  __shared__ float m_lds[kWaves][kCols], l_lds[kWaves][kCols];
  __shared__ uint32_t wave_steps[kWaves];
  __shared__ union {
    half8_t q[QT][NC][2][NT][64];
    float o[kWaves][kCols][68];  // (once Q has been used)
  } lds;
  __shared__ float scale_lds[kCols];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, m16 = lane & 15, g = lane >> 4;
  const int G = a.H / a.Hk, D = a.D, Dp = padded(D), P = a.P;
  uint32_t at = 0, end = 0, pair = 0;  // this workgroup's steps, and the (request, tile) they are at
  Where w;
  if constexpr (SHARED) {
    const uint32_t n = a.R * a.q_tiles, each = (n + 64 * kWaves - 1) / (64 * kWaves);
    const uint32_t i0 = min(n, tid * each), i1 = min(n, i0 + each);
    auto steps_of = [&](uint32_t i) {
      Where v;
      v.r = i / a.q_tiles;
      v.tile = i % a.q_tiles;
      return find_rows<false>(a, v, kCols) ? max(1u, (uint32_t)(v.k_end + kStep - 1) / kStep) : 0u;
    };
    uint32_t mine = 0;
    for (uint32_t i = i0; i < i1; ++i) {
      const uint32_t x = steps_of(i);
      before[i] = mine;
      mine += x;
    }
    uint32_t sum = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const uint32_t o = __shfl_up(sum, off, 64);
      if (lane >= off) sum += o;
    }
    if (lane == 63) wave_steps[wave] = sum;
    __syncthreads();
    uint32_t base = sum - mine;
    for (int v = 0; v < wave; ++v) base += wave_steps[v];
    for (uint32_t i = i0; i < i1; ++i) before[i] += base;
    if (tid == 64 * kWaves - 1) before[n] = base + mine;
    __syncthreads();
    if (blockIdx.x == 0)
      for (uint32_t i = tid; i <= n; i += 64 * kWaves) a.before[i] = before[i];
    const Share sh(before, a);
    const uint32_t part = blockIdx.x / (uint32_t)a.Hk;
    w.hk = (int)(blockIdx.x % (uint32_t)a.Hk);
    at = part * sh.per;
    end = min(at + sh.per, sh.total);
    if (at >= end) return;
    pair = 0;  // the last (request, tile) with before[pair] <= at
    for (uint32_t hi = n; hi - pair > 1;) {
      const uint32_t mid = (pair + hi) / 2;
      if (uniform(before[mid]) <= at)
        pair = mid;
      else
        hi = mid;
    }
  } else {
    uint32_t id = linear_block();
    w.tile = id % a.q_tiles;
    id /= a.q_tiles;
    w.hk = (int)(id % (uint32_t)a.Hk);
    w.r = id / (uint32_t)a.Hk;
    if (w.r >= a.R || !find_rows<true>(a, w, kCols)) return;
  }
  bool begins = true;  // the first of this workgroup's tiles
  while (true) {
  int k0 = 0, k1;
  bool direct = true;
  if constexpr (SHARED) {
    w.r = pair / a.q_tiles;
    w.tile = pair % a.q_tiles;
    find_rows<true>(a, w, kCols);
    const uint32_t s0 = uniform(before[pair]), n = uniform(before[pair + 1]) - s0, s1 = min(s0 + n, end);
    k0 = (int)(at - s0) * kStep;
    k1 = min(w.k_end, (int)(s1 - s0) * kStep);
    direct = at == s0 && s1 == s0 + n;
    at = s1;
  } else {
    k1 = w.k_end;
  }
  const int col0 = w.col0;
  const uint32_t *table = a.table + (size_t)w.r * a.max_pages;

  // Q as the products take it, in LDS for all waves (16 columns converted by one of
  // them each), and where each column's keys end.
  int k_end[QT];
  const int min_end = w.end_of(a, col0 / G);  // of the workgroup's columns: the first one's
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int c = min(col0 + 16 * t + m16, w.n_cols - 1), j = c / G;
    k_end[t] = w.end_of(a, j);
    if (t % kWaves != wave) continue;
    const size_t row = (size_t)(w.q0 + j) * a.q_stride + (size_t)(w.hk * G + c % G) * D;
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
    // (A negative scale's sign goes into q.)
    if (g == 0) scale_lds[16 * t + m16] = __builtin_amdgcn_ldexpf(fabsf(a.scale) * kLog2e, -e);
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        half8_t q[2];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float y = __builtin_amdgcn_ldexpf(a.scale < 0.f ? -x[n][8 * h + i] : x[n][8 * h + i], e);
          q[0][i] = (half_t)y;
          q[1][i] = (half_t)(y - (float)q[0][i]);
        }
#pragma unroll
        for (int e2 = 0; e2 < NT; ++e2) lds.q[t][n][h][e2][lane] = q[e2];
      }
  }
  __syncthreads();
  float col_scale[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) col_scale[t] = scale_lds[16 * t + m16];

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

  // The pages that this lane reads in a step: that of the K rows (group m16 / 4 of
  // the step's four groups of 16 keys), and that of the V columns and of the scores
  // it gets (group g). `at` counts groups of 16 keys, split into a page's index and
  // the place within; a step moves all by 4 * kWaves groups.
  struct Place {
    uint32_t index, off, page;
  };
  struct KTile {
    u32x4 c[NC][4];
  };
  struct VTile {
    u32x4 c[NV];
    float ks, vs;
    bool ok;
  };
  const uint32_t p16 = (uint32_t)P >> 4, move_i = 4 * kWaves / p16, move_o = 4 * kWaves % p16;
  const uint32_t last_index = k1 > 0 ? (uint32_t)(k1 - 1) / (uint32_t)P : 0;
  auto place_of = [&](int t0, int group) {
    const uint32_t at = ((uint32_t)t0 >> 4) + group;
    return Place{at / p16, at % p16, 0u};
  };
  // (Steps past the end look up its last page.)
  auto look_up = [&](Place &p) { p.page = table[min(p.index, last_index)]; };
  auto advance = [&](Place &p) {
    p.index += move_i;
    p.off += move_o;
    if (p.off >= p16) {
      p.off -= p16;
      ++p.index;
    }
  };
  const uint32_t page_bytes = (uint32_t)a.Hk * (uint32_t)(P * Dp);
  // Lanes past a row's last 16 bytes read those again: Q is 0 there.
  const unsigned char *k_lane = a.k + (size_t)w.hk * (P * Dp) + (m16 & 3) * Dp;
  const unsigned char *v_lane = a.v + (size_t)w.hk * (P * Dp) + (size_t)m16 * P;
  int k_col[NC];
#pragma unroll
  for (int n = 0; n < NC; ++n) k_col[n] = min(64 * n + 16 * g, Dp - 16);
  auto load_k = [&](KTile &x, const Place &p) {
    const uint32_t page = p.page < a.n_pages ? p.page : 0u;
    const unsigned char *kp = k_lane + ((uint64_t)page * page_bytes + __umul24(16 * p.off, Dp));
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int t = 0; t < 4; ++t) x.c[n][t] = *reinterpret_cast<const u32x4 *>(kp + (k_col[n] + 4 * t * Dp));
  };
  auto load_v = [&](VTile &x, const Place &p) {
    x.ok = p.page < a.n_pages;
    const uint32_t page = x.ok ? p.page : 0u;
    const size_t head = (size_t)page * (uint32_t)a.Hk + w.hk;
    x.ks = a.k_scales[head];
    x.vs = a.v_scales[head];
    const unsigned char *vp = v_lane + ((uint64_t)page * page_bytes + 16 * p.off);
#pragma unroll
    for (int n = 0; n < NV; ++n) x.c[n] = *reinterpret_cast<const u32x4 *>(vp + min(16 * n, Dp - 16) * P);
  };
  auto score = [&](const KTile &kt, f32x4 (&s)[QT][4]) {
    // (Q is read from LDS in every step: kept in registers it would cost a wave per SIMD.)
    asm volatile("" ::: "memory");
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int t = 0; t < QT; ++t) s[t][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        half8_t q[QT][NT];
#pragma unroll
        for (int t = 0; t < QT; ++t)
#pragma unroll
          for (int e = 0; e < NT; ++e) q[t][e] = lds.q[t][n][h][e][lane];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const half8_t kh = widen8<E4M3>(kt.c[n][j][2 * h], kt.c[n][j][2 * h + 1]);
#pragma unroll
          for (int t = 0; t < QT; ++t)
#pragma unroll
            for (int e = 0; e < NT; ++e) s[t][j] = mfma(kh, q[t][e], s[t][j]);
          if (j % 2 == 1) __builtin_amdgcn_sched_barrier(0);
        }
      }
  };
  auto absorb = [&](f32x4 (&s)[QT][4], VTile &vt, int t0) {
    float f[QT], vs[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      // >= 0, or NaN. (A scale of 0 is as good as 1e-36, and -infinity times that is no NaN.)
      f[t] = vt.ks * col_scale[t];
      f[t] = f[t] < 1e-36f ? 1e-36f : f[t];
      vs[t] = vt.vs;
    }
    // Where not every column sees all 64 keys: what it does not see gets the score -infinity,
    // whose probability is 0; where it sees none of the lane's 16 keys, the page's scales are
    // left out too (they may be NaN). The codes of keys past the end hold anything (e4m3: a NaN).
    if (!(t0 + 64 <= min(k1, min_end) && __all(vt.ok))) {
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        const int n = vt.ok ? min(k1, k_end[t]) - (t0 + 16 * g) : 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[t][i >> 2][i & 3] = i < n ? s[t][i >> 2][i & 3] : -INFINITY;
        f[t] = n > 0 ? f[t] : 1.f;
        vs[t] = n > 0 ? vs[t] : 0.f;
      }
      const int left = vt.ok ? k1 - (t0 + 16 * g) : 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int b = left - 4 * i;  // bytes of this dword to keep
        const unsigned keep = b >= 4 ? 0xffffffffu : b <= 0 ? 0u : (1u << (8 * b)) - 1u;
#pragma unroll
        for (int n = 0; n < NV; ++n) vt.c[n][i] &= keep;
      }
    }
    half8_t p[QT][2][NT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      float top = s[t][0][0];
#pragma unroll
      for (int i = 1; i < 16; ++i) top = fmaxf(top, s[t][i >> 2][i & 3]);
      top = times(top, f[t]);
      const float m_new = fmaxf(m[t], column_max(top));
      const float base = m_new == -INFINITY ? 0.f : m_new;
      const Power dm(m[t] - base);
      const float lv = __builtin_amdgcn_logf(vs[t]), reach = column_max(top - base + lv);
      const float r_new = fmaxf(fmaxf(r[t] + dm.whole, __builtin_ceilf(reach)), -300.f);
      if (__any(m_new != m[t] || r_new != r[t])) {
        const float ao = __builtin_amdgcn_ldexpf(dm.part, (int)(dm.whole + (r[t] - r_new)));
        l[t] *= __builtin_amdgcn_ldexpf(dm.part, (int)dm.whole);
#pragma unroll
        for (int n = 0; n < NV; ++n) o[t][n] *= ao;
        m[t] = m_new;
        r[t] = r_new;
      }
      float add = -base, back = 1.f;
      int x = 14 - (int)r_new;
      // base is a rounded product: the fused one below is off from it by up to 2^-25 of a score, for the
      // largest too. From 2^20 on that is more than the weights have room for.
      if (__any(fabsf(base) > 0x1p20f)) {
        const bool large = fabsf(base) > 0x1p20f;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          s[t][i >> 2][i & 3] = large ? times(s[t][i >> 2][i & 3], f[t]) - base : s[t][i >> 2][i & 3];
        f[t] = large ? 1.f : f[t];
        add = large ? 0.f : add;
      }
      // A page may have a scale far above 2^r where its probabilities are as small: 2^k of the factor
      // then goes into the exponentials (so that it stays in fp32's range) and out of their sum.
      if (__any(lv - r_new > 100.f)) {
        const int k = lv - r_new > 100.f ? (int)(lv - r_new) - 50 : 0;
        add += (float)k;
        back = __builtin_amdgcn_ldexpf(1.f, -k);
        x -= k;
      }
      const float pv = __builtin_amdgcn_ldexpf(vs[t], x);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float e = __builtin_amdgcn_exp2f(fmaf(s[t][i >> 2][i & 3], f[t], add));
        l[t] = fmaf(e, back, l[t]);
        const float u = e * pv;
        const half_t hi = (half_t)u;
        p[t][i >> 3][0][i & 7] = hi;
        if constexpr (NT == 2) p[t][i >> 3][1][i & 7] = (half_t)(u - (float)hi);
      }
    }
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      if (16 * n >= Dp) continue;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const half8_t vh = widen8<E4M3>(vt.c[n][2 * h], vt.c[n][2 * h + 1]);
#pragma unroll
        for (int t = 0; t < QT; ++t)
#pragma unroll
          for (int e = 0; e < NT; ++e) o[t][n] = mfma(vh, p[t][h][e], o[t][n]);
      }
      if (n % 2 == 1) __builtin_amdgcn_sched_barrier(0);
    }
  };

  int t0 = k0 + 64 * wave;
  if (t0 < k1) {
    Place pk = place_of(t0, m16 >> 2), pv = place_of(t0, g);
    look_up(pk);
    look_up(pv);
    // V of this step and K of the next are on their way while the other is used: K's
    // registers are free again after the scores, V's after the products.
    KTile kt;
    VTile vt;
    load_k(kt, pk);
    advance(pk);
    look_up(pk);
    for (; t0 < k1; t0 += kStep) {
      load_v(vt, pv);
      advance(pv);
      look_up(pv);
      __builtin_amdgcn_sched_barrier(0);
      f32x4 s[QT][4];
      score(kt, s);
      __builtin_amdgcn_sched_barrier(0);
      if (t0 + kStep < k1) load_k(kt, pk);
      advance(pk);
      look_up(pk);
      __builtin_amdgcn_sched_barrier(0);
      absorb(s, vt, t0);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // The waves' results, 16 columns of d at a time. A column's output is
  // normalised here, so that it stays in the values' range.
  const size_t slot = SHARED ? (size_t)(2 * blockIdx.x + (begins ? 0 : 1)) * a.cols : 0;
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
    const Power dm(m[t] - base);
    weight[t] = ll == 0.f ? 0.f : dm.part / ll;
    shift[t] = (int)(r[t] + dm.whole) - 14;
    if (wave == 0 && g == 0 && col0 + c < w.n_cols) {
      const int h = w.hk * G + (col0 + c) % G;
      const size_t row = w.q0 + (col0 + c) / G;
      if (direct) {
        if (a.lse) a.lse[(size_t)h * a.n_tokens + row] = (mm + __builtin_log2f(ll)) * kLn2;
      } else {
        float *ml = a.part_ml + 2 * (slot + c);
        ml[0] = mm;
        ml[1] = ll;
      }
    }
  }
#pragma unroll
  for (int half = 0; half < NC; ++half) {
    if (half > 0) __syncthreads();
#pragma unroll
    for (int n = 4 * half; n < 4 * half + 4; ++n)
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        f32x4 x = o[t][n] * weight[t];
        x = scaled(x, shift[t]);
        *reinterpret_cast<f32x4 *>(&lds.o[wave][16 * t + m16][16 * (n - 4 * half) + 4 * g]) = x;
      }
    __syncthreads();
#pragma unroll
    for (int e = tid; e < 16 * kCols; e += 64 * kWaves) {
      const int c = e >> 4, d = 64 * half + 4 * (e & 15);
      if (col0 + c >= w.n_cols || d >= D) continue;
      f32x4 x = *reinterpret_cast<const f32x4 *>(&lds.o[0][c][4 * (e & 15)]);
#pragma unroll
      for (int v = 1; v < kWaves; ++v) x += *reinterpret_cast<const f32x4 *>(&lds.o[v][c][4 * (e & 15)]);
      if (direct) {
        const int h = w.hk * G + (col0 + c) % G;
        const size_t row = w.q0 + (col0 + c) / G;
        store_out(a, (row * a.H + h) * D + d, D - d, x, BF16);
      } else {
        *reinterpret_cast<f32x4 *>(a.part_o + (slot + c) * Dp + d) = x;
      }
    }
  }
  if constexpr (!SHARED) return;
  if (at >= end) return;
  // The next tile that has steps.
  begins = false;
  do ++pair;
  while (uniform(before[pair + 1]) <= at);
  __syncthreads();
  }
}

// The tiles that were cut between workgroups: out = sum_i (l_i 2^(m_i - m) / l) o_i
// over the pieces i. A quarter of a wave takes a column, a lane four or eight of its
// values, 16 pieces' (m, l) at a time. Few columns (a generated token) are shared by the
// workgroup's four waves where there are more than kAhead pieces, so that all
// are read at once. Bound by the latency of two dependent reads: what says where the pieces
// are, then (m, l) and the first kAhead outputs together: 5-6 us (chunks of 3 x 500 queries with
// a wave to a column, one after the other, 13).
constexpr int kReduceWaves = 4, kAhead = 8;
__host__ __device__ inline uint32_t reduce_cols(uint32_t cols) { return cols > 16 ? 16 : 4; }
template <int NC>
__global__ __launch_bounds__(64 * kReduceWaves) void attention_reduce_kernel(AttnArgs a, int cols_per_tile, bool bf16) {
  __shared__ float ml_lds[kReduceWaves][4][2];
  __shared__ f32x4 o_lds[kReduceWaves][NC][64];
  const uint32_t per_group = reduce_cols(a.cols), col_groups = (a.cols + per_group - 1) / per_group;
  uint32_t id = linear_block();
  const int c0 = (int)(id % col_groups * per_group);
  id /= col_groups;
  Where w;
  w.tile = id % a.q_tiles;
  id /= a.q_tiles;
  w.hk = (int)(id % (uint32_t)a.Hk);
  w.r = id / (uint32_t)a.Hk;
  if (w.r >= a.R) return;
  const uint32_t i0 = w.r * a.q_tiles + w.tile;
  const uint32_t b0 = a.before[i0], b1 = a.before[i0 + 1];
  const Share sh(a.before, a);
  const bool any = find_rows<true>(a, w, cols_per_tile);
  const uint32_t s0 = uniform(b0), n = uniform(b1) - s0;
  const uint32_t first = s0 / sh.per, parts = n == 0 ? 0 : (s0 + n - 1) / sh.per - first + 1;
  if (!any || parts <= 1) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = (int)uniform(tid >> 6), l16 = lane & 15, G = a.H / a.Hk, D = a.D,
            Dp = padded(D);
  const bool second = s0 % sh.per != 0;  // the first piece lies in slot 1 of its workgroup
  auto slot_of = [&](uint32_t i) {
    return (size_t)(2 * ((first + i) * (uint32_t)a.Hk + w.hk) + (i == 0 && second ? 1 : 0)) * a.cols;
  };
  // shared: wave v takes the pieces v, v + 4, ... of all four columns; else all of its own four.
  const bool shared = per_group == 4;
  if (shared && parts <= kAhead && wave > 0) return;
  const bool split = shared && parts > kAhead;
  const int c = c0 + (shared ? 0 : 4 * wave) + (lane >> 4);
  const bool on = c < (int)a.cols && w.col0 + c < w.n_cols;
  const uint32_t p0 = split ? wave : 0, step = split ? kReduceWaves : 1;
  const uint32_t mine = parts > p0 ? (parts - p0 + step - 1) / step : 0;  // this wave's pieces: p0 + step * j
  // Running over 16 pieces at a time: m, l and the output, always normalised, so that it stays in the
  // values' range.
  float m = -INFINITY, l = 0.f;
  f32x4 x[NC];
#pragma unroll
  for (int k = 0; k < NC; ++k) x[k] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (uint32_t j0 = 0; j0 < mine; j0 += 16) {
    float mp = -INFINITY, lp = 0.f;
    if (on && j0 + l16 < mine) {
      const float *ml = a.part_ml + 2 * (slot_of(p0 + step * (j0 + l16)) + c);
      mp = ml[0];
      lp = ml[1];
    }
    f32x4 y[kAhead][NC];
    auto load = [&](uint32_t j) {
#pragma unroll
      for (uint32_t i = 0; i < kAhead; ++i)
#pragma unroll
        for (int k = 0; k < NC; ++k) {
          const int d = 64 * k + 4 * l16;
          y[i][k] = f32x4{0.f, 0.f, 0.f, 0.f};
          if (on && j + i < mine && d < Dp)
            y[i][k] = *reinterpret_cast<const f32x4 *>(a.part_o + (slot_of(p0 + step * (j + i)) + c) * Dp + d);
        }
    };
    load(j0);
    float top = mp;
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    const float m_new = fmaxf(m, top), base = m_new == -INFINITY ? 0.f : m_new;
    const Power old(m - base), piece(mp - base);
    m = m_new;
    // (l of a piece, and so its weight, is 0 where it saw nothing, and NaN where that is its sum.)
    lp *= piece.part;
    float sum = __builtin_amdgcn_ldexpf(lp, (int)piece.whole);
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) sum += __shfl_xor(sum, o, 64);
    const float before = l * old.part;
    l = __builtin_amdgcn_ldexpf(before, (int)old.whole) + sum;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    lp *= inv;
#pragma unroll
    for (int k = 0; k < NC; ++k) x[k] = before * inv * scaled(x[k], (int)old.whole);
#pragma unroll
    for (uint32_t half = 0; half < 2; ++half) {
      if (half == 1) {
        if (j0 + kAhead >= mine) break;
        load(j0 + kAhead);
      }
#pragma unroll
      for (uint32_t i = 0; i < kAhead; ++i) {
        const int from = (lane & 48) + (int)(half * kAhead + i), whole = __shfl((int)piece.whole, from, 64);
        const float f = __shfl(lp, from, 64);
#pragma unroll
        for (int k = 0; k < NC; ++k) x[k] += f * scaled(y[i][k], whole);
      }
    }
  }
  if (split) {
    if (l16 == 0) {
      ml_lds[wave][lane >> 4][0] = m;
      ml_lds[wave][lane >> 4][1] = l;
    }
#pragma unroll
    for (int k = 0; k < NC; ++k) o_lds[wave][k][lane] = x[k];
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int v = 1; v < kReduceWaves; ++v) m = fmaxf(m, ml_lds[v][lane >> 4][0]);
    const float base = m == -INFINITY ? 0.f : m;
    float f[kReduceWaves];
    int whole[kReduceWaves];
    l = 0.f;
#pragma unroll
    for (int v = 0; v < kReduceWaves; ++v) {
      const Power dm(ml_lds[v][lane >> 4][0] - base);
      f[v] = ml_lds[v][lane >> 4][1] * dm.part;
      whole[v] = (int)dm.whole;
      l += __builtin_amdgcn_ldexpf(f[v], whole[v]);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      x[k] = scaled(x[k], whole[0]) * (f[0] * inv);  // (wave 0's own)
#pragma unroll
      for (int v = 1; v < kReduceWaves; ++v) x[k] += scaled(o_lds[v][k][lane], whole[v]) * (f[v] * inv);
    }
  }
  if (!on) return;
  const int h = w.hk * G + (w.col0 + c) % G;
  const size_t row = w.q0 + (w.col0 + c) / G, out = (row * a.H + h) * D;
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    const int d = 64 * k + 4 * l16;
    if (d < D) store_out(a, out + d, D - d, x[k], bf16);
  }
  if (l16 == 0 && a.lse) a.lse[(size_t)h * a.n_tokens + row] = (m + __builtin_log2f(l)) * kLn2;
}

// How a call is cut: columns (query tokens times heads of a kv head) by 16, 32 or 48. 48
// share each widened code with half as many columns again, where d_head lets them fit
// registers: 2 x 720 queries of 4096 keys, 12 heads of 64, 76 us, so 84 (bf16 56, so 62), though
// fewer tiles may share out less evenly: 3 x 500 of 900 to 4096 keys 64 us, so 62;
// 8 x 64 queries leave a third of them empty, 37 us, so 32; and where the work isn't shared
// out a second round of workgroups costs more (4 x 512 queries of 512 keys 24 us, so 23).
// (64 columns spill registers: 3 x 500 queries 79 us, so 61.)
//
// The work is shared out where sequences may be longer than kShareFrom keys (kShareFromFew, up
// to 16 columns) and the (request, tile) pairs fit LDS; else one workgroup takes each tile and
// no merge is launched. 64 requests of up to 2048 keys take 39 us shared out, 32 not; one of
// 1536 11 either way on the GPU, 21 and 16.5 with its calls; but one of 4096 11.6 and 23.6, 32 of up to
// 4096 33 and 38, and 2 x 200 queries of 2048 keys 25 and 27.
constexpr uint32_t kShareFrom = 1024, kShareFromFew = 2048, kMaxPairs = 4096, kManyColumns = 192;
struct Cut {
  uint32_t qt, cols, q_tiles, parts;  // parts: 0, not shared out
  size_t part_bytes, bytes;
};
Cut cut_of(uint32_t n_requests, uint32_t max_q, uint32_t max_len, uint32_t n_heads, uint32_t n_kv_heads, uint32_t d_head) {
  Cut c{};
  const uint64_t cols = (uint64_t)max_q * (n_heads / n_kv_heads);
  const uint64_t tiles = n_requests * ((cols + 47) / 48);  // of 48
  const bool at_once = max_len > kShareFrom ? tiles <= kMaxPairs : tiles * n_kv_heads <= kCus * kResident;
  c.qt = cols <= 16 ? 1 : cols >= kManyColumns && d_head <= 64 && at_once ? 3 : 2;
  c.cols = (uint32_t)std::min<uint64_t>(cols, 16 * c.qt);
  c.q_tiles = (uint32_t)((cols + 16 * c.qt - 1) / (16 * c.qt));
  const uint64_t pairs = (uint64_t)n_requests * c.q_tiles;
  if (max_len <= (c.qt == 1 ? kShareFromFew : kShareFrom) || pairs > kMaxPairs) return c;
  // As many workgroups as run at a time.
  c.parts = std::max(1u, kCus * kResident / n_kv_heads);
  const uint64_t slots = 2ull * c.parts * n_kv_heads * c.cols;
  c.part_bytes = slots * padded((int)d_head) * sizeof(float);
  c.bytes = c.part_bytes + slots * 2 * sizeof(float) + (pairs + 1) * sizeof(uint32_t);
  return c;
}

template <bool E4M3, int NT, int NC, int QT>
void launch(const AttnArgs &a, hipStream_t s) {
  if (a.parts > 0)
    hipLaunchKernelGGL((attention_kernel<E4M3, NT, NC, QT, true>), dim3(a.parts * (uint32_t)a.Hk), dim3(64 * kWaves),
                       ((size_t)a.R * a.q_tiles + 1) * sizeof(uint32_t), s, a);
  else
    hipLaunchKernelGGL((attention_kernel<E4M3, NT, NC, QT, false>), linear_grid((size_t)a.R * a.Hk * a.q_tiles),
                       dim3(64 * kWaves), 0, s, a);
}
template <bool E4M3, int NT>
void launch_shape(const AttnArgs &a, uint32_t qt, hipStream_t s) {
  if (a.D <= 64 && qt == 1)
    launch<E4M3, NT, 1, 1>(a, s);
  else if (a.D <= 64 && qt == 2)
    launch<E4M3, NT, 1, 2>(a, s);
  else if (a.D <= 64)
    launch<E4M3, NT, 1, 3>(a, s);
  else if (qt == 1)
    launch<E4M3, NT, 2, 1>(a, s);
  else
    launch<E4M3, NT, 2, 2>(a, s);
}

}  // namespace
}  // namespace dfattn

using namespace dfattn;
using namespace dfattn::kv8;

extern "C" {

// A request's columns (queries times heads of a kv head) are counted in 32 bits.
static bool too_many_columns(uint32_t n_tokens, uint32_t max_query_len, uint32_t group) {
  return (uint64_t)std::min(max_query_len, n_tokens) * group > (1ull << 30);
}

size_t dfattn_kv8_attention_workspace_bytes(uint32_t n_requests, uint32_t n_tokens, uint32_t max_query_len,
                                            uint32_t max_seq_len, uint32_t n_heads, uint32_t n_kv_heads,
                                            uint32_t d_head) {
  if (n_requests == 0 || n_tokens == 0 || max_query_len == 0 || n_kv_heads == 0 || n_heads == 0 ||
      n_heads % n_kv_heads != 0 || n_heads > 65535u || n_requests > 65535u || n_tokens > (1u << 30) || d_head == 0 ||
      d_head > 128 || too_many_columns(n_tokens, max_query_len, n_heads / n_kv_heads))
    return 0;
  return cut_of(n_requests, std::min(max_query_len, n_tokens), max_seq_len, n_heads, n_kv_heads, d_head).bytes;
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
  if (n_heads > 65535u || n_requests > 65535u || n_tokens > (1u << 30) ||
      (uint64_t)max_pages * page_size > (1ull << 30) || too_many_columns(n_tokens, max_query_len, n_heads / n_kv_heads))
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
  Cut c = cut_of(n_requests, max_query_len, max_seq_len, n_heads, n_kv_heads, d_head);
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
  // The steps are counted in 32 bits.
  const uint64_t most = (uint64_t)n_requests * c.q_tiles * (((uint64_t)max_pages * page_size + kStep - 1) / kStep);
  if (workspace == nullptr || most >= (1ull << 31)) c.parts = 0;
  a.parts = c.parts;
  if (c.parts > 0) {
    a.part_o = static_cast<float *>(workspace);
    a.part_ml = a.part_o + c.part_bytes / sizeof(float);
    a.before = reinterpret_cast<uint32_t *>(a.part_ml + 2ull * 2 * c.parts * n_kv_heads * c.cols);
  }
  a.R = n_requests;
  a.n_tokens = n_tokens;
  a.max_q = max_query_len;
  a.max_pages = max_pages;
  a.n_pages = n_pages;
  a.q_tiles = c.q_tiles;
  a.cols = c.cols;
  a.H = (int)n_heads;
  a.Hk = (int)n_kv_heads;
  a.D = (int)d_head;
  a.P = (int)page_size;
  a.q_stride = q_row_stride;
  a.scale = scale;
  a.causal = causal != 0;
  a.q_vec = d_head % 4 == 0 && q_row_stride % 4 == 0 && aligned_to(q, 4 * item);
  a.out_vec = d_head % 4 == 0 && aligned_to(out, 4 * item);
  const uint64_t tiles = (uint64_t)n_requests * n_kv_heads * c.q_tiles;
  const uint64_t reductions = tiles * ((c.cols + reduce_cols(c.cols) - 1) / reduce_cols(c.cols));
  if (reductions >= (1ull << 31))
    return record_error(DFATTN_ERR_OVERFLOW, std::string(fn) + ": shape is too large");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool e4m3 = kv_dtype == DFATTN_KV_E4M3, bf16 = act_dtype == DFATTN_KV_BF16;
  if (e4m3 && bf16)
    launch_shape<true, 1>(a, c.qt, s);
  else if (e4m3)
    launch_shape<true, 2>(a, c.qt, s);
  else if (bf16)
    launch_shape<false, 1>(a, c.qt, s);
  else
    launch_shape<false, 2>(a, c.qt, s);
  st = launched(fn);
  if (st != DFATTN_OK || c.parts == 0) return st;
  if (d_head <= 64)
    hipLaunchKernelGGL(attention_reduce_kernel<1>, linear_grid(reductions), dim3(64 * kReduceWaves), 0, s, a,
                       (int)(16 * c.qt), bf16);
  else
    hipLaunchKernelGGL(attention_reduce_kernel<2>, linear_grid(reductions), dim3(64 * kReduceWaves), 0, s, a,
                       (int)(16 * c.qt), bf16);
  return launched(fn);
}

}  // extern "C"
