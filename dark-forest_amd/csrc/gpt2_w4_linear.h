// gpt2_w4_linear.h — the products of the 4-bit linear layers (gfx950), compiled
// once for each format.
#pragma once

#include "gpt2_device.h"
#include "gpt2_w4.h"

#include <algorithm>
#include <type_traits>

namespace dfattn {
namespace w4 {
namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// Eight codes as a matrix operand. int4: codes 0..15 are e4m3 numbers of 2^-9 (its subnormals
// go on into its first binade without a seam), four bytes at a time: inputs 0 2, 4 6, 1 3, 5 7. e2m1: in order.
template <bool E2M1>
__device__ __forceinline__ bf16x8 operand_of(unsigned c) {
  u32x4 r;
  if constexpr (E2M1) {
    r[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, 1.f, 0));
    r[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, 1.f, 1));
    r[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, 1.f, 2));
    r[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, 1.f, 3));
  } else {
    const unsigned lo = c & 0x0f0f0f0fu, hi = c >> 4 & 0x0f0f0f0fu;
    r[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.f, false));
    r[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.f, true));
    r[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.f, false));
    r[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.f, true));
  }
  return __builtin_bit_cast(bf16x8, r);
}

// Eight activations of a row as they lie in memory, and as matrix operands (fp32: three
// bf16 terms, whose sum is the value: 8 bits each of 24) in operand_of's order.
template <bool BF16>
struct Eight;
template <>
struct Eight<true> {
  u32x4 r;
  static constexpr int kTerms = 1;
  __device__ __forceinline__ void load(const char *p) { __builtin_memcpy(&r, p, 16); }
  __device__ __forceinline__ float value(int j) const { return __uint_as_float(j & 1 ? r[j / 2] & 0xffff0000u : r[j / 2] << 16); }
  __device__ __forceinline__ void load_some(const char *p, int n) {  // the first n
    unsigned x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = j < n ? reinterpret_cast<const unsigned short *>(p)[j] : 0u;
    r = {x[0] | x[1] << 16, x[2] | x[3] << 16, x[4] | x[5] << 16, x[6] | x[7] << 16};
  }
  template <bool E2M1>
  __device__ __forceinline__ void terms(bf16x8 (&t)[1]) const {
    u32x4 o = r;
    if constexpr (!E2M1)
      o = {__builtin_amdgcn_perm(r[1], r[0], 0x05040100u), __builtin_amdgcn_perm(r[3], r[2], 0x05040100u),
           __builtin_amdgcn_perm(r[1], r[0], 0x07060302u), __builtin_amdgcn_perm(r[3], r[2], 0x07060302u)};
    t[0] = __builtin_bit_cast(bf16x8, o);
  }
};
template <>
struct Eight<false> {
  float r[8];
  static constexpr int kTerms = 3;
  __device__ __forceinline__ void load(const char *p) { __builtin_memcpy(r, p, 32); }
  __device__ __forceinline__ float value(int j) const { return r[j]; }
  __device__ __forceinline__ void load_some(const char *p, int n) {
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = j < n ? reinterpret_cast<const float *>(p)[j] : 0.f;
  }
  template <bool E2M1>
  __device__ __forceinline__ void terms(bf16x8 (&t)[3]) const {
    constexpr int kOrder[2][8] = {{0, 2, 4, 6, 1, 3, 5, 7}, {0, 1, 2, 3, 4, 5, 6, 7}};
    u32x4 o[3];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float v[2] = {r[kOrder[E2M1][2 * i]], r[kOrder[E2M1][2 * i + 1]]};
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        o[k][i] = __builtin_amdgcn_perm(__float_as_uint(v[1]), __float_as_uint(v[0]), 0x07060302u);
        if (k < 2) {
#pragma unroll
          for (int e = 0; e < 2; ++e) v[e] -= __uint_as_float(__float_as_uint(v[e]) & 0xffff0000u);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) t[k] = __builtin_bit_cast(bf16x8, o[k]);
  }
};

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Workgroup b runs on XCD b mod 8: neighbouring blocks of outputs to one XCD, since they share
// the lines of scales and zeros.
__device__ __forceinline__ uint32_t xcd_block(uint32_t b, uint32_t n) {
  const uint32_t each = n / 8, more = n % 8, x = b % 8;  // (the first `more` XCDs have one more)
  return x * each + min(x, more) + b / 8;
}

// out = x W^T: v_mfma_f32_16x16x32_bf16 with 16 rows of x as A and 16 outputs as B, so that a lane's
// results are of one output, its scale one number, and 16 lanes store 64 bytes. A wave takes T x 16
// outputs and a part of the inputs, 128 at a time: 16 bytes of codes a lane and output (four
// lanes have a row's 64 bytes). In groups of 128 inputs those are its part of four products as they lie; in smaller ones two
// rounds of swaps between the quarters of the wave make four operands of 32 consecutive inputs, so that a product stays
// within a group. Each group's sum is scaled once, in fp32: out += s (sum q x - zero sum x), sum x by a product with ones.
// The waves' sums meet in LDS in the order of the inputs.
// Bound: with few weights latency (4 rows of 768 x 2304 in fp32 4.7 us, in bf16 4.0); with many what each wave has in flight (4 rows of
// 4096 x 16384 in bf16 13.7 us, 2.5 TB/s of codes: the vector unit is busy 29 % of the time, the matrix pipe 7 %, and the
// waves wait for half of theirs). The activations straight from L2: through LDS was no faster.
template <Format F, bool BF16, int GROUP, int T>
__global__ __launch_bounds__(512) void stream_kernel(LinearArgs a) {
  constexpr bool E2M1 = F == kE2M1;
  constexpr int kGroups = 128 / GROUP, kSteps = GROUP / 32;  // groups a tile of 128 inputs, products a group
  constexpr int kTerms = Eight<BF16>::kTerms, kItem = BF16 ? 2 : 4;
  constexpr int kStep = GROUP == 128 ? 8 : 32, kQuarter = GROUP == 128 ? 32 : 8;  // inputs from a product's to the next one's, a quarter's
  extern __shared__ f32x4 lds[];
  const uint32_t lane = threadIdx.x & 63, col = lane & 15, quarter = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // (the same in all lanes: scalar branches)
  const uint32_t kw = wave % a.k_waves, nw = wave / a.k_waves, n_waves = (blockDim.x >> 6) / a.k_waves;
  const uint32_t n0 = (xcd_block(blockIdx.x, gridDim.x) * n_waves + nw) * (16 * T), m0 = blockIdx.y * 16;
  const uint32_t tiles = (a.K + 127) / 128, t0 = tiles * kw / a.k_waves, t1 = tiles * (kw + 1) / a.k_waves;
  const unsigned char *codes[T];
  uint32_t n[T];
#pragma unroll
  for (int t = 0; t < T; ++t) {
    n[t] = min(n0 + 16 * t + col, a.N - 1);
    codes[t] = a.codes + (size_t)n[t] * a.row_bytes + 16 * quarter;
  }

  struct Codes {
    u32x4 c[T];
  };
  auto load_codes = [&](uint32_t tile, Codes &d) {
    if (tile * 64 + 64 <= a.row_bytes) {
#pragma unroll
      for (int t = 0; t < T; ++t) d.c[t] = *reinterpret_cast<const u32x4 *>(codes[t] + tile * 64);
    } else {
#pragma unroll
      for (int t = 0; t < T; ++t) {
        d.c[t] = u32x4{};
        if (tile * 64 + 16 * quarter < a.row_bytes) d.c[t] = *reinterpret_cast<const u32x4 *>(codes[t] + tile * 64);
      }
    }
  };
  // Scales (and zeros) of the four groups from `first` on, one a quarter; 0 behind the inputs.
  struct Scales {
    unsigned scale[T], zero[F == kU4 ? T : 1];
  };
  auto load_scales = [&](uint32_t first, Scales &d) {
    const uint32_t g = first + quarter;
    const size_t at = (size_t)min(g, a.groups - 1) * a.N;
#pragma unroll
    for (int t = 0; t < T; ++t) {
      d.scale[t] = a.scales[at + n[t]];
      if constexpr (F == kU4) d.zero[t] = a.zeros[at + n[t]];
    }
  };
  const bool live = m0 + col < a.M;
  const char *x = static_cast<const char *>(a.x) + (size_t)m0 * a.stride * kItem;
  struct Inputs {
    Eight<BF16> x[4];
  };
  // (Rows past the last one load nothing: a lane's row reaches results of that row only.)
  auto load_x = [&](uint32_t tile, Inputs &d) {
    const uint32_t k = tile * 128 + kQuarter * quarter;
    const char *at = x + ((size_t)(live ? col : 0) * a.stride + k) * kItem;
    if (tile * 128 + 128 <= a.K) {
      if (live) {
#pragma unroll
        for (int s = 0; s < 4; ++s) d.x[s].load(at + s * (kStep * kItem));
      }
    } else {
#pragma unroll
      for (int s = 0; s < 4; ++s) d.x[s].load_some(at + s * (kStep * kItem), live ? (int)a.K - (int)k - s * kStep : 0);
    }
  };

  f32x4 sum[T];
#pragma unroll
  for (int t = 0; t < T; ++t) sum[t] = f32x4{};
  const bf16x8 ones = __builtin_bit_cast(bf16x8, u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u});
  auto swap32 = [](unsigned &x, unsigned &y) {
    const auto r = __builtin_amdgcn_permlane32_swap(x, y, false, false);
    x = r[0];
    y = r[1];
  };
  auto swap16 = [](unsigned &x, unsigned &y) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, y, false, false);
    x = r[0];
    y = r[1];
  };
  // Each quarter's value in all lanes.
  auto spread = [&](unsigned v, unsigned (&to)[4]) {
    unsigned low = v, high = v;
    swap32(low, high);  // quarters 0 1 0 1, 2 3 2 3
    unsigned low2 = low, high2 = high;
    swap16(low, low2);
    swap16(high, high2);
    to[0] = low, to[1] = low2, to[2] = high, to[3] = high2;
  };
  // One tile; the scales of its groups are values `at` .. of four.
  auto use = [&](const Codes &d, const Inputs &in, const unsigned (&scale)[T][4], const unsigned (&zero)[T][4],
                 int at) {
    bf16x8 term[4][kTerms];
#pragma unroll
    for (int s = 0; s < 4; ++s) in.x[s].template terms<E2M1>(term[s]);
    f32x4 xs[kGroups];
    if constexpr (!E2M1) {
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        xs[g] = f32x4{};
#pragma unroll
        for (int s = g * kSteps; s < (g + 1) * kSteps; ++s)
#pragma unroll
          for (int k = 0; k < kTerms; ++k) xs[g] = mfma16(term[s][k], ones, xs[g]);
      }
    }
#pragma unroll
    for (int t = 0; t < T; ++t) {
      unsigned v0 = d.c[t][0], v1 = d.c[t][1], v2 = d.c[t][2], v3 = d.c[t][3];
      if constexpr (GROUP != 128) {
        swap32(v0, v2);
        swap32(v1, v3);
        swap16(v0, v1);
        swap16(v2, v3);
      }
      const unsigned v[4] = {v0, v1, v2, v3};
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        f32x4 acc = {};
#pragma unroll
        for (int s = g * kSteps; s < (g + 1) * kSteps; ++s) {
          const bf16x8 w = operand_of<E2M1>(v[s]);
#pragma unroll
          for (int k = 0; k < kTerms; ++k) acc = mfma16(term[s][k], w, acc);
        }
        const float f = __uint_as_float(scale[t][at + g] << 16), z = F == kU4 ? (float)zero[t][at + g] : 8.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[t][e] = fmaf(f, E2M1 ? acc[e] : fmaf(-z, xs[g][e], acc[e]), sum[t][e]);
      }
    }
  };

  // Four tiles a round. Codes come kAhead tiles ahead, scales a round, activations (from L2) one tile.
  constexpr int kAhead = T == 4 ? 1 : 3;
  Codes d[kAhead + 1];
  Scales sc[2][kGroups];
  Inputs in[2];
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (t0 + i < t1) load_codes(t0 + i, d[i]);
#pragma unroll
  for (int j = 0; j < kGroups; ++j) load_scales(t0 * kGroups + 4 * j, sc[0][j]);
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int s = 0; s < 4; ++s) in[i].x[s].load_some(nullptr, 0);
  if (t0 < t1) load_x(t0, in[0]);
  auto round = [&](uint32_t tile, Scales (&now)[kGroups], Scales (&next)[kGroups]) {
#pragma unroll
    for (int j = 0; j < kGroups; ++j) load_scales((tile + 4) * kGroups + 4 * j, next[j]);
    unsigned scale[T][4], zero[T][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // (Loads come back in order: the activations, which are waited for next, first.)
      if (tile + i + 1 < t1) load_x(tile + i + 1, in[(i + 1) % 2]);
      if (tile + i + kAhead < t1) load_codes(tile + i + kAhead, d[(i + kAhead) % (kAhead + 1)]);
      if (i * kGroups % 4 == 0) {
        const int j = i * kGroups / 4;
        const bool real = tile * kGroups + 4 * j + quarter < a.groups;  // (behind the inputs the sums are 0)
#pragma unroll
        for (int t = 0; t < T; ++t) {
          spread(real ? now[j].scale[t] : 0u, scale[t]);
          if constexpr (F == kU4) spread(now[j].zero[t], zero[t]);
        }
      }
      if (tile + i < t1) use(d[i % (kAhead + 1)], in[i % 2], scale, zero, i * kGroups % 4);
    }
  };
  for (uint32_t tile = t0; tile < t1; tile += 8) {
    round(tile, sc[0], sc[1]);
    if (tile + 4 < t1) round(tile + 4, sc[1], sc[0]);
  }

  // 16 rows of 16 outputs: a lane has output `col` of rows 4 quarter ...
  auto finish = [&](int t, f32x4 y) {
    const uint32_t at = n0 + 16 * t + col;
    if (at >= a.N) return;
    const float bias = a.bias != nullptr ? a.bias[at] : 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t m = m0 + 4 * quarter + e;
      if (m >= a.M) continue;
      float v = y[e] + bias;
      if (a.gelu) v = gelu_f(v);
      const size_t o = (size_t)m * a.N + at;
      if (a.residual != nullptr) v += load_value<BF16>(a.residual, o);
      store_value<BF16>(a.out, o, v);
    }
  };
  if (a.k_waves == 1) {
#pragma unroll
    for (int t = 0; t < T; ++t) finish(t, sum[t]);
    return;
  }
  f32x4 *mine = lds + (size_t)nw * a.k_waves * (T * 64);
#pragma unroll
  for (int t = 0; t < T; ++t) mine[(kw * T + t) * 64 + lane] = sum[t];
  __syncthreads();
  for (uint32_t i = kw; i < T; i += a.k_waves) {
    f32x4 y = mine[i * 64 + lane];
    for (uint32_t w = 1; w < a.k_waves; ++w) y += mine[(w * T + i) * 64 + lane];
    finish((int)i, y);
  }
}

// One or two rows: a matrix-vector product on the vector unit. L lanes (16, 32 or 64) share out up to 32 L inputs of a
// row, 32 of them each, which stay in registers as fp32 while the codes of kLoads outputs stream by (16 bytes a lane, whole
// rows of codes together); the products are fp32 multiply-adds of exact code values. A lane's 32 inputs are in one
// group: its sum is scaled once. At the end kLoads sums of L lanes are added by swaps that halve
// their number with the lanes', then along 16 lanes.
// Bound: with few weights latency (one row of 768 x 2304 3.3 us in fp32, a launch that does nothing 1.6); with many
// memory and the vector unit in turn, since all waves run in step: one multiply-add a code and row besides the conversions, 50 % of
// the time (4096 x 16384 in bf16 10.5 us, 3.3 TB/s, stream_kernel 13; 8192 x 28672 28 us, 4.3). More codes in flight, or waves that stay for more outputs, no faster.
__device__ __forceinline__ float row_sum(float v) {  // of 16 neighbouring lanes, in all of them
  v += dpp<0x128>(v);
  v += dpp<0x124>(v);
  v += dpp<0x122>(v);
  return v + dpp<0x121>(v);
}
template <Format F>
__device__ __forceinline__ void values_of(unsigned c, float (&v)[8]) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  if constexpr (F == kE2M1) {
    const f32x2 r[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 1),
                        __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 3)};
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = r[j / 2][j % 2];
  } else {  // (0..15 as e4m3 numbers of 2^-9, as in operand_of)
    const unsigned lo = c & 0x0f0f0f0fu, hi = c >> 4 & 0x0f0f0f0fu;
    const f32x2 r[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp8(lo, 512.f, false), __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(lo, 512.f, true),
                        __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi, 512.f, false), __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi, 512.f, true)};
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = r[(j & 1) * 2 + j / 4][j / 2 % 2];
  }
}

template <Format F, bool BF16, int ROWS, int L, int RB>
__global__ __launch_bounds__(512) void vector_kernel(LinearArgs a) {
  constexpr int kSub = 64 / L, kLoads = RB / kSub, kItem = BF16 ? 2 : 4;
  __shared__ float sums[8][ROWS][RB];
  const uint32_t lane = threadIdx.x & 63, sub = lane / L;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t kw = wave % a.k_waves, nw = wave / a.k_waves, n_waves = (blockDim.x >> 6) / a.k_waves;
  const uint32_t n0 = (xcd_block(blockIdx.x, gridDim.x) * n_waves + nw) * RB, n = n0 + sub * kLoads;  // the lane's outputs: from n on
  const uint32_t units = (a.K + 31) / 32, chunks = (units + a.units - 1) / a.units;
  const bool inside = n0 + RB <= a.N;
  float acc[kLoads][ROWS] = {};
  for (uint32_t chunk = kw; chunk < chunks; chunk += a.k_waves) {
    const uint32_t unit = chunk * a.units + lane % L;
    const bool mine = lane % L < a.units && unit < units;
    u32x4 c[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      c[i] = u32x4{};
      if (mine) c[i] = *reinterpret_cast<const u32x4 *>(a.codes + (size_t)min(n + i, a.N - 1) * a.row_bytes + unit * 16);
    }
    float x[ROWS][32], xs[ROWS];
#pragma unroll
    for (int m = 0; m < ROWS; ++m) {
      const char *at = static_cast<const char *>(a.x) + ((size_t)m * a.stride + unit * 32) * kItem;
      if (!mine) {  // (apart from a row's end, whose single loads the wave would else take for these lanes)
#pragma unroll
        for (int j = 0; j < 32; ++j) x[m][j] = 0.f;
      } else if (unit * 32 + 32 <= a.K) {
        if constexpr (BF16) {
          unsigned r[16];
          __builtin_memcpy(r, at, 64);
#pragma unroll
          for (int j = 0; j < 32; ++j) x[m][j] = __uint_as_float(j & 1 ? r[j / 2] & 0xffff0000u : r[j / 2] << 16);
        } else {
          __builtin_memcpy(x[m], at, 128);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const char *from = at + 8 * e * kItem;
          const uint32_t k = unit * 32 + 8 * e;
          if (k + 8 <= a.K) {
            Eight<BF16> v;
            v.load(from);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[m][8 * e + j] = v.value(j);
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[m][8 * e + j] = 0.f;
            if (k < a.K) {
#pragma unroll
              for (int j = 0; j < 7; ++j)
                if (k + j < a.K) x[m][8 * e + j] = load_value<BF16>(from, j);
            }
          }
        }
      }
    }
    unsigned short scale[kLoads];
    unsigned char zero[kLoads];
    const size_t g = mine ? (size_t)(unit * 32 >> a.log_group) * a.N : 0;
    if (inside) {
      __builtin_memcpy(scale, a.scales + g + n, 2 * kLoads);
      if constexpr (F == kU4) __builtin_memcpy(zero, a.zeros + g + n, kLoads);
    } else {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        scale[i] = a.scales[g + min(n + i, a.N - 1)];
        if constexpr (F == kU4) zero[i] = a.zeros[g + min(n + i, a.N - 1)];
      }
    }
#pragma unroll
    for (int m = 0; m < ROWS; ++m) {
      xs[m] = 0.f;
      if (F != kE2M1) {
#pragma unroll
        for (int j = 0; j < 32; j += 4) xs[m] += (x[m][j] + x[m][j + 1]) + (x[m][j + 2] + x[m][j + 3]);
      }
    }
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      float part[ROWS][2] = {};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        float v[8];
        values_of<F>(c[i][w], v);
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int m = 0; m < ROWS; ++m) part[m][j & 1] = fmaf(v[j], x[m][8 * w + j], part[m][j & 1]);
      }
      const float s = mine ? bf16_value(scale[i]) : 0.f, z = F == kU4 ? (float)zero[i] : 8.f;
#pragma unroll
      for (int m = 0; m < ROWS; ++m) {
        const float p = part[m][0] + part[m][1];
        acc[i][m] = fmaf(s, F == kE2M1 ? p : fmaf(-z, xs[m], p), acc[i][m]);
      }
    }
  }
  // Sums over the lanes; a lane's output is then j + where().
  constexpr int kLeft = L == 64 ? (kLoads + 3) / 4 : L == 32 ? (kLoads + 1) / 2 : kLoads;
  const uint32_t q = lane >> 4;
  const uint32_t where = L == 64 ? (q & 1) * (kLoads / 4) + (q >> 1) * (kLoads / 2) : L == 32 ? sub * kLoads + (q & 1) * (kLoads / 2) : q * kLoads;
#pragma unroll
  for (int m = 0; m < ROWS; ++m) {
    float v[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) v[i] = acc[i][m];
    if constexpr (L == 64) {
#pragma unroll
      for (int i = 0; i < kLoads / 2; ++i) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]), __float_as_uint(v[i + kLoads / 2]), false, false);
        v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
      }
    }
    if constexpr (L >= 32) {
#pragma unroll
      for (int i = 0; i < kLeft; ++i) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[i]), __float_as_uint(v[i + kLeft]), false, false);
        v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
      }
    }
#pragma unroll
    for (int i = 0; i < kLeft; ++i) {
      v[i] = row_sum(v[i]);
      if ((lane & 15) == 0) sums[wave][m][where + i] = v[i];
    }
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < n_waves * ROWS * RB; i += blockDim.x) {
    const uint32_t w = i / (ROWS * RB), m = i / RB % ROWS, j = i % RB;
    const uint32_t at = (xcd_block(blockIdx.x, gridDim.x) * n_waves + w) * RB + j;
    if (at >= a.N) continue;
    float y = sums[w * a.k_waves][m][j];
    for (uint32_t k = 1; k < a.k_waves; ++k) y += sums[w * a.k_waves + k][m][j];
    if (a.bias != nullptr) y += a.bias[at];
    if (a.gelu) y = gelu_f(y);
    const size_t o = (size_t)m * a.N + at;
    if (a.residual != nullptr) y += load_value<BF16>(a.residual, o);
    store_value<BF16>(a.out, o, y);
  }
}

// More rows: a workgroup of four waves takes 32 rows and 128 outputs, a wave 32 of those. x goes through LDS, 128 inputs at a
// time in two buffers, as operands that are made once for the four waves: [term][product][16 rows][quarter][row], 16 bytes
// each, the row's place turned by the 8 inputs' number so that neither the writes (16 pieces of a row) nor the reads meet in
// banks. Codes come straight from memory, as above. A group's products are scaled once, sum += s (sum q x); what
// the zero points take off, sum over the groups of (sum x)(zero s), is a product itself: four groups at a time on the fp32
// matrix instruction, with the groups' sums of x by products with ones, 16 rows each by two of the waves.
// Where rows and outputs give too few workgroups, `splits` share out the inputs and leave fp32 sums, which join_kernel adds.
// Bound: the vector unit, which turns codes into operands once for every 32 rows, and the matrix pipe behind it (2000 rows of 4096 x
// 4096 in bf16, groups of 128: 108 us, 620 TFLOP/s; VALU busy 47 %, matrix pipe 28 % of the time, hardly at once; without any loads or conversions
// of codes the products alone take 70). More rows a wave, which would convert less often, need registers that the sums of a group and
// of the layer take already: 64 rows and 256 outputs were both slower. Operands of codes made once for four waves, in LDS, were not tried.
// With few rows of wide layers what is in flight: 16 rows of 768 x 50257, e2m1, are 393 workgroups of six steps for 256 CUs, a
// barrier in each and one tile of codes ahead (fp32 12 us, vector unit 26 %, matrix pipe 11 %; bf16 10.8, 25 % and 5 %; the waves
// wait for half of their time in both).
// With HALVES = 2 eight waves do, four for each half of the inputs, and the halves' sums meet in LDS.
template <Format F, bool BF16, int GROUP, int R, int HALVES>
__global__ __launch_bounds__(kThreads * HALVES, 2) void matrix_kernel(LinearArgs a) {  // (2: no sums in accumulation registers)
  constexpr bool E2M1 = F == kE2M1;
  constexpr int T = kMatrixOutputs / 64;
  constexpr int kGroups = 128 / GROUP, kSteps = GROUP / 32;
  constexpr int kTerms = Eight<BF16>::kTerms, kItem = BF16 ? 2 : 4;
  __shared__ f32x4 operands_of_half[HALVES][2][kTerms][4][R][64];
  __shared__ f32x4 x_sums_of_half[HALVES][2][4][R * 4];  // of four groups
  const uint32_t lane = threadIdx.x & 63, col = lane & 15, quarter = lane >> 4, thread = threadIdx.x % kThreads;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(thread >> 6), half = HALVES == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / kThreads);
  auto &operands = operands_of_half[half];
  auto &x_sums = x_sums_of_half[half];
  const uint32_t n0 = (xcd_block(blockIdx.x, gridDim.x) * 4 + wave) * (16 * T), m0 = blockIdx.y * (16 * R);
  const uint32_t tiles = (a.K + 127) / 128;
  const uint32_t parts = gridDim.z * HALVES, my_part = blockIdx.z * HALVES + half;
  const uint32_t t0 = (uint32_t)((uint64_t)tiles * my_part / parts), t1 = (uint32_t)((uint64_t)tiles * (my_part + 1) / parts);
  const uint32_t steps = HALVES == 1 ? t1 - t0 : (tiles + parts - 1) / parts;  // (the same for both halves: they meet at barriers)
  const uint32_t g1 = min(t1 * kGroups, a.groups);
  const unsigned char *codes[T];
  uint32_t n[T];
#pragma unroll
  for (int t = 0; t < T; ++t) {
    n[t] = min(n0 + 16 * t + col, a.N - 1);
    codes[t] = a.codes + (size_t)n[t] * a.row_bytes;
  }
  struct Codes {
    u32x4 c[T];
  };
  auto load_codes = [&](uint32_t tile, Codes &d) {
    const uint32_t mine = tile * 64 + 16 * quarter, at = mine < a.row_bytes ? mine : 0;  // (x is 0 behind the inputs; a row may be 16 bytes)
#pragma unroll
    for (int t = 0; t < T; ++t) d.c[t] = *reinterpret_cast<const u32x4 *>(codes[t] + at);
  };
  struct Scales {
    unsigned scale[T], zero[F == kU4 ? T : 1];  // of group first + quarter
  };
  auto load_scales = [&](uint32_t first, Scales &d) {
    const size_t at = (size_t)min(first + quarter, a.groups - 1) * a.N;
#pragma unroll
    for (int t = 0; t < T; ++t) {
      d.scale[t] = a.scales[at + n[t]];
      if constexpr (F == kU4) d.zero[t] = a.zeros[at + n[t]];
    }
  };
  // Staging: a thread has 8 inputs of R rows.
  const uint32_t octet = thread & 15, row = thread >> 4;
  const uint32_t step = GROUP == 128 ? octet & 3 : octet >> 2, part = GROUP == 128 ? octet >> 2 : octet & 3;
  struct Inputs {
    Eight<BF16> x[R];
  };
  auto load_x = [&](uint32_t tile, Inputs &in) {
    const uint32_t k = tile * 128 + octet * 8;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint32_t m = m0 + 16 * r + row;
      const char *at = static_cast<const char *>(a.x) + ((size_t)min(m, a.M - 1) * a.stride + k) * kItem;
      if (tile * 128 + 128 <= a.K)
        in.x[r].load(at);
      else
        in.x[r].load_some(at, (int)a.K - (int)k);
    }
  };
  auto stage = [&](int buffer, const Inputs &in) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      bf16x8 term[kTerms];
      in.x[r].template terms<E2M1>(term);
#pragma unroll
      for (int k = 0; k < kTerms; ++k) operands[buffer][k][step][r][part * 16 + (row ^ octet)] = __builtin_bit_cast(f32x4, term[k]);
    }
  };
  auto operand = [&](int buffer, int k, int s, uint32_t r) {
    const uint32_t o = GROUP == 128 ? quarter * 4 + s : s * 4 + quarter;
    return __builtin_bit_cast(bf16x8, operands[buffer][k][s][r][quarter * 16 + (col ^ o)]);
  };

  f32x4 sum[T][R];
#pragma unroll
  for (int t = 0; t < T; ++t)
#pragma unroll
    for (int r = 0; r < R; ++r) sum[t][r] = f32x4{};
  auto swap32 = [](unsigned &x, unsigned &y) {
    const auto r = __builtin_amdgcn_permlane32_swap(x, y, false, false);
    x = r[0];
    y = r[1];
  };
  auto swap16 = [](unsigned &x, unsigned &y) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, y, false, false);
    x = r[0];
    y = r[1];
  };
  unsigned scale[T][4];  // of the four groups at hand
  float taken[T] = {};   // - zero * scale of group `quarter` of the four before
  // The four groups from `first` on come next: their scales, from `d`.
  auto next_four = [&](uint32_t first, const Scales &d, float (&take)[T]) {
    const bool real = first + quarter < g1;  // (behind them x is 0, or another split's)
#pragma unroll
    for (int t = 0; t < T; ++t) {
      unsigned low = real ? d.scale[t] : 0u, high = low;
      take[t] = -bf16_value((unsigned short)low) * (F == kU4 ? (float)d.zero[t] : 8.f);
      swap32(low, high);  // quarters 0 1 0 1, 2 3 2 3
      unsigned low2 = low, high2 = high;
      swap16(low, low2);
      swap16(high, high2);
      scale[t][0] = low, scale[t][1] = low2, scale[t][2] = high, scale[t][3] = high2;
    }
  };
  // What the zero points of four groups take off.
  auto take_off = [&](uint32_t first, int fours) {
    if constexpr (!E2M1) {
      const bool real = first + quarter < g1;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float xs = reinterpret_cast<const float *>(x_sums[fours][quarter])[16 * r + col];
#pragma unroll
        for (int t = 0; t < T; ++t) sum[t][r] = __builtin_amdgcn_mfma_f32_16x16x4f32(real ? xs : 0.f, taken[t], sum[t][r], 0, 0, 0);
      }
    }
  };
  const bf16x8 ones = __builtin_bit_cast(bf16x8, u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u});
  // One tile; its groups are numbers `at` .. of the four.
  auto use = [&](int buffer, const Codes &d, int at, int fours) {
    if (!E2M1 && wave < (uint32_t)R) {
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        f32x4 xs = {};
#pragma unroll
        for (int s = g * kSteps; s < (g + 1) * kSteps; ++s)
#pragma unroll
          for (int k = 0; k < kTerms; ++k) xs = mfma16(operand(buffer, k, s, wave), ones, xs);
        if (col == 0) x_sums[fours][at + g][4 * wave + quarter] = xs;
      }
    }
    unsigned v[T][4];
#pragma unroll
    for (int t = 0; t < T; ++t) {
#pragma unroll
      for (int s = 0; s < 4; ++s) v[t][s] = d.c[t][s];
      if constexpr (GROUP != 128) {
        swap32(v[t][0], v[t][2]);
        swap32(v[t][1], v[t][3]);
        swap16(v[t][0], v[t][1]);
        swap16(v[t][2], v[t][3]);
      }
    }
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      if (kGroups > 1) __builtin_amdgcn_sched_barrier(0);  // (one group's sums at a time: else 256 registers do not do)
      f32x4 acc[T][R];
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int r = 0; r < R; ++r) acc[t][r] = f32x4{};
#pragma unroll
      for (int s = g * kSteps; s < (g + 1) * kSteps; ++s) {
        bf16x8 w[T];
#pragma unroll
        for (int t = 0; t < T; ++t) w[t] = operand_of<E2M1>(v[t][s]);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int k = 0; k < kTerms; ++k) {
            const bf16x8 in = operand(buffer, k, s, r);
#pragma unroll
            for (int t = 0; t < T; ++t) acc[t][r] = mfma16(in, w[t], acc[t][r]);
          }
      }
#pragma unroll
      for (int t = 0; t < T; ++t) {
        const float f = __uint_as_float(scale[t][at + g] << 16);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int e = 0; e < 4; ++e) sum[t][r][e] = fmaf(f, acc[t][r][e], sum[t][r][e]);
      }
    }
  };
  // Rounds of four tiles, which hold kGroups times four groups. Codes and activations come one tile ahead (two: 2000 rows of
  // 4096 x 4096 122 us for 113, as three workgroups a CU are left of four).
  Codes d[2];
  Inputs in;
  Scales sc;
  if (t0 < t1) {
    load_x(t0, in);
    load_codes(t0, d[0]);
    load_scales(t0 * kGroups, sc);
    stage(0, in);
  }
  __syncthreads();
  for (uint32_t first = 0; first < steps; first += 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (first + i >= steps) break;
      const uint32_t tile = t0 + first + i;
      if (HALVES == 1 || tile < t1) {
        const bool more = tile + 1 < t1;
        const uint32_t group = tile * kGroups;
        if (more) {
          load_x(tile + 1, in);  // (loads come back in order: what is waited for first, first)
          load_codes(tile + 1, d[(i + 1) % 2]);
        }
        // (The sums of x of the four groups before were written before the last barrier.)
        const int fours = kGroups == 1 ? (int)(first / 4 % 2) : i * kGroups / 4 % 2;
        if (i * kGroups % 4 == 0) {
          if (tile > t0) take_off(group - 4, fours ^ 1);
          next_four(group, sc, taken);
          load_scales(group + 4, sc);
        }
        use(i % 2, d[i % 2], i * kGroups % 4, fours);
        if (more) stage((i + 1) % 2, in);
      }
      __syncthreads();
    }
  }
  if (t0 < t1) {
    const uint32_t last = (t1 - t0 - 1) * kGroups / 4;  // the last four groups
    take_off(t0 * kGroups + 4 * last, (int)(last % 2));
  }
  // With two halves each ends every other 16 outputs.
  constexpr int kEnds = HALVES == 2 ? 1 : T;
  f32x4 end[kEnds][R];
  if constexpr (HALVES == 2) {
    static_assert(T == 2 && sizeof(operands) >= 4 * R * 64 * sizeof(f32x4), "a half's sums take its operands' place");
    f32x4 *mine = &operands_of_half[half][0][0][0][0][0], *other = &operands_of_half[half ^ 1][0][0][0][0][0];
    const bool second = half != 0;
    auto pick = [&](const f32x4 &x, const f32x4 &y) {  // (number by number: the arrays stay in registers)
      f32x4 z;
#pragma unroll
      for (int e = 0; e < 4; ++e) z[e] = second ? y[e] : x[e];
      return z;
    };
#pragma unroll
    for (int r = 0; r < R; ++r) mine[(wave * R + r) * 64 + lane] = pick(sum[1][r], sum[0][r]);
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) end[0][r] = pick(sum[0][r], sum[1][r]) + other[(wave * R + r) * 64 + lane];
  } else {
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int r = 0; r < R; ++r) end[t][r] = sum[t][r];
  }
#pragma unroll
  for (int t = 0; t < kEnds; ++t) {
    const uint32_t at = n0 + 16 * (HALVES == 2 ? half : t) + col;
    if (at >= a.N) continue;
    const float bias = a.bias != nullptr ? a.bias[at] : 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t m = m0 + 16 * r + 4 * quarter + e;
        if (m >= a.M) continue;
        const size_t o = (size_t)m * a.N + at;
        if (a.partial != nullptr) {
          a.partial[(size_t)blockIdx.z * a.M * a.N + o] = end[t][r][e];
          continue;
        }
        float y = end[t][r][e] + bias;
        if (a.gelu) y = gelu_f(y);
        if (a.residual != nullptr) y += load_value<BF16>(a.residual, o);
        store_value<BF16>(a.out, o, y);
      }
  }
}

// The splits' sums, and the layer's end (16.4 MB of sums of two splits, with GELU, 7.3 us; four outputs at a time no less).
template <bool BF16>
__global__ __launch_bounds__(kThreads) void join_kernel(LinearArgs a, uint32_t splits) {
  const size_t all = (size_t)a.M * a.N, step = (size_t)gridDim.x * kThreads;
  for (size_t o = (size_t)blockIdx.x * kThreads + threadIdx.x; o < all; o += step) {
    float y = a.partial[o];
    for (uint32_t z = 1; z < splits; ++z) y += a.partial[z * all + o];
    if (a.bias != nullptr) y += a.bias[o % a.N];
    if (a.gelu) y = gelu_f(y);
    if (a.residual != nullptr) y += load_value<BF16>(a.residual, o);
    store_value<BF16>(a.out, o, y);
  }
}

}  // namespace

template <Format F, bool BF16>
void launch_vector(const LinearArgs &args, hipStream_t stream) {
  LinearArgs a = args;
  const uint32_t units = (a.K + 31) / 32, chunks = (units + 63) / 64;
  const int L = units <= 16 ? 16 : units <= 32 ? 32 : 64;
  a.units = (units + chunks - 1) / chunks;
  // Short rows of many outputs: 16 a wave (50257 of 768 inputs 11 us, 4 a wave 14); else 4.
  const bool many = L < 64 && a.N >= 16384;
  const uint32_t blocks = (a.N + (many ? 15 : 3)) / (many ? 16 : 4);
  // Some 4096 waves, as far as the inputs go; workgroups of up to 8 waves where there are many.
  while (a.k_waves < std::min(chunks, 8u) && blocks * a.k_waves < 4096) ++a.k_waves;
  uint32_t n_waves = 1;
  while (a.k_waves * n_waves * 2 <= 8 && blocks / n_waves >= 1024) n_waves *= 2;
  auto go = [&](auto rows, auto l, auto r) {
    constexpr int kRb = decltype(r)::value;
    const uint32_t per = n_waves * kRb;
    hipLaunchKernelGGL((vector_kernel<F, BF16, decltype(rows)::value, decltype(l)::value, kRb>), dim3((a.N + per - 1) / per),
                       dim3(64 * a.k_waves * n_waves), 0, stream, a);
  };
  using std::integral_constant;
  auto with_rb = [&](auto rows, auto l) {
    if (many)
      go(rows, l, integral_constant<int, 16>{});
    else
      go(rows, l, integral_constant<int, 4>{});
  };
  auto with_l = [&](auto rows) {
    if (L == 16)
      with_rb(rows, integral_constant<int, 16>{});
    else if (L == 32)
      with_rb(rows, integral_constant<int, 32>{});
    else
      go(rows, integral_constant<int, 64>{}, integral_constant<int, 4>{});
  };
  if (a.M == 1)
    with_l(integral_constant<int, 1>{});
  else
    with_l(integral_constant<int, 2>{});
}

template <Format F, bool BF16, int GROUP>
void launch_stream(const LinearArgs &args, hipStream_t stream) {
  LinearArgs a = args;
  // A wave takes 64, 32 or 16 outputs, as long as there are many (and registers do); up to 8 of them share out the inputs.
  constexpr uint32_t kMost = BF16 && GROUP > 32 ? 4 : 2;
  const uint32_t n_tiles = (a.N + 15) / 16, tiles = (a.K + 127) / 128;
  uint32_t T = n_tiles >= 1024 ? kMost : n_tiles >= 512 && BF16 ? 2 : 1;
  // (of at least three tiles each where there are waves enough)
  const uint32_t row_blocks = (a.M + kStreamRows - 1) / kStreamRows, blocks = n_tiles / T * row_blocks;
  while (a.k_waves < 8 && a.k_waves * 2 <= tiles &&
         (blocks * a.k_waves < 512 || (blocks * a.k_waves < 2048 && a.k_waves * 6 <= tiles)))
    a.k_waves *= 2;
  uint32_t n_waves = 1;
  while (a.k_waves * n_waves < 4 && n_tiles / T / (2 * n_waves) >= 256) n_waves *= 2;
  const uint32_t outputs = 16 * T * n_waves, waves = a.k_waves * n_waves;
  auto go = [&](auto t) {
    hipLaunchKernelGGL((stream_kernel<F, BF16, GROUP, decltype(t)::value>), dim3((a.N + outputs - 1) / outputs, row_blocks),
                       dim3(64 * waves), a.k_waves == 1 ? 0 : waves * T * 1024, stream, a);
  };
  if (T == 1)
    go(std::integral_constant<int, 1>{});
  else if (T == 2)
    go(std::integral_constant<int, 2>{});
  else if constexpr (kMost == 4)
    go(std::integral_constant<int, 4>{});
}

template <Format F, bool BF16, int GROUP>
void launch_matrix(const LinearArgs &args, float *workspace, hipStream_t stream) {
  LinearArgs a = args;
  uint32_t splits = workspace == nullptr ? 1 : splits_of(a.M, a.N, a.K);
  // bf16: two of the splits in one workgroup, which saves their sums' way through memory (500 rows of 4096 x 4096 36 us for 31),
  // where two such workgroups fit on every CU or each has few steps: with one a CU eight waves wait for each other at every
  // step (128 rows of 4096 x 4096, 8 steps, 18.7 us and 16.3; 256 rows, 16 steps and no join_kernel, 25.1 and 20.7, in
  // groups of 32 26.6 and 26.4; 128 rows of 16384 x 4096, 32 steps, 44 and 49).
  const size_t blocks = (size_t)((a.N + kMatrixOutputs - 1) / kMatrixOutputs) * ((a.M + kMatrixRows - 1) / kMatrixRows);
  const bool halves = BF16 && a.M > 16 && splits > 1 && (blocks * splits >= 1024 || (a.K + 127) / 128 <= (GROUP > 32 && splits == 2 ? 16 : 8) * splits);
  if (halves) splits /= 2;
  if (splits > 1) a.partial = workspace;
  const dim3 grid((a.N + kMatrixOutputs - 1) / kMatrixOutputs, (a.M + kMatrixRows - 1) / kMatrixRows, splits);
  if (a.M <= 16) {
    hipLaunchKernelGGL((matrix_kernel<F, BF16, GROUP, 1, 1>), grid, dim3(kThreads), 0, stream, a);
  } else if (halves) {
    if constexpr (BF16) hipLaunchKernelGGL((matrix_kernel<F, BF16, GROUP, kMatrixRows / 16, 2>), grid, dim3(2 * kThreads), 0, stream, a);
  } else {
    hipLaunchKernelGGL((matrix_kernel<F, BF16, GROUP, kMatrixRows / 16, 1>), grid, dim3(kThreads), 0, stream, a);
  }
  if (splits == 1) return;
  const size_t groups = ((size_t)a.M * a.N + kThreads - 1) / kThreads;
  hipLaunchKernelGGL((join_kernel<BF16>), dim3((uint32_t)std::min<size_t>(2048, groups)), dim3(kThreads), 0, stream, a, splits);
}

// The products in one format (a source file each).
template <Format F>
void launch_linear_format(const LinearArgs &a, bool bf16, uint32_t group, float *workspace, hipStream_t stream) {
  Path path = path_of(a.M, a.N, a.K, bf16);
  // (Without a workspace the inputs are not shared out.)
  if (path == kMatrix && a.M <= kStreamRows && workspace == nullptr && a.N < 32768 && splits_of(a.M, a.N, a.K) > 1)
    path = a.M <= kVectorRows ? kVector : kStream;
  auto with_group = [&](auto b, auto g) {
    constexpr bool B = decltype(b)::value;
    constexpr int G = decltype(g)::value;
    if (path == kMatrix)
      launch_matrix<F, B, G>(a, workspace, stream);
    else
      launch_stream<F, B, G>(a, stream);
  };
  auto with = [&](auto b) {
    if (path == kVector) return launch_vector<F, decltype(b)::value>(a, stream);
    if (group == 32)
      with_group(b, std::integral_constant<int, 32>{});
    else if (group == 64)
      with_group(b, std::integral_constant<int, 64>{});
    else
      with_group(b, std::integral_constant<int, 128>{});
  };
  if (bf16)
    with(std::true_type{});
  else
    with(std::false_type{});
}

}  // namespace w4
}  // namespace dfattn
