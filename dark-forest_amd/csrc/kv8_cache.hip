// kv8_cache.hip — the paged 8-bit cache of a batch of requests: tables and slot
// maps from lengths, the quantising append and the read-back (gfx950).
#include "kv8.h"

#include <algorithm>
#include <type_traits>

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
// the workgroups share out the tokens and the fresh pages. 4 us for 64 tokens, 7.8 for
// 65536 of 500 requests (four tokens a thread, one after the other, 11): the latency of the
// lengths, then of a binary search in LDS and a page id.
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
  bool vec;  // rows of activations may be read, or written, four values at a time
};

// Four values of activations as they lie in memory, columns d .. of a head of one
// row: zero from D (left = D - d) on.
// VEC: all rows may be read four values at a time.
template <bool BF16, bool VEC>
struct Quad {
  std::conditional_t<BF16, uint2, float4> r;
  // From element `at` of src, which is the same in all lanes.
  __device__ __forceinline__ void load(const char *src, uint32_t at, int left) {
    const char *p = src + at * (BF16 ? 2u : 4u);
    if constexpr (VEC) {  // (left is 4 or more)
      r = *reinterpret_cast<const decltype(r) *>(p);
      return;
    }
    unsigned x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      x[j] = left <= j ? 0u : BF16 ? reinterpret_cast<const unsigned short *>(p)[j] : reinterpret_cast<const unsigned *>(p)[j];
    if constexpr (BF16)
      r = make_uint2(x[0] | x[1] << 16, x[2] | x[3] << 16);
    else
      r = make_float4(__uint_as_float(x[0]), __uint_as_float(x[1]), __uint_as_float(x[2]), __uint_as_float(x[3]));
  }
  __device__ __forceinline__ void clear() { r = {}; }
  __device__ __forceinline__ float4 value() const {
    if constexpr (BF16)
      return make_float4(__uint_as_float(r.x << 16), __uint_as_float(r.x & 0xffff0000u), __uint_as_float(r.y << 16),
                         __uint_as_float(r.y & 0xffff0000u));
    else
      return r;
  }
};

// Lanes 4 i + j, j = 0..3, hold four bytes each: byte k of lane j moves to byte j of
// lane k.
__device__ __forceinline__ unsigned transpose4(unsigned x, int lane) {
  const unsigned x0 = __builtin_amdgcn_mov_dpp(x, 0x00, 0xf, 0xf, false), x1 = __builtin_amdgcn_mov_dpp(x, 0x55, 0xf, 0xf, false);
  const unsigned x2 = __builtin_amdgcn_mov_dpp(x, 0xaa, 0xf, 0xf, false), x3 = __builtin_amdgcn_mov_dpp(x, 0xff, 0xf, 0xf, false);
  const unsigned pick = 0x0400u + 0x0101u * (lane & 3);  // this lane's byte of the first and of the second
  const unsigned lo = __builtin_amdgcn_perm(x1, x0, pick), hi = __builtin_amdgcn_perm(x3, x2, pick);
  return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}

constexpr int kAppendWaves = 4, kWindow = 48;
constexpr uint32_t kAppendGroups = 1024, kFewTokens = 1024;

// One side (K or V) of one page and head: its scale, and its codes.
template <bool E4M3>
struct Side {
  unsigned char *codes;
  float s, inv, ratio;
  bool dead;
  // From the bits of the new rows' largest magnitude (an infinity or a NaN is above all
  // numbers) and the scale of the rows that are kept (0: none). With such a row, or after
  // one, the scale is NaN, and with it every value; the codes are 0 (a NaN among them would
  // reach attention's rows that do not see the page: their probability there is 0, and 0 * NaN is NaN).
  __device__ __forceinline__ void scale(unsigned top, float old) {
    s = fmaxf(old, pow2_scale<E4M3>(__uint_as_float(top)));
    dead = top >= 0x7f800000u || old != old;
    if (dead) s = __builtin_nanf("");
    inv = dead ? 0.f : 1.f / s;
    ratio = dead ? 0.f : old * inv;
  }
  __device__ __forceinline__ unsigned encode(float4 v) const {
    return dead ? 0u : encode4<E4M3>(make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
  }
  // The rows before `off`, to the new scale, by `lanes` lanes of which this is `lane`: row
  // by row of K, column by column of V (whose last four bytes may hold newer rows).
  __device__ __forceinline__ void recode(bool is_v, int off, int P, int D, int lane, int lanes) const {
    const int Dp = padded(D), per_line = is_v ? (off + 3) >> 2 : Dp >> 2, lines = is_v ? D : off;
    for (int e = lane; e < per_line * lines; e += lanes) {
      const int line = e / per_line, q = e % per_line;
      unsigned *at = reinterpret_cast<unsigned *>(codes + line * (is_v ? P : Dp)) + q;
      const unsigned c = *at, keep = is_v && 4 * q + 4 > off ? ~0u << (8 * (off - 4 * q)) : 0u;
      const float4 v = decode4<E4M3>(c);
      const unsigned to = dead ? 0u : encode4<E4M3>(make_float4(v.x * ratio, v.y * ratio, v.z * ratio, v.w * ratio));
      *at = (to & ~keep) | (c & keep);
    }
  }
};

// The largest magnitude of values as they lie in memory: without their signs floats are in
// the order of their bits.
template <bool BF16>
struct Look {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  unsigned top = 0, pair = 0;  // (pair: two of bf16)
  template <bool VEC>
  __device__ __forceinline__ void at(const Quad<BF16, VEC> &q) {
    if constexpr (BF16) {
      auto more = [&](unsigned x) {
        pair = __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2, pair),
                                                                      __builtin_bit_cast(u16x2, x & 0x7fff7fffu)));
      };
      more(q.r.x);
      more(q.r.y);
    } else {
      auto more = [&](float x) { top = max(top, __float_as_uint(x) & 0x7fffffffu); };
      more(q.r.x);
      more(q.r.y);
      more(q.r.z);
      more(q.r.w);
    }
  }
  __device__ __forceinline__ unsigned bits() const { return BF16 ? max(pair << 16, pair & 0xffff0000u) : top; }
};

// The largest of a wave's bits.
__device__ __forceinline__ unsigned wave_top(unsigned x) {
  const float m = wave_max(__uint_as_float(min(x, 0x7f7fffffu)));
  return __any(x >= 0x7f800000u) ? 0x7f800000u : __float_as_uint(m);
}

// The append goes by runs, rows of one page whose slots follow each other (a row that stands behind
// another one of its page and does not follow it is left out). A workgroup finds those
// that start among kWindow tokens (their slots and the next ones are one load) and
// takes every `phases`-th of them. A run's rows are taken per kv head and side (K or
// V): the largest magnitude, the scale, the codes; rows already there are coded
// again where the scale grew.
// A run of one row (a generated token): 16 lanes to a head's row, or 32 (WIDE: more
// than 64 columns), four or two of them a wave.
// A longer one: a wave to a head and side (SPLIT, pages of 64 rows and more: all four
// share it), 16 rows of the page and 64 columns at a time: lane 4 i + j holds columns
// 4 i .. of rows j, 4 + j, 8 + j and 12 + j. V's codes are transposed within four
// lanes, so that each has 16 rows of one column, which lie together. The rows are read
// once to look and, but for the last 16, once more from the caches to write (two
// groups' loads on their way at a time need 130 to 250 registers: 8000 tokens 31 us for 22).
// Measured: 40 single rows (12 heads of 64, fp32) 5.6 us, a launch's latency; 8197
// tokens of four prompts (8 heads of 128, bf16) 26 us for 50 MB, where each wave waits
// for its slots, its rows and its stores one after the other; 8000 tokens (12 of 64, fp32)
// 18 us for 61 MB. (128 registers at most for 64 columns: 19 us for 22, 96 spill, 36 us; for
// 128 columns 128 spill, 38 us for 27.)
template <bool E4M3, bool BF16, bool WIDE, bool SPLIT, bool VEC>
__global__ __launch_bounds__(64 * kAppendWaves, WIDE ? 3 : 4) void append_kernel(CacheArgs a, uint32_t phases) {
  constexpr int kHalves = WIDE ? 2 : 1;
  __shared__ unsigned top_lds[kAppendWaves];
  const size_t i0 = (size_t)linear_block() * kWindow;
  if (i0 >= a.n) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane & 3, P = a.P, D = a.D, Dp = padded(D);
  const uint32_t n_slots = (uint32_t)a.n_pages * (uint32_t)P;
  const size_t row_bytes = a.stride * (BF16 ? 2 : 4);
  const uint32_t phase = blockIdx.z % phases, z = blockIdx.z / phases, nz = gridDim.z / phases;
  // Lane l holds the slot of token i0 - 1 + l.
  const size_t token = i0 + lane;  // (one more than the lane's)
  const uint32_t slots = token > 0 && token <= a.n ? a.slots[token - 1] : DFATTN_NO_SLOT;
  const uint32_t slot_page = slots / (uint32_t)P, before = __shfl_up(slots, 1, 64), page_before = __shfl_up(slot_page, 1, 64);
  const bool valid = lane > 0 && slots < n_slots, same = valid && slot_page == page_before;
  const unsigned long long links = __ballot(same && slots == before + 1);
  // A row of the page of the one before it never starts a run: two runs of one page would race.
  unsigned long long starts = __ballot(valid && !same && lane <= kWindow);
  for (uint32_t nth = 0; starts; starts &= starts - 1, ++nth) {
    if (nth % phases != phase) continue;
    const int first = __builtin_ctzll(starts);
    const size_t i = i0 + first - 1;
    const uint32_t slot = __builtin_amdgcn_readlane(slots, first);
    const size_t page = slot / (uint32_t)P;
    const int off = (int)(slot % (uint32_t)P);
    const unsigned long long rest = ~(links >> first >> 1);
    int len = 1 + (rest ? __builtin_ctzll(rest) : 64);  // rows of the run
    if (first + len >= 64) {  // (zeros were shifted in: the run may go on behind the lanes)
      len = 64 - first;
      while (true) {
        const size_t t = i + len + lane;
        const unsigned long long gone =
            ~__ballot(len + lane < P - off && t < a.n && a.slots[t] == slot + (uint32_t)(len + lane));
        len += gone ? __builtin_ctzll(gone) : 64;
        if (gone) break;
      }
    }

    if (len == 1) {
      constexpr int kLanes = 16 * kHalves;
      const int task = (int)(z * kAppendWaves + wave) * (64 / kLanes) + lane / kLanes;
      for (int k = 0; k * (int)(nz * kAppendWaves) * (64 / kLanes) < 2 * a.H; ++k) {
        const int t = task + k * (int)(nz * kAppendWaves) * (64 / kLanes), head_no = t >> 1, d = 4 * (lane % kLanes);
        const bool is_v = t & 1, on = t < 2 * a.H;
        const size_t head = page * a.H + (on ? head_no : 0);
        float *scale = (is_v ? a.v_scales : a.k_scales) + head;
        const float old = on && off > 0 ? *scale : 0.f;
        Quad<BF16, VEC> x;
        x.clear();
        if (on && d < D)
          x.load(static_cast<const char *>(is_v ? a.v : a.k) + i * row_bytes, (uint32_t)(head_no * D + d), D - d);
        Look<BF16> look;
        look.at(x);
        unsigned top = look.bits();
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) top = max(top, (unsigned)__shfl_xor((int)top, o, 64));
        Side<E4M3> side;
        side.codes = (is_v ? a.v_pool : a.k_pool) + head * (size_t)(P * Dp);
        side.scale(top, old);
        if (!on) continue;
        if (d == 0) *scale = side.s;
        if (off > 0 && side.ratio != 1.f) side.recode(is_v, off, P, D, lane % kLanes, kLanes);
        const unsigned c = side.encode(x.value());
        if (d >= Dp) continue;
        if (!is_v) {
          *reinterpret_cast<unsigned *>(side.codes + off * Dp + d) = c;
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r) side.codes[(d + r) * P + off] = (unsigned char)(c >> (8 * r));
        }
      }
      continue;
    }

    const int last = off + len - 1, m0 = (off >> 4) + (SPLIT ? wave : 0), m1 = last >> 4, step = SPLIT ? kAppendWaves : 1;
    const int n_tasks = 2 * a.H;
    for (int task = SPLIT ? (int)z : (int)(z * kAppendWaves) + wave; task < n_tasks;
         task += SPLIT ? (int)nz : (int)nz * kAppendWaves) {
      const int h = task >> 1;
      const bool is_v = task & 1;
      const char *src = static_cast<const char *>(is_v ? a.v : a.k) + i * row_bytes + (size_t)(h * D) * (BF16 ? 2 : 4);
      const size_t head = page * a.H + h;
      float *scale = (is_v ? a.v_scales : a.k_scales) + head;
      const float old = off > 0 ? *scale : 0.f;
      // Rows 16 m + 4 j + sub of the page; what is outside the run is zero.
      auto load = [&](int m, Quad<BF16, VEC> (&x)[4][kHalves]) {
        const uint32_t at = (uint32_t)(16 * m + sub - off) * (uint32_t)a.stride + 4 * (lane >> 2);
        if (16 * m >= off && 16 * m + 15 <= last) {
#pragma unroll
          for (int half = 0; half < kHalves; ++half) {
            const int d = 64 * half + 4 * (lane >> 2);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j][half].clear();
            if (d < D) {
#pragma unroll
              for (int j = 0; j < 4; ++j) x[j][half].load(src, at + 4 * j * (uint32_t)a.stride + 64 * half, D - d);
            }
          }
          return;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int top = 16 * m + 4 * j, row = top + sub;
          const bool any = top <= last && top + 3 >= off;
#pragma unroll
          for (int half = 0; half < kHalves; ++half) {
            const int d = 64 * half + 4 * (lane >> 2);
            x[j][half].clear();
            if (any && row >= off && row <= last && d < D) x[j][half].load(src, at + 4 * j * (uint32_t)a.stride + 64 * half, D - d);
          }
        }
      };
      Look<BF16> look;
      auto look_at = [&](const Quad<BF16, VEC> (&x)[4][kHalves]) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int half = 0; half < kHalves; ++half) look.at(x[j][half]);
      };
      Quad<BF16, VEC> x[4][kHalves];
      int m = m0 - step;
      while (m + step <= m1) {
        m += step;
        load(m, x);
        look_at(x);
      }
      unsigned top = wave_top(look.bits());
      if constexpr (SPLIT) {
        __syncthreads();  // (the task before has been read)
        if (lane == 0) top_lds[wave] = top;
        __syncthreads();
#pragma unroll
        for (int v = 0; v < kAppendWaves; ++v) top = max(top, top_lds[v]);
      }
      Side<E4M3> side;
      side.codes = (is_v ? a.v_pool : a.k_pool) + head * (size_t)(P * Dp);
      side.scale(top, old);
      const bool writes = !SPLIT || wave == 0;
      if (writes && lane == 0) *scale = side.s;
      // (V's bytes of the run's first rows may share four with kept ones: the wave that has the
      // run's first group codes them again, before it writes its own.)
      if (writes && off > 0 && side.ratio != 1.f) side.recode(is_v, off, P, D, lane, 64);
      auto put = [&](int m, const Quad<BF16, VEC> (&x)[4][kHalves]) {
        const bool whole = 16 * m >= off && 16 * m + 15 <= last;
#pragma unroll
        for (int half = 0; half < kHalves; ++half) {
          const int d = 64 * half + 4 * (lane >> 2), column = d + sub;
          if (!is_v) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int row = 16 * m + 4 * j + sub;
              const unsigned c = side.encode(x[j][half].value());
              if (row >= off && row <= last && d < Dp) *reinterpret_cast<unsigned *>(side.codes + row * Dp + d) = c;
            }
          } else {
            u32x4 t;
#pragma unroll
            for (int j = 0; j < 4; ++j) t[j] = transpose4(side.encode(x[j][half].value()), lane);
            if (column >= Dp) continue;
            unsigned char *at = side.codes + column * P + 16 * m;
            if (whole) {
              *reinterpret_cast<u32x4 *>(at) = t;
            } else {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int top = 16 * m + 4 * j;
                if (top > last || top + 3 < off) continue;
                if (top >= off && top + 3 <= last) {
                  *reinterpret_cast<unsigned *>(at + 4 * j) = t[j];
                } else {
#pragma unroll
                  for (int r = 0; r < 4; ++r)
                    if (top + r >= off && top + r <= last) at[4 * j + r] = (unsigned char)(t[j] >> (8 * r));
                }
              }
            }
          }
        }
      };
      while (m >= m0) {
        put(m, x);
        m -= step;
        if (m >= m0) load(m, x);
      }
    }
  }
}

// ---------------------------------------------------------------- read
// A wave takes four rows of the list and 64 columns of a head at a time, K and V together
// (8309 rows of 8 heads of 128 to fp32, 85 MB, 22 us, one after the other 23; to bf16, 51 MB, 19), lane 4 i + j columns
// 4 i .. of row j. V's codes of four consecutive rows of a page are read as the append
// writes them; other rows byte by byte.
constexpr int kReadWaves = 4;
constexpr uint32_t kReadGroups = 4096;
template <bool E4M3, bool BF16>
__global__ __launch_bounds__(64 * kReadWaves) void read_kernel(CacheArgs a) {
  const size_t i0 = ((size_t)linear_block() * kReadWaves + (threadIdx.x >> 6)) * 4;
  if (i0 >= a.n) return;
  const int lane = threadIdx.x & 63, sub = lane & 3, P = a.P, D = a.D, Dp = padded(D), shift = Dp > 64 ? 1 : 0;
  const size_t i = i0 + sub, dm = (size_t)a.H * D;
  const uint32_t slot = i < a.n ? a.slots[i] : DFATTN_NO_SLOT;
  const bool in = slot < (uint32_t)a.n_pages * (uint32_t)P;
  const size_t page = in ? slot / (uint32_t)P : 0;
  const int off = in ? (int)(slot % (uint32_t)P) : 0;
  const uint32_t slot0 = __builtin_amdgcn_mov_dpp(slot, 0x00, 0xf, 0xf, false);
  const bool together = __all(in && slot0 % 4 == 0 && slot == slot0 + sub);
  const int tasks = a.H << shift;
  auto put = [&](void *out, size_t at, int d, unsigned c, float s) {
    float4 v = decode4<E4M3>(c);
    v = in ? make_float4(v.x * s, v.y * s, v.z * s, v.w * s) : make_float4(0.f, 0.f, 0.f, 0.f);
    if (a.vec) {
      if constexpr (BF16)
        *reinterpret_cast<uint2 *>(static_cast<unsigned short *>(out) + at) =
            make_uint2(bf16_bits(v.x) | bf16_bits(v.y) << 16, bf16_bits(v.z) | bf16_bits(v.w) << 16);
      else
        *reinterpret_cast<float4 *>(static_cast<float *>(out) + at) = v;
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float y = (&v.x)[r];
        if (d + r >= D) break;
        if constexpr (BF16)
          static_cast<unsigned short *>(out)[at + r] = (unsigned short)bf16_bits(y);
        else
          static_cast<float *>(out)[at + r] = y;
      }
    }
  };
  for (int task = blockIdx.z; task < tasks; task += gridDim.z) {
    const int h = task >> shift, d = 64 * (task & shift) + 4 * (lane >> 2);
    if (!together && d >= D) continue;
    const size_t head = page * a.H + h, base = head * (size_t)(P * Dp);
    const unsigned k = d < Dp ? *reinterpret_cast<const unsigned *>(a.k_pool + base + off * Dp + d) : 0u;
    unsigned v = 0;
    if (together) {
      if (d + sub < Dp) v = *reinterpret_cast<const unsigned *>(a.v_pool + base + (d + sub) * P + (off & ~3));
      v = transpose4(v, lane);
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) v |= (unsigned)a.v_pool[base + (d + r) * P + off] << (8 * r);
    }
    if (i >= a.n || d >= D) continue;
    const float ks = a.k_scales[head], vs = a.v_scales[head];
    const size_t at = i * dm + (size_t)(h * D + d);
    put(a.k_out, at, d, k, ks);
    put(a.v_out, at, d, v, vs);
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
  // Every workgroup reads all lengths while others write: nothing may be written in place.
  const struct {
    const uint32_t *p;
    size_t n;
  } spans[] = {{block_table, (size_t)n_requests * max_pages}, {seq_lens, n_requests}, {query_start, n_requests + 1u},
               {slot_map, token_capacity}, {counts, 3}, {cached_lens, n_requests}, {new_lens, n_requests},
               {free_pages, n_free}, {free_start, 1}};
  for (int i = 0; i < 5; ++i)
    for (int j = i + 1; j < 9; ++j)
      if (spans[i].n > 0 && spans[j].n > 0 && spans[i].p < spans[j].p + spans[j].n && spans[j].p < spans[i].p + spans[i].n)
        return record_error(DFATTN_ERR_SHAPE, std::string(fn) + ": outputs must not overlap inputs or each other");
  PlanArgs a{cached_lens, new_lens, free_pages, free_start, block_table, seq_lens, query_start, slot_map, counts,
             n_free, n_requests, max_pages, token_capacity, page_size, n_pages};
  // A token a thread, up to two workgroups a CU.
  const uint32_t work = std::max(token_capacity, n_requests + 1);
  const uint32_t grid = std::min(512u, (work + kPlanThreads - 1) / kPlanThreads);
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
  if (n_tokens > (1u << 31) || row_stride > (1u << 21))
    return record_error(DFATTN_ERR_OVERFLOW, std::string(fn) + ": too many tokens, or a row_stride above 2^21");
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
  const size_t four = act_dtype == DFATTN_KV_F32 ? 16 : 8;
  a.vec = d_head % 4 == 0 && row_stride % 4 == 0 && aligned_to(k, four) && aligned_to(v, four);
  // About kAppendGroups workgroups: 250 to 300 a us start, empty or not (8000 of them for a
  // prompt of 8197 tokens took 30 us for that alone; 2048 took 19 us for 1000 single rows, 1024 take
  // 13.5). A window's runs are dealt to several while there are fewer.
  const bool wide = d_head > 64, split = page_size >= 64;
  const uint32_t windows = (n_tokens + kWindow - 1) / kWindow;
  // The heads' sides that a workgroup takes at once: few tokens are taken to be runs of one
  // row, which need fewer workgroups (256 rows of 12 heads: 10 us for 15); for many that
  // leaves waves without work where the runs are longer (8000 tokens: 25 us for 22).
  const uint32_t per_group = split ? 1 : n_tokens <= kFewTokens ? kAppendWaves * (wide ? 2 : 4) : kAppendWaves;
  const uint32_t tasks = std::min((2 * n_kv_heads + per_group - 1) / per_group, 1024u);
  const uint32_t phases = std::min<uint32_t>(kWindow, std::max<uint64_t>(1, kAppendGroups / ((uint64_t)windows * tasks)));
  dim3 grid = linear_grid(windows);
  grid.z = phases * tasks;
  by_types(act_dtype, kv_dtype, [&](auto e4m3, auto bf16) {
    constexpr bool E = decltype(e4m3)::value, B = decltype(bf16)::value;
    auto go = [&](auto wide_, auto split_, auto vec_) {
      hipLaunchKernelGGL((append_kernel<E, B, decltype(wide_)::value, decltype(split_)::value, decltype(vec_)::value>), grid,
                         dim3(64 * kAppendWaves), 0, static_cast<hipStream_t>(stream), a, phases);
    };
    auto go_vec = [&](auto wide_, auto split_) {
      if (a.vec)
        go(wide_, split_, std::true_type{});
      else
        go(wide_, split_, std::false_type{});
    };
    if (wide && split)
      go_vec(std::true_type{}, std::true_type{});
    else if (wide)
      go_vec(std::true_type{}, std::false_type{});
    else if (split)
      go_vec(std::false_type{}, std::true_type{});
    else
      go_vec(std::false_type{}, std::false_type{});
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
  const size_t four = act_dtype == DFATTN_KV_F32 ? 16 : 8;
  a.vec = d_head % 4 == 0 && aligned_to(k_out, four) && aligned_to(v_out, four);
  // Heads to workgroups of their own as long as there are few waves.
  const uint32_t groups = (n_rows + 4 * kReadWaves - 1) / (4 * kReadWaves), tasks = n_kv_heads * (d_head > 64 ? 2 : 1);
  dim3 grid = linear_grid(groups);
  grid.z = std::min(tasks, std::max(1u, kReadGroups / groups));
  by_types(act_dtype, kv_dtype, [&](auto e4m3, auto bf16) {
    hipLaunchKernelGGL((read_kernel<decltype(e4m3)::value, decltype(bf16)::value>), grid, dim3(64 * kReadWaves), 0,
                       static_cast<hipStream_t>(stream), a);
  });
  return launched(fn);
}

}  // extern "C"
