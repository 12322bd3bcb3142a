// gpt2_w4.h — what the 4-bit linear layers' kernels share: formats, types and
// the products' arguments.
//
// codes [outputs, row bytes], input 2 b in the low half of byte b; scales bf16
// and zeros (one byte) [groups, outputs].
#pragma once

#include "dfattn_internal.h"
#include "dfgpt2.h"

namespace dfattn {
namespace w4 {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;

enum Format { kI4 = DFGPT2_W4_I4, kU4 = DFGPT2_W4_U4, kE2M1 = DFGPT2_W4_E2M1 };

__device__ __forceinline__ float bf16_value(unsigned short b) { return __uint_as_float((unsigned)b << 16); }
// To the nearest, ties to even; a NaN stays one.
__device__ __forceinline__ unsigned short bf16_bits(float f) {
  const unsigned u = __float_as_uint(f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return (unsigned short)(u >> 16 | 0x40u);
  return (unsigned short)((u + 0x7fffu + (u >> 16 & 1u)) >> 16);
}
template <bool BF16>
__device__ __forceinline__ float load_value(const void *p, size_t i) {
  if constexpr (BF16)
    return bf16_value(static_cast<const unsigned short *>(p)[i]);
  else
    return static_cast<const float *>(p)[i];
}
template <bool BF16>
__device__ __forceinline__ void store_value(void *p, size_t i, float v) {
  if constexpr (BF16)
    static_cast<unsigned short *>(p)[i] = bf16_bits(v);
  else
    static_cast<float *>(p)[i] = v;
}

// v of the lane that a DPP control names.
template <int CONTROL>
__device__ __forceinline__ unsigned dpp(unsigned v) {
  return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CONTROL, 0xf, 0xf, false);
}
template <int CONTROL>
__device__ __forceinline__ float dpp(float v) {
  return __uint_as_float(dpp<CONTROL>(__float_as_uint(v)));
}

struct LinearArgs {
  const void *x;
  const unsigned char *codes;
  const unsigned short *scales;
  const unsigned char *zeros;
  const float *bias;
  const void *residual;
  void *out;
  float *partial;  // (matrix_kernel) [splits, M, N], or NULL
  size_t stride;
  uint32_t M, N, K, row_bytes, groups;
  uint32_t log_group;
  uint32_t k_waves;  // waves of a workgroup that share out the inputs of one block of outputs
  uint32_t units;    // (vector_kernel) 32 inputs each, of one wave
  int gelu;
};

// matrix_kernel's workgroups take kMatrixRows x kMatrixOutputs results, stream_kernel's kStreamRows rows.
constexpr uint32_t kVectorRows = 2, kStreamRows = 16, kMatrixRows = 32, kMatrixOutputs = 128;

// Which kernel takes M rows of N outputs and K inputs. One or two rows: vector_kernel (two of 4096 x 4096 in bf16 6.0 us,
// stream_kernel 7). More: stream_kernel, which reads all codes for every 16 rows but is one launch, up to a number of
// weights' uses, then matrix_kernel, with the inputs shared out. (us, stream_kernel and matrix_kernel:)
//   fp32: 64 rows of 768 x 2304 8.6 and 10.5, 128 13.1 and 12.4; 32 of 2048 x 2048 8.3 and 9.5, 48 12.5 and 9.7;
//   bf16: 192 rows of 768 x 2304 9.7 and 12.6; 64 of 2048 x 2048 8.3 and 8.7, 96 10.7 and 9.9;
//   1000 rows of 64 x 64 4.4 and 6.8, of 768 x 128 7.6 and 9.6.
// matrix_kernel also takes 2 to 16 rows of layers wide enough for its workgroups (16 rows of 768 x 50257 in fp32 21 and 13, in bf16
// 12.6 and 10.8; 2 rows, vector_kernel's 16 and 12, 14.7 and 10.6), of large ones (fp32: 4 rows of 4096 x 16384 19 to 22 and 18, 16
// rows 25 and 19, but of 4096 x 4096 10 and 11; bf16: 16 rows of 8192 x 28672 48 and 40, of 4096 x 16384 15 and 16) and in
// fp32 of many inputs for more than 8 rows (16 rows of 8192 x 1024 20 and 15, 8 rows 15 and 15).
// Wide is the same number of outputs whatever the inputs. At that border (2 to 16 rows of 32752 and of 32768 outputs, i4; the
// second is matrix_kernel) in fp32 64 inputs 5.0 to 7.5 and 4.5 to 5.3, 256 6.4 to 8.7 and 7.3 to 9.4, 768 9.5 to 13.1 and 10.5 to
// 12.7; in bf16 256 inputs 5.5 to 6.9 and 6.8 to 8.9, 768 8.6 to 9.9 and 9.1 to 11.2, 2048 14.3 to 15.9 and 14.8 to 16.2, 3968
// 25.2 to 28.5 and 23.3 to 24.5: with 256 to 768 inputs and bf16 the other kernels would still be up to a quarter faster there.
enum Path { kVector, kStream, kMatrix };
inline Path path_of(uint32_t M, uint32_t N, uint32_t K, bool bf16) {
  const uint64_t weights = (uint64_t)N * K;
  if (M == 1) return kVector;
  if (N >= 32768) return kMatrix;
  if (M > kStreamRows) return M <= 1024 && (M + 15) / 16 * weights <= (bf16 ? 22u << 20 : 10u << 20) ? kStream : kMatrix;
  if (bf16 ? M > kVectorRows && weights >= 1u << 27 : weights >= 1u << 25 || (M > 8 && K >= 8192)) return kMatrix;
  return M <= kVectorRows ? kVector : kStream;
}

// Splits of the inputs for matrix_kernel: up to 8, for no more than some 512 workgroups, or two where there are
// up to 512 and many inputs (4096 x 4096 in bf16: 500 rows 42 us whole, 40 in two, 48 in four; 64 rows 23 us whole, 15 in four
// and in eight). In fp32, where no two of the splits are one workgroup's, the sums' way through memory costs more than it
// brings from some 400 rows on (500 rows of 4096 x 4096 70 us in two and 68 whole, 400 of 768 x 2304 17 and 14).
inline uint32_t splits_of(uint32_t M, uint32_t N, uint32_t K) {
  const uint64_t groups = (uint64_t)((M + kMatrixRows - 1) / kMatrixRows) * ((N + kMatrixOutputs - 1) / kMatrixOutputs);
  const uint32_t tiles = (K + 127) / 128;
  uint32_t s = 1;
  while (s < 8 && groups * s * 2 <= 512 && s * 2 <= tiles) s *= 2;
  return s == 1 && groups <= 512 && tiles >= 16 ? 2 : s;
}

template <Format F>
void launch_linear_format(const LinearArgs &a, bool bf16, uint32_t group, float *workspace, hipStream_t stream);

}  // namespace w4
}  // namespace dfattn
