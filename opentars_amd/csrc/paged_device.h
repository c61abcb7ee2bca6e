// Device helpers shared by the paged cache's kernels.
#pragma once

#include "kernels.h"
#include "paged_index.h"

namespace tars {

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));

// 16-bit element types: bits to fp32 (exact) and back (to nearest even).
struct Bf16 {
  static constexpr uint32_t kExponent = 0x7F80;  // all ones: infinite or NaN
  static __device__ __forceinline__ float wide(uint32_t bits) { return __uint_as_float(bits << 16); }
  static __device__ __forceinline__ uint32_t pair(float lo, float hi) {
    const v2bf r = {static_cast<__bf16>(lo), static_cast<__bf16>(hi)};
    return __builtin_bit_cast(uint32_t, r);
  }
  // Two of the four e4m3 values in x (the low or the high half): exact.
  template <bool HIGH>
  static __device__ __forceinline__ uint32_t from_e4m3(uint32_t x) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, HIGH));
  }
  static __device__ __forceinline__ v4f mfma_16x16x32(uint4 a, uint4 b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ v4f mfma_16x16x16(uint2 a, uint2 b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(v4s, a), __builtin_bit_cast(v4s, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ v16f mfma_32x32x16(uint4 a, uint4 b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  }
};
struct Fp16 {
  static constexpr uint32_t kExponent = 0x7C00;
  static __device__ __forceinline__ float wide(uint32_t bits) {
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(bits)));
  }
  static __device__ __forceinline__ uint32_t pair(float lo, float hi) {
    const v2h r = {static_cast<_Float16>(lo), static_cast<_Float16>(hi)};
    return __builtin_bit_cast(uint32_t, r);
  }
  template <bool HIGH>
  static __device__ __forceinline__ uint32_t from_e4m3(uint32_t x) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, HIGH));
  }
  static __device__ __forceinline__ v4f mfma_16x16x32(uint4 a, uint4 b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ v4f mfma_16x16x16(uint2 a, uint2 b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(v4h, a), __builtin_bit_cast(v4h, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ v16f mfma_32x32x16(uint4 a, uint4 b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  }
};

// Four neighbouring values of an output row, rounded once: fp32 or T.
template <class T>
__device__ __forceinline__ void store4(char* row, int at, int f32, float a, float b, float c, float d) {
  if (f32) *reinterpret_cast<float4*>(row + 4 * at) = make_float4(a, b, c, d);
  else *reinterpret_cast<uint2*>(row + 2 * at) = make_uint2(T::pair(a, b), T::pair(c, d));
}

// The sequence that packed row `row` belongs to (seqs: none), the same in every lane: the number of sequences that
// end at or before it, 64 at a time.
__device__ __forceinline__ int seq_of_row(const KvSeqs& s, int row) {
  int n = 0;
  for (int b = 0; b < s.seqs; b += 64) {
    const int i = b + static_cast<int>(threadIdx.x & 63);
    const bool ended = i < s.seqs && iclamp(s.starts[i + 1], 0, s.rows) <= row;
    const int here = __popcll(__ballot(ended));
    n += here;
    if (here < 64) break;
  }
  return __builtin_amdgcn_readfirstlane(n);
}

}  // namespace tars
