// Device helpers shared by the paged cache's kernels.
#pragma once

#include "kernels.h"
#include "paged_index.h"

namespace tars {

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));

// 16-bit element types: bits to fp32 (exact) and back (to nearest even).
struct Bf16 {
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
};
struct Fp16 {
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
};

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
