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
  static constexpr float kLargest = 0;           // as good as fp32's
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
  static constexpr float kLargest = 65504.0f;
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

__device__ __forceinline__ int inclusive_sum(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);  // row_shr 1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // row_bcast 15 to rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // row_bcast 31 to rows 2 and 3
  return x;
}

// Over the lanes of one row: l % R.
template <int R, class Op>
__device__ __forceinline__ float over_row(float x, Op op) {
  if constexpr (R == 16) {
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = op(__uint_as_float(s[0]), __uint_as_float(s[1]));
  }
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return op(__uint_as_float(s[0]), __uint_as_float(s[1]));
}

// What a difference of K / V head h's raw scores is multiplied by to be an exponent of 2: scale times log2(e), and K's scale.
// Within fp32's normal numbers: at 0 a hidden score, -inf, would be NaN, and at infinity the largest score's distance from
// itself. The scores are kept raw, and only their differences, 0 or less, multiplied: scale q k itself may pass fp32.
__device__ __forceinline__ float score_scale(const PagedAttnArgs& a, int h) {
  const float sc = a.scale * 1.44269504f * (a.pool.kscale ? a.pool.kscale[h] : 1.0f);
  return sc < 0x1p-126f ? 0x1p-126f : sc > 0x1.fffffep127f ? 0x1.fffffep127f : sc;
}

// Masks without comparisons, whose results would crowd the scalar registers.
template <class T>
__device__ __forceinline__ uint32_t not_finite(uint32_t x) {  // 0xFFFF in each half that is infinite or NaN
  const uint32_t e = T::kExponent << 16 | T::kExponent, rest = (x & e) ^ e;  // 0 where the exponent is all ones
  const uint32_t top = ~(rest + 0x7FFF7FFFu) & 0x80008000u;
  return (top << 1) - (top >> 15);
}
__device__ __forceinline__ uint32_t nan_e4m3(uint32_t x) {    // 0xFF in each byte that is an e4m3 NaN
  const uint32_t top = ((x & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
  return (top << 1) - (top >> 7);
}

// Four neighbouring values of an output row, rounded once: fp32 or T. mean: they are means of T's values, without a scale, by
// numerators rounded to T, whose rounding may take binary16's largest value to infinity: half a step is enough. (bf16's
// largest is fp32's but for the rounding; numerators in two parts are off by 2^-22.)
template <class T>
__device__ __forceinline__ float within(float x, bool mean) {
  if (!mean || T::kLargest == 0) return x;
  x = x > T::kLargest && x < INFINITY ? T::kLargest : x;
  return x < -T::kLargest && x > -INFINITY ? -T::kLargest : x;
}
template <class T>
__device__ __forceinline__ void store4(char* row, int at, int f32, float a, float b, float c, float d, bool mean = false) {
  if (f32) *reinterpret_cast<float4*>(row + 4 * at) = make_float4(a, b, c, d);
  else
    *reinterpret_cast<uint2*>(row + 2 * at) =
        make_uint2(T::pair(within<T>(a, mean), within<T>(b, mean)), T::pair(within<T>(c, mean), within<T>(d, mean)));
}

// The number of sequences, of `seqs`, that ended(b) holds for, which holds for the first ones: 64 of every 4096, 64 and 1
// at a time. Where it does not, any number up to seqs.
template <class F>
__device__ __forceinline__ int count_first(int seqs, F ended) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int step = seqs > 4096 ? 4096 : seqs > 64 ? 64 : 1; step; step >>= 6) {
    const int b = n + (lane + 1) * step - 1;
    n += step * __popcll(__ballot(b < seqs && ended(min(b, seqs - 1))));
  }
  return __builtin_amdgcn_readfirstlane(n);
}

// The sequence that packed row `row` belongs to (seqs: none), the same in every lane: the number of sequences that end at
// or before it.
__device__ __forceinline__ int seq_of_row(const KvSeqs& s, int row) {
  return count_first(s.seqs, [&](int b) { return iclamp(s.starts[b + 1], 0, s.rows) <= row; });
}

// Whether one of the accumulators is not finite (or their sum is not, of which nothing comes but a search): an infinity or
// NaN stays one in a sum.
template <class Acc, int N>
__device__ __forceinline__ bool not_all_finite(const Acc (&o)[N]) {
  float z[4] = {0, 0, 0, 0};  // four chains
#pragma unroll
  for (int t = 0; t < N; ++t)
#pragma unroll
    for (int e = 0; e < static_cast<int>(sizeof(Acc) / 4); ++e) z[e & 3] += o[t][e];
  const float sum = z[0] + z[1] + (z[2] + z[3]);
  return !(sum - sum == 0);
}

// Four columns y of a row joined from n parts, the parts' own v(p): an infinity of a part whose weight fp32 rounds to 0 made
// NaN there. A weight is positive: such a column is the sum of the parts' infinities and NaN, if they have any.
template <class F>
__device__ __forceinline__ void join_unfinite(float4& y, int n, F v) {
  if (y.x == y.x && y.y == y.y && y.z == y.z && y.w == y.w) return;
  const auto add = [](float z, float x) { return x - x == 0 ? z : z + x; };
  float4 z = make_float4(0, 0, 0, 0);
#pragma unroll 1
  for (int p = 0; p < n; ++p) {
    const float4 x = v(p);
    z = make_float4(add(z.x, x.x), add(z.y, x.y), add(z.z, x.z), add(z.w, x.w));
  }
  y = make_float4(z.x == 0 ? y.x : z.x, z.y == 0 ? y.y : z.y, z.z == 0 ? y.z : z.z, z.w == 0 ? y.w : z.w);
}

// A set of up to 128 columns.
struct Columns {
  uint64_t lo = 0, hi = 0;
  static __device__ __forceinline__ uint64_t below(int n) { return n <= 0 ? 0 : n >= 64 ? ~0ull : (1ull << n) - 1; }
  __device__ __forceinline__ void add(Range r) {
    lo |= below(r.hi) & ~below(r.lo);
    hi |= below(r.hi - 64) & ~below(r.lo - 64);
  }
  __device__ __forceinline__ bool has(int x) const { return (x < 64 ? lo >> x : hi >> (x - 64)) & 1; }
};

// Sets the outputs that V's infinities and NaN reach to the sum of those they see, at the positions of the steps `at(i)` of STEP
// positions, i in [t0, t1), of sequence b. What such a value made of an output in the products (nothing where it was left
// out, an infinity or NaN otherwise) does not count. The columns are [c0, c0 + cols), 128 at most, of K / V head h; column x
// is query head h * group + x % group of row first + x / group, at position p0 + x / group. sound(x): the column's sum of
// numerators is finite (an output of one whose is not stays NaN), or it is a row of a part; part(x): its row of a part in
// the workspace, or null where its output is final. A thread per column of V, 16 positions of a page at a time; all of the
// workgroup's outputs are written, and the barrier behind that passed.
template <class T, bool E4M3, int D, int STEP, class At, class F, class G>
__device__ void set_unfinite(const PagedAttnArgs& a, int b, int h, int len, At at, int t0, int t1, int p0, int first, int c0, int cols,
                             F part, G sound) {
  static_assert(STEP % 16 == 0, "16 positions of one page at a time");
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    Columns nan, plus, minus, all;
    all.add({0, cols});
#pragma unroll 1
    for (int i = t0 * (STEP / 16); i < t1 * (STEP / 16) && (nan.lo != all.lo || nan.hi != all.hi); ++i) {
      const int j0 = at(i / (STEP / 16)) * STEP + i % (STEP / 16) * 16;
      if (j0 >= len) break;
      const int page = a.seqs.table[b * a.seqs.ld_table + (j0 >> a.pool.page_shift)];
      if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(a.pool.pages)) continue;
      const char* block = a.pool.v + h * a.pool.v_head + page * a.pool.v_page + (j0 & ((1 << a.pool.page_shift) - 1)) * a.pool.v_slot;
      const auto value = [&](int k) {
        const char* row = block + k * a.pool.v_slot;
        return E4M3 ? T::template from_e4m3<false>(reinterpret_cast<const uint8_t*>(row)[d]) & 0xFFFFu
                    : static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(row)[d]);
      };
      uint32_t bad = 0;
#pragma unroll
      for (int k = 0; k < 16; ++k) bad |= static_cast<uint32_t>(not_finite<T>(value(k)) != 0) << k;
#pragma unroll 1
      for (; bad; bad &= bad - 1) {
        const int k = __builtin_ctz(bad), j = j0 + k;
        if (j >= len) break;
        const float v = T::wide(value(k));
        const Range seen = seen_by(j, p0, a.group, c0, cols, a.window, a.sinks);
        if (v != v) nan.add(seen);
        else if (v > 0) plus.add(seen);
        else minus.add(seen);
      }
    }
    if ((nan.lo | nan.hi | plus.lo | plus.hi | minus.lo | minus.hi) == 0) continue;
#pragma unroll 1
    for (int x = 0; x < cols; ++x) {
      const bool up = plus.has(x), down = minus.has(x), no = nan.has(x) || (up && down);
      if (!(up || down || no) || !sound(c0 + x)) continue;
      const float v = no ? NAN : up ? INFINITY : -INFINITY;
      const int t = (c0 + x) / a.group, head = h * a.group + c0 + x - t * a.group;
      if (float* to = part(c0 + x)) to[d] = v;
      else if (a.out_f32) reinterpret_cast<float*>(a.y + (first + t) * a.ldy)[head * D + d] = v;
      else reinterpret_cast<uint16_t*>(a.y + (first + t) * a.ldy)[head * D + d] = static_cast<uint16_t>(T::pair(v, 0.0f));
    }
  }
}

}  // namespace tars
