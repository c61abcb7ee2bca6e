// Microscaled 4-bit floating point (OCP MXFP4): quantisation of rows, and products of two such matrices.
//
// 32 consecutive k share a scale 2^(b - 127): b is the exponent field of the block's largest magnitude as fp32, less 2 (the
// largest code, 6, has exponent 2), 0 at least; 255, NaN, where the block holds an infinity or NaN. A code is x / scale
// rounded to nearest even at e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6), 6 past it: x / scale is below 8. The quotient is exact, a power
// of two away, so the conversion instruction's rounding is the only one.
//
// y[m][n] = sum over k of x[m][k] w[n][k], on the matrix instructions that take codes and scales as they are: 16 x 16 outputs
// and 128 k each, a lane's operand being the 16 bytes of one block of one row. Products of codes are exact and the sums fp32.
#include <algorithm>

#include "paged_device.h"
#include "wave_reduce.h"

namespace tars {
namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef uint16_t v2u16 __attribute__((ext_vector_type(2)));

constexpr int kFp4 = 4;  // the matrix instruction's code for e2m1

// The first operand's rows are the output's rows 4 (lane / 16) + i, the second's its columns lane % 16.
__device__ __forceinline__ v4f mfma_fp4(uint4 a, int sa, uint4 b, int sb, v4f c) {
  const v8i x = {static_cast<int>(a.x), static_cast<int>(a.y), static_cast<int>(a.z), static_cast<int>(a.w), 0, 0, 0, 0};
  const v8i y = {static_cast<int>(b.x), static_cast<int>(b.y), static_cast<int>(b.z), static_cast<int>(b.w), 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, kFp4, kFp4, 0, sa, 0, sb);
}

// A block's scale byte from the exponent field of its largest magnitude, and the scale as the conversions take it.
__device__ __forceinline__ int scale_byte(int exponent) { return exponent == 255 ? 255 : max(exponent - 2, 0); }
__device__ __forceinline__ float scale_of(int byte) { return __uint_as_float(byte == 0 ? 1u << 22 : static_cast<uint32_t>(byte) << 23); }

// Element types of the rows that are quantised: E pairs or single values of 32 bits each.
struct XBf16 {
  static constexpr int kSize = 2;
  // the largest magnitude of the elements in n dwords, in an order that max_of keeps
  static __device__ __forceinline__ uint32_t magnitude(uint32_t w) { return w & 0x7FFF7FFFu; }
  static __device__ __forceinline__ uint32_t max_of(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(v2u16, a), __builtin_bit_cast(v2u16, b)));
  }
  static __device__ __forceinline__ int exponent(uint32_t m) { return static_cast<int>(max(m & 0xFFFFu, m >> 16) >> 7); }
  template <int AT>
  static __device__ __forceinline__ uint32_t codes(uint32_t old, const uint32_t* w, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(old, __builtin_bit_cast(v2bf, w[AT]), scale, AT);
  }
};
struct XFp16 {
  static constexpr int kSize = 2;
  static __device__ __forceinline__ uint32_t magnitude(uint32_t w) { return w & 0x7FFF7FFFu; }
  static __device__ __forceinline__ uint32_t max_of(uint32_t a, uint32_t b) { return XBf16::max_of(a, b); }
  static __device__ __forceinline__ int exponent(uint32_t m) {
    return static_cast<int>(__float_as_uint(Fp16::wide(max(m & 0xFFFFu, m >> 16))) >> 23);
  }
  template <int AT>
  static __device__ __forceinline__ uint32_t codes(uint32_t old, const uint32_t* w, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(old, __builtin_bit_cast(v2h, w[AT]), scale, AT);
  }
};
struct XFp32 {
  static constexpr int kSize = 4;
  static __device__ __forceinline__ uint32_t magnitude(uint32_t w) { return w & 0x7FFFFFFFu; }
  static __device__ __forceinline__ uint32_t max_of(uint32_t a, uint32_t b) { return max(a, b); }
  static __device__ __forceinline__ int exponent(uint32_t m) { return static_cast<int>(m >> 23); }
  template <int AT>
  static __device__ __forceinline__ uint32_t codes(uint32_t old, const uint32_t* w, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(old, __uint_as_float(w[2 * AT]), __uint_as_float(w[2 * AT + 1]), scale, AT);
  }
};
// Eight elements' codes.
template <class X>
__device__ __forceinline__ uint32_t eight_codes(const uint32_t* w, float scale) {
  uint32_t c = 0;
  c = X::template codes<0>(c, w, scale);
  c = X::template codes<1>(c, w, scale);
  c = X::template codes<2>(c, w, scale);
  return X::template codes<3>(c, w, scale);
}

// ---- quantisation: four lanes to a block, eight elements each
template <class X>
__global__ __launch_bounds__(256) void mx4_quant_kernel(Mx4QuantArgs a) {
  constexpr int kWords = 2 * X::kSize;
  const int row = blockIdx.y + blockIdx.z * 65535;
  if (row >= a.M) return;
  const int at = blockIdx.x * 256 + threadIdx.x, block = at / 4, blocks = a.K / 32;  // whole quads on either side of each test
  if (block >= blocks) {
    // the bytes behind a row's scales, up to the padded row's end
    if (block < a.pad_blocks && at % 4 == 0) a.scales[row * a.ld_scales + block] = 0;
    return;
  }
  const char* x = a.x + row * a.ldx + static_cast<int64_t>(at) * 8 * X::kSize;
  uint32_t w[kWords];
#pragma unroll
  for (int i = 0; i < kWords; i += 4) *reinterpret_cast<uint4*>(w + i) = *reinterpret_cast<const uint4*>(x + 4 * i);
  uint32_t m = X::magnitude(w[0]);
#pragma unroll
  for (int i = 1; i < kWords; ++i) m = X::max_of(m, X::magnitude(w[i]));
  m = X::max_of(m, static_cast<uint32_t>(dpp<kDppQuadXor1>(m)));
  m = X::max_of(m, static_cast<uint32_t>(dpp<kDppQuadXor2>(m)));
  const int byte = scale_byte(X::exponent(m));
  const uint32_t c = eight_codes<X>(w, scale_of(byte));
  *reinterpret_cast<uint32_t*>(a.values + row * a.ld_values + 4 * at) = byte == 255 ? 0 : c;  // NaN whatever the codes
  if (at % 4 == 0) a.scales[row * a.ld_scales + block] = static_cast<uint8_t>(byte);
}

// ---- the second operand of a product: a matrix in 4 bits, or one that is quantised in the registers
struct Codes {};

struct Operand {
  uint4 v;
  int s;
};
template <class X>
__device__ __forceinline__ Operand load_x(const Mx4GemmArgs& a, int row, int block) {
  Operand r;
  if constexpr (__is_same(X, Codes)) {
    r.v = *reinterpret_cast<const uint4*>(a.x.values + row * a.x.ld_values + 16 * block);
    r.s = a.x.scales[row * a.x.ld_scales + block];
  } else {
    constexpr int kWords = 8 * X::kSize;
    const char* x = a.rows + row * a.ld_rows + static_cast<int64_t>(block) * 32 * X::kSize;
    uint32_t w[kWords];
#pragma unroll
    for (int i = 0; i < kWords; i += 4) *reinterpret_cast<uint4*>(w + i) = *reinterpret_cast<const uint4*>(x + 4 * i);
    uint32_t m = X::magnitude(w[0]);
#pragma unroll
    for (int i = 1; i < kWords; ++i) m = X::max_of(m, X::magnitude(w[i]));
    r.s = scale_byte(X::exponent(m));
    const float scale = scale_of(r.s);
    r.v = make_uint4(eight_codes<X>(w, scale), eight_codes<X>(w + kWords / 4, scale), eight_codes<X>(w + kWords / 2, scale),
                     eight_codes<X>(w + 3 * kWords / 4, scale));
  }
  return r;
}

// Outputs n .. n + 3 of row m, those below N.
__device__ __forceinline__ void store_outputs(const Mx4GemmArgs& a, int m, int n, v4f y) {
  if (a.bias)
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] += a.bias[min(n + i, a.N - 1)];
  char* row = a.y + m * a.ldy;
  if (a.out == 0) {
    float* to = reinterpret_cast<float*>(row) + n;
    if (a.wide_store) *reinterpret_cast<v4f*>(to) = y;
    else
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < a.N) to[i] = y[i];
    return;
  }
  const uint32_t lo = a.out == 1 ? Bf16::pair(y[0], y[1]) : Fp16::pair(y[0], y[1]);
  const uint32_t hi = a.out == 1 ? Bf16::pair(y[2], y[3]) : Fp16::pair(y[2], y[3]);
  uint16_t* to = reinterpret_cast<uint16_t*>(row) + n;
  if (a.wide_store) {
    *reinterpret_cast<uint2*>(to) = make_uint2(lo, hi);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < a.N) to[i] = static_cast<uint16_t>((i < 2 ? lo : hi) >> (16 * (i & 1)));
  }
}

// ---- few rows: a wave takes NT tiles of 16 weight rows and MT of 16 rows, over its share of K, straight from memory; the KW
// waves that share the tiles add theirs in LDS, in order.
constexpr int kFewWaves = 8;

template <class X, int MT, int NT>
__global__ __launch_bounds__(64 * kFewWaves) void mx4_few_kernel(Mx4GemmArgs a, int kw) {
  __shared__ v4f part[kFewWaves][MT * NT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const int share = wave % kw, group = blockIdx.x * (kFewWaves / kw) + wave / kw;
  const int n0 = group * 16 * NT, m0 = blockIdx.y * 16 * MT;
  const int blocks = a.K / 32, steps = ceil_div(blocks, 4);
  v4f c[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) c[i][j] = v4f{0, 0, 0, 0};
  if (n0 < a.N) {
    const char* wv[NT];
    const uint8_t* ws[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int64_t n = min(n0 + 16 * j + r, a.N - 1);
      wv[j] = a.w.values + n * a.w.ld_values;
      ws[j] = a.w.scales + n * a.w.ld_scales;
    }
    const int per = ceil_div(steps, kw), s1 = min(steps, (share + 1) * per);
    for (int s = share * per; s < s1; ++s) {
      const int block = 4 * s + g;
      const bool in = block < blocks;
      const int at = in ? block : 0;
      Operand w[NT], x[MT];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        w[j].v = *reinterpret_cast<const uint4*>(wv[j] + 16 * at);
        w[j].s = in ? ws[j][at] : 0;
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int m = m0 + 16 * i + r;
        x[i] = {make_uint4(0, 0, 0, 0), 0};
        if (in && m < a.M) x[i] = load_x<X>(a, m, at);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) c[i][j] = mfma_fp4(w[j].v, w[j].s, x[i].v, x[i].s, c[i][j]);
    }
  }
  if (kw > 1) {
    if (share)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) part[wave][i * NT + j][lane] = c[i][j];
    __syncthreads();
    if (share) return;
    for (int k = 1; k < kw; ++k)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) c[i][j] += part[wave + k][i * NT + j][lane];
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int m = m0 + 16 * i + r, n = n0 + 16 * j + 4 * g;
      if (m < a.M && n < a.N) store_outputs(a, m, n, c[i][j]);
    }
}

template <class X>
hipError_t few(const Mx4GemmArgs& a, hipStream_t s) {
  const int tiles = ceil_div(a.N, 16), steps = ceil_div(a.K, 128);
  int kw = 1;
  while (kw < kFewWaves && tiles * kw < 2048 && 2 * kw <= steps) kw *= 2;
  const dim3 block(64 * kFewWaves);
  const int groups = ceil_div(tiles, kFewWaves / kw);
  if (a.M <= 16) hipLaunchKernelGGL((mx4_few_kernel<X, 1, 1>), dim3(groups, 1), block, 0, s, a, kw);
  else if (a.M <= 32) hipLaunchKernelGGL((mx4_few_kernel<X, 2, 1>), dim3(groups, 1), block, 0, s, a, kw);
  else hipLaunchKernelGGL((mx4_few_kernel<X, 4, 1>), dim3(groups, ceil_div(a.M, 64)), block, 0, s, a, kw);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_mx4_quant(const Mx4QuantArgs& a, hipStream_t s) {
  const dim3 grid(ceil_div(a.pad_blocks * 4, 256), std::min(a.M, 65535), ceil_div(a.M, 65535)), block(256);
  if (a.dtype == 0) hipLaunchKernelGGL(mx4_quant_kernel<XFp32>, grid, block, 0, s, a);
  else if (a.dtype == 1) hipLaunchKernelGGL(mx4_quant_kernel<XBf16>, grid, block, 0, s, a);
  else hipLaunchKernelGGL(mx4_quant_kernel<XFp16>, grid, block, 0, s, a);
  return hipGetLastError();
}

// Rows up to which the product quantises its operand itself.
constexpr int kFusedRows = 16;

bool mx4_quantises(int M) { return M <= kFusedRows; }

int64_t mx4_parts_bytes(int, int, int) { return 0; }

hipError_t launch_mx4_gemm(const Mx4GemmArgs& a, hipStream_t s) {
  if (a.dtype < 0) return few<Codes>(a, s);
  return a.dtype == 0 ? few<XFp32>(a, s) : a.dtype == 1 ? few<XBf16>(a, s) : few<XFp16>(a, s);
}

}  // namespace tars
