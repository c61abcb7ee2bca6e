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

template <int N>
struct Int {
  static constexpr int value = N;
};
// f(Int<0>), ..., f(Int<N - 1>), each decided when it is compiled.
template <int N, int I = 0, class F>
__device__ __forceinline__ void each(const F& f) {
  if constexpr (I < N) {
    f(Int<I>{});
    each<N, I + 1>(f);
  }
}

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

__device__ __forceinline__ uint32_t pair(int out, float a, float b) { return out == 1 ? Bf16::pair(a, b) : Fp16::pair(a, b); }

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
  const uint32_t lo = pair(a.out, y[0], y[1]), hi = pair(a.out, y[2], y[3]);
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

// ---- many rows: a workgroup of 2 x WN waves takes 32 FM rows of x and 16 FN WN of w, a wave 16 FM and 16 FN
//
// Stages of 128 k pass through a ring of three in LDS, by direct loads: a row's 64 bytes at a time, its four 16-byte blocks
// permuted so that a fragment's reads meet every bank once (the hardware takes 16 lanes of a 16-byte read together: lanes 0-3,
// 12-15 and 20-27 of each 32, and the rest). A stage's fragments are read, and a later stage loaded, between the products of the
// one before, an instruction or two behind each product, which is as many as a product hides; so nothing waits for LDS behind a
// barrier. x's fragments but the last kTwice are read over the ones that were just multiplied; those and w's have two places,
// so that the last read of a stage is well before its barrier.
//
// Scales come for four stages at a time: a row's 16 bytes, transposed as 4 x 4 on their way, so that a lane's dword holds the
// four stages' scales of its block, of which the product's operand selects the byte.
//
// Fragment j of w holds rows 64 (j / 4) + 16 (r / 4) + 4 (j % 4) + r % 4: the outputs of a lane's four neighbouring fragments
// are then 16 neighbours of a row.
__device__ __forceinline__ int x_swap(int row) { return -(row >> 2) & 3; }
__device__ __forceinline__ int w_swap(int row) { return -(row >> 4) & 3; }
// The row of w whose scales lie in place `at`: a fragment's 16 rows in neighbouring ones.
__device__ __forceinline__ int w_scale_row(int at) { return (at & ~63) | (at >> 2 & 3) << 4 | (at >> 4 & 3) << 2 | (at & 3); }

// Byte i of word g of the result is byte g of word i.
__device__ __forceinline__ uint4 transposed(uint4 v) {
  const auto perm = [](uint32_t hi, uint32_t lo, uint32_t s) { return __builtin_amdgcn_perm(hi, lo, s); };
  const uint32_t a = perm(v.y, v.x, 0x05010400u), b = perm(v.y, v.x, 0x07030602u);  // x0 y0 x1 y1, x2 y2 x3 y3
  const uint32_t c = perm(v.w, v.z, 0x05010400u), d = perm(v.w, v.z, 0x07030602u);
  return make_uint4(perm(c, a, 0x05040100u), perm(c, a, 0x07060302u), perm(d, b, 0x05040100u), perm(d, b, 0x07060302u));
}

template <int S>
__device__ __forceinline__ v4f mfma_fp4_scale(uint4 a, int sa, uint4 b, int sb, v4f c) {
  const v8i x = {static_cast<int>(a.x), static_cast<int>(a.y), static_cast<int>(a.z), static_cast<int>(a.w), 0, 0, 0, 0};
  const v8i y = {static_cast<int>(b.x), static_cast<int>(b.y), static_cast<int>(b.z), static_cast<int>(b.w), 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, kFp4, kFp4, S, sa, S, sb);
}

constexpr int kGroup = 8;  // tiles of x that take turns over a tile of w

template <int FM, int FN, int WN, bool TAIL>
__global__ __launch_bounds__(128 * WN, 4 / WN + (WN == 4)) void mx4_tile_kernel(Mx4GemmArgs a, int mt, int nt) {
  constexpr int kWaves = 2 * WN, BM = 32 * FM, BN = 16 * FN * WN, L = (BM + BN) / 16 / kWaves, XL = BM / 16 / kWaves;
  constexpr int SL = (BM + BN + 64 * kWaves - 1) / (64 * kWaves);
  static_assert(BM % (16 * kWaves) == 0 && BN % (16 * kWaves) == 0 && BM % 64 == 0 && FN % 4 == 0, "whole loads");
  constexpr int kStage = (BM + BN) * 64, kScales = SL * kWaves * 1024;
  constexpr int kTwice = 1, kOnce = FM - kTwice, kSlots = FM * FN;
  __shared__ __align__(1024) char lds[3 * kStage + 2 * kScales];  // the ring, scales as they come, scales transposed
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int wm = wave & 1, wn = wave >> 1;
  // consecutive tiles of an XCD: kGroup tiles of x by all of w's
  const int id = xcd_block(blockIdx.x, gridDim.x), per = kGroup * nt, first = id / per * kGroup, deep = min(kGroup, mt - first);
  const int m0 = (first + id % per % deep) * BM, n0 = id % per / deep * BN;
  // stages by fours; what is behind K counts for nothing
  const int blocks = a.K / 32, pieces = ceil_div(blocks, 16), stages = 4 * pieces;

  const char* const xb = a.x.values + m0 * a.x.ld_values;
  const char* const wb = a.w.values + n0 * a.w.ld_values;
  const uint8_t* const xsb = a.x.scales + m0 * a.x.ld_scales;
  const uint8_t* const wsb = a.w.scales + n0 * a.w.ld_scales;
  uint32_t off[L], soff[SL];
  int chunk[L];
#pragma unroll
  for (int u = 0; u < L; ++u) {  // 16 rows to a load, x's first
    const int row = 16 * (wave + kWaves * u) + lane / 4, mine = u < XL ? row : row - BM;
    chunk[u] = (lane & 3) ^ (u < XL ? x_swap(mine) : w_swap(mine));
    off[u] = u < XL ? min(mine, a.M - 1 - m0) * static_cast<uint32_t>(a.x.ld_values) : min(mine, a.N - 1 - n0) * static_cast<uint32_t>(a.w.ld_values);
    if (!TAIL) off[u] += 16 * chunk[u];
  }
#pragma unroll
  for (int u = 0; u < SL; ++u) {
    const int row = min(64 * (wave + kWaves * u) + lane, BM + BN - 1), mine = row < BM ? row : w_scale_row(row - BM);
    soff[u] = row < BM ? min(mine, a.M - 1 - m0) * static_cast<uint32_t>(a.x.ld_scales) : min(mine, a.N - 1 - n0) * static_cast<uint32_t>(a.w.ld_scales);
  }
  const uint32_t ring = lds_addr(lds);
  // load u of stage st
  auto issue_one = [&](int st, uint32_t dst, int u) __attribute__((always_inline)) {
    const char* base = u < XL ? xb : wb;
    if constexpr (TAIL) {  // behind K: the row's first block, whose scales are taken for 0
      const int block = 4 * st + chunk[u];
      ring_load16(base, off[u] + (block < blocks ? 16 * block : 0), dst + 1024 * kWaves * u);
    } else {
      ring_load16(base + 64 * st, off[u], dst + 1024 * kWaves * u);
    }
  };
  auto stage_at = [&](int slot) __attribute__((always_inline)) { return __builtin_amdgcn_readfirstlane(ring + kStage * slot + 1024 * wave); };
  auto issue_scales = [&](int piece) __attribute__((always_inline)) {
    const uint32_t dst = __builtin_amdgcn_readfirstlane(ring + 3 * kStage + 1024 * wave);
#pragma unroll
    for (int u = 0; u < SL; ++u) ring_load16((64 * (wave + kWaves * u) < BM ? xsb : wsb) + 16 * piece, soff[u], dst + 1024 * kWaves * u);
  };
  // a thread's own loads of scales
  char* const raw = lds + 3 * kStage + 16 * threadIdx.x;
  auto transpose_scales = [&](int piece) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < SL; ++u) {
      uint4 v = *reinterpret_cast<const uint4*>(raw + 1024 * kWaves * u);
      if constexpr (TAIL) {
        uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int left = blocks - 16 * piece - 4 * k;
          w[k] = left >= 4 ? w[k] : left <= 0 ? 0 : w[k] & ((1u << 8 * left) - 1);
        }
        v = make_uint4(w[0], w[1], w[2], w[3]);
      }
      *reinterpret_cast<uint4*>(raw + kScales + 1024 * kWaves * u) = transposed(v);
    }
  };
  // the wave's fragments in a stage and their scales
  const char* const x_at = lds + 64 * (wm * (BM / 2) + r) + 16 * (g ^ x_swap(r));
  const char* const w_at = lds + 64 * (BM + wn * (16 * FN) + 16 * (r / 4) + r % 4) + 16 * (g ^ w_swap(16 * (r / 4)));
  const char* const xs_at = lds + 3 * kStage + kScales + 16 * (wm * (BM / 2) + r) + 4 * g;
  const char* const ws_at = lds + 3 * kStage + kScales + 16 * (BM + wn * (16 * FN) + r) + 4 * g;
  struct Fragments {
    uint4 w[FN], x[kTwice];
  };
  uint4 x[kOnce];
  int xs[FM], ws[FN];
  auto read_w = [&](int at, int j) __attribute__((always_inline)) {
    return *reinterpret_cast<const uint4*>(w_at + at + 64 * (64 * (j / 4) + 4 * (j % 4)));
  };
  auto read_x = [&](int at, int i) __attribute__((always_inline)) { return *reinterpret_cast<const uint4*>(x_at + at + 1024 * i); };
  auto read_xs = [&](int i) __attribute__((always_inline)) { return *reinterpret_cast<const int*>(xs_at + 256 * i); };
  auto read_ws = [&](int j) __attribute__((always_inline)) { return *reinterpret_cast<const int*>(ws_at + 256 * j); };
  v4f c[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) c[i][j] = v4f{0, 0, 0, 0};
  // Keeps the sums from row `from` on in their registers, and the products on their side of a branch.
  auto hold = [&](int from) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        if (i < from) continue;
        asm volatile("" : "+v"(c[i][j]));
      }
  };
  auto barrier = [&]() __attribute__((always_inline)) {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  issue_scales(0);
#pragma unroll
  for (int st = 0; st < 3; ++st)
#pragma unroll
    for (int u = 0; u < L; ++u) issue_one(st, stage_at(st), u);
  wait_vmcnt<L>();
  asm volatile("" ::: "memory");
  transpose_scales(0);
  wait_lgkm0();
  barrier();
  Fragments f0, f1;
#pragma unroll
  for (int j = 0; j < FN; ++j) f0.w[j] = read_w(0, j);
#pragma unroll
  for (int i = 0; i < FM; ++i) (i < kOnce ? x[i] : f0.x[i - kOnce]) = read_x(0, i);
#pragma unroll
  for (int i = 0; i < FM; ++i) xs[i] = read_xs(i);
#pragma unroll
  for (int j = 0; j < FN; ++j) ws[j] = read_ws(j);
  wait_lgkm0();
  barrier();
  int slot = 0;  // of stage st
  // Multiplies stage st's fragments, st % 4 = S, and reads the next one's (behind the last stage: of whatever is there, not used).
  auto step = [&](auto s_, int st, Fragments& now, Fragments& next) __attribute__((always_inline)) {
    constexpr int S = decltype(s_)::value;
    const int after = slot + 1 == 3 ? 0 : slot + 1, at = kStage * after;
    // the loads of the stage after the next two, or of the last again: their number does not change
    const int ahead = min(st + 3, stages - 1);
    const uint32_t dst = stage_at(slot);
    if constexpr (S == 0) issue_scales(min((st >> 2) + 1, pieces - 1));
    issue_fence();
    each<kSlots>([&](auto t_) __attribute__((always_inline)) {
      constexpr int t = decltype(t_)::value, i = t / FN, j = t % FN;
      c[i][j] = mfma_fp4_scale<S>(now.w[j], ws[j], i < kOnce ? x[i < kOnce ? i : 0] : now.x[i < kOnce ? 0 : i - kOnce], xs[i], c[i][j]);
      each<L>([&](auto u) __attribute__((always_inline)) {
        if constexpr (decltype(u)::value * kSlots / L == t) issue_one(ahead, dst, decltype(u)::value);
      });
      if constexpr (t % FN == 0 && t > 0 && t / FN <= kOnce) x[t / FN - 1] = read_x(at, t / FN - 1);
      each<FN + kTwice>([&](auto k_) __attribute__((always_inline)) {
        constexpr int k = decltype(k_)::value;
        if constexpr (k * (kOnce * FN) / (FN + kTwice) + 1 == t) {
          if constexpr (k < FN) next.w[k] = read_w(at, k);
          else next.x[k - FN] = read_x(at, FM - kTwice + k - FN);
        }
      });
      if constexpr (S == 2 && t == 2) transpose_scales(min((st >> 2) + 1, pieces - 1));
      if constexpr (S == 3) {  // the next four stages' scales, x's over its own
        if constexpr (t % FN == 1 && t > FN) xs[t / FN - 1] = read_xs(t / FN - 1);
      }
      issue_fence();
    });
    if constexpr (S == 3) {
      xs[FM - 1] = read_xs(FM - 1);
#pragma unroll
      for (int j = 0; j < FN; ++j) ws[j] = read_ws(j);
    }
    hold(0);
    wait_lgkm0();
    wait_vmcnt<L>();
    barrier();
    slot = after;
  };
  hold(0);
  int st = 0;
  do {
    step(Int<0>{}, st, f0, f1);
    step(Int<1>{}, st + 1, f1, f0);
    step(Int<2>{}, st + 2, f0, f1);
    step(Int<3>{}, st + 3, f1, f0);
  } while ((st += 4) < stages);
  wait_vmcnt<0>();  // the ring's last loads, before its room gets another use
  barrier();

  // (the lane again, so that nothing of it is kept over the stages)
  int thread = threadIdx.x;
  asm volatile("" : "+v"(thread));
  const int nw = n0 + wn * (16 * FN), mw = m0 + wm * (BM / 2), col = thread & 15, part = thread >> 4 & 3;
  if (a.wide_rows && n0 + BN <= a.N) {  // 16 neighbours to a lane, 64 to a row, 32-bit offsets
    const auto all = [&](auto out_, auto bias_) __attribute__((always_inline)) {
      constexpr int out = decltype(out_)::value, e = out == 0 ? 4 : 2;
      char* const tile = a.y + mw * a.ldy + static_cast<int64_t>(nw) * e;
      const float* const bias = a.bias + nw;
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int m = 16 * i + col;
        const uint32_t at = m * static_cast<uint32_t>(a.ldy) + 16 * part * e;
#pragma unroll
        for (int j = 0; j < FN; j += 2) {
          const int n = 64 * (j / 4) + 4 * (j % 4);
          v4f y = c[i][j], z = c[i][j + 1];
          if constexpr (decltype(bias_)::value) {
            const float4 b = *reinterpret_cast<const float4*>(bias + 16 * part + n), d = *reinterpret_cast<const float4*>(bias + 16 * part + n + 4);
            y += v4f{b.x, b.y, b.z, b.w};
            z += v4f{d.x, d.y, d.z, d.w};
          }
          if (mw + m < a.M) {
            if constexpr (out == 0) {
              *reinterpret_cast<v4f*>(tile + (at + 4 * n)) = y;
              *reinterpret_cast<v4f*>(tile + (at + 4 * n + 16)) = z;
            } else {
              *reinterpret_cast<uint4*>(tile + (at + 2 * n)) = make_uint4(pair(out, y[0], y[1]), pair(out, y[2], y[3]), pair(out, z[0], z[1]), pair(out, z[2], z[3]));
            }
          }
        }
        hold(i + 1);
        issue_fence();
      }
    };
    const auto of = [&](auto out) __attribute__((always_inline)) {
      if (a.bias) all(out, Int<1>{});
      else all(out, Int<0>{});
    };
    if (a.out == 0) of(Int<0>{});
    else if (a.out == 1) of(Int<1>{});
    else of(Int<3>{});
    return;
  }
  // the output's edge, or rows that are not aligned: 16 rows at a time through the wave's own part of the ring
  constexpr int kCols = 16 * FN, kPitch = kCols + 4;
  static_assert(kWaves * 16 * kPitch * 4 <= 3 * kStage, "a wave's 16 rows fit");
  float* mine = reinterpret_cast<float*>(lds) + wave * 16 * kPitch;
#pragma unroll
  for (int i = 0; i < FM; ++i) {
#pragma unroll
    for (int j = 0; j < FN; ++j)
      *reinterpret_cast<v4f*>(mine + col * kPitch + 64 * (j / 4) + 16 * part + 4 * (j % 4)) = c[i][j];
    hold(i + 1);
    wait_lgkm0();
    issue_fence();
#pragma unroll 1
    for (int k = thread & 63; k < 16 * kCols; k += 64) {
      const int m = mw + 16 * i + k / kCols, n = nw + k % kCols;
      if (m < a.M && n < a.N) {
        const float y = mine[k / kCols * kPitch + k % kCols] + (a.bias ? a.bias[n] : 0.0f);
        char* to = a.y + m * a.ldy;
        if (a.out == 0) reinterpret_cast<float*>(to)[n] = y;
        else reinterpret_cast<uint16_t*>(to)[n] = static_cast<uint16_t>(pair(a.out, y, 0.0f));
      }
    }
    wait_lgkm0();
    issue_fence();
  }
}

template <int FM, int FN, int WN>
hipError_t tiles(const Mx4GemmArgs& a, hipStream_t s) {
  const int mt = ceil_div(a.M, 32 * FM), nt = ceil_div(a.N, 16 * FN * WN);
  const dim3 grid(mt * nt), block(128 * WN);
  if (a.K % 512) hipLaunchKernelGGL((mx4_tile_kernel<FM, FN, WN, true>), grid, block, 0, s, a, mt, nt);
  else hipLaunchKernelGGL((mx4_tile_kernel<FM, FN, WN, false>), grid, block, 0, s, a, mt, nt);
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
  if (a.dtype < 0 && a.M > 64)
    return static_cast<int64_t>(ceil_div(a.M, 256)) * ceil_div(a.N, 256) >= 200 ? tiles<8, 4, 4>(a, s) : tiles<4, 4, 2>(a, s);
  if (a.dtype < 0) return few<Codes>(a, s);
  return a.dtype == 0 ? few<XFp32>(a, s) : a.dtype == 1 ? few<XBf16>(a, s) : few<XFp16>(a, s);
}

}  // namespace tars
