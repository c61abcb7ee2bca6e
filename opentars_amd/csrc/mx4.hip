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

// ---- quantisation: four lanes to a block, eight elements each: 16 or 32 bytes a lane, so that a wave's loads are whole lines; no
// element is read twice. 2011 x 4096 bf16 takes 7.0 us, 3.0 TB/s of reads and writes, most of it the launch's start and end.
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

// ---- a block of x as a product's operand: in 4 bits, or quantised here
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

// The swap of the four 16-byte blocks of a row's 64 bytes in LDS, such that the reads of a fragment's 16 rows, row r by lane r, meet
// every bank once: the hardware takes 16 lanes of a 16-byte read together, lanes 0-3, 12-15 and 20-27 of each 32, and the rest.
__device__ __forceinline__ int swap_of(int r) { return -(r >> 2) & 3; }

// ---- few rows: the workgroup keeps all of x in LDS, in 4 bits, its waves read w's rows once
//
// A wave takes tiles of 16 rows of w over its share of K; the kw waves that share a tile add theirs in LDS, in order. w comes by
// direct loads into the wave's own two slots of four steps of 128 k: lanes that are neighbours then read neighbouring bytes of a
// row (an operand's lanes are rows apart: read straight into it, 83 MB took 25 us, the loads' addresses what bounded it; so
// 14.4, 5.7 TB/s, and 16.5 where 20 such matrices take turns, which no cache holds). One slot is loaded while the other is
// multiplied, the first one while x is quantised.
//
// Smaller products are chains of latencies, launch, x, the first slot, the next: 37 x 12288 x 1536 takes 7.6 us, one of them x's
// quantising (6.5 with x in 4 bits), for 1.7 of bytes, and waves wait 61 % of their time.
constexpr int kFewWaves = 8, kFewSteps = 4, kFewSlot = kFewSteps * 1024 + 256;

template <class X, int MT>
__global__ __launch_bounds__(64 * kFewWaves) void mx4_few_kernel(Mx4GemmArgs a, int kw, int per) {
  extern __shared__ __align__(1024) char few_lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int share = wave % kw, tiles = ceil_div(a.N, 16), blocks = a.K / 32, steps = ceil_div(blocks, 4);
  const int first = min(steps, share * per), end = min(steps, first + per), loads = min(per, kFewSteps);
  char* const slots = few_lds + 2 * kFewSlot * wave;
  char* const xv = few_lds + 2 * kFewSlot * kFewWaves;                  // block b of row m: 16 bytes at b M + m
  uint8_t* const xs = reinterpret_cast<uint8_t*>(xv) + 16 * blocks * a.M;
  v4f* const part = reinterpret_cast<v4f*>(xv + (17 * blocks * a.M + 15) / 16 * 16);
  const int stride = gridDim.x * (kFewWaves / kw);
  int tile = blockIdx.x * (kFewWaves / kw) + wave / kw;

  const int load_row = lane >> 2, load_chunk = (lane & 3) ^ swap_of(load_row);
  const auto issue = [&](int tile, int s0, int slot) __attribute__((always_inline)) {
    const uint32_t dst = __builtin_amdgcn_readfirstlane(lds_addr(slots) + kFewSlot * slot);
    const char* v = a.w.values + min(16 * tile + load_row, a.N - 1) * a.w.ld_values;
#pragma unroll
    for (int u = 0; u < kFewSteps; ++u)
      if (u < loads) {
        const int block = 4 * (s0 + u) + load_chunk;
        ring_load16(v + 16 * (block < blocks ? block : 0), dst + 1024 * u);
      }
    if (lane < 16) ring_load16(a.w.scales + min(16 * tile + lane, a.N - 1) * a.w.ld_scales + (s0 & ~3) * 4, dst + 1024 * kFewSteps);
  };
  const auto wait_loads = [&](bool behind) __attribute__((always_inline)) {  // for a slot, with another's loads behind it
    if (!behind) wait_vmcnt<0>();
    else if (loads == 1) wait_vmcnt<2>();
    else if (loads == 2) wait_vmcnt<3>();
    else wait_vmcnt<5>();
    asm volatile("" ::: "memory");
  };
  const auto barrier = [&]() __attribute__((always_inline)) {
    asm volatile("" ::: "memory");
    wait_lgkm0();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  if (tile < tiles && first < end) issue(tile, first, 0);
  // a block to a thread: 16 x 4096 x 4096 from bf16 takes 5.7 us with weights that a cache holds (three of a thread's at once 6.8,
  // four lanes to a block 8.8)
  for (int i = threadIdx.x; i < blocks * a.M; i += 64 * kFewWaves) {
    const int m = i / blocks, b = i - m * blocks;
    const Operand o = load_x<X>(a, m, b);
    *reinterpret_cast<uint4*>(xv + 16 * (b * a.M + m)) = o.v;
    xs[b * a.M + m] = static_cast<uint8_t>(o.s);
  }
  barrier();
  int row[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) row[i] = min(16 * i + r, a.M - 1);
  const int value_at = 64 * r + 16 * (g ^ swap_of(r)), scale_at = 1024 * kFewSteps + 16 * r + g;
  int slot = 0;
  for (int base = blockIdx.x * (kFewWaves / kw); base < tiles; base += stride, tile += stride) {  // the same for every wave
    v4f c[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) c[i] = v4f{0, 0, 0, 0};
    if (tile < tiles)
      for (int s0 = first; s0 < end; s0 += kFewSteps) {
        const bool last = s0 + kFewSteps >= end, more = !last || tile + stride < tiles;
        wait_lgkm0();  // the other slot has been read
        if (more) issue(last ? tile + stride : tile, last ? first : s0 + kFewSteps, slot ^ 1);
        wait_loads(more);
        const char* from = slots + kFewSlot * slot;
#pragma unroll
        for (int u = 0; u < kFewSteps; ++u)
          if (u < loads) {
            const int block = 4 * (s0 + u) + g;
            // behind K or the wave's share: any block, with scales whose products are below fp32's smallest number
            const bool in = s0 + u < end && block < blocks;
            const int at = (in ? block : 0) * a.M;
            const uint4 v = *reinterpret_cast<const uint4*>(from + value_at + 1024 * u);
            const int w = from[scale_at + 4 * ((s0 + u) & 3)] & 255, ws = in ? w : 0;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              const uint4 x = *reinterpret_cast<const uint4*>(xv + 16 * (at + row[i]));
              const int s = in ? xs[at + row[i]] : 0;
              c[i] = mfma_fp4(v, ws, x, s, c[i]);
            }
          }
        slot ^= 1;
      }
    if (kw > 1) {
      if (share)
#pragma unroll
        for (int i = 0; i < MT; ++i) part[(wave * MT + i) * 64 + lane] = c[i];
      barrier();
      if (!share)
        for (int k = 1; k < kw; ++k)
#pragma unroll
          for (int i = 0; i < MT; ++i) c[i] += part[((wave + k) * MT + i) * 64 + lane];
      if (base + stride < tiles) barrier();
    }
    if (share == 0 && tile < tiles)
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int m = 16 * i + r, n = 16 * tile + 4 * g;
        if (m < a.M && n < a.N) store_outputs(a, m, n, c[i]);
      }
  }
}

// Whether x fits a workgroup's LDS beside the slots.
constexpr int kLds = 160 << 10;
int64_t few_lds_bytes(int M, int K, int kw) {
  return 2 * kFewSlot * kFewWaves + (17ll * (K / 32) * M + 15) / 16 * 16 + (kw > 1 ? kFewWaves * 1024 * ceil_div(M, 16) : 0);
}
// Waves to a tile of w, for 2048 waves in all, or 1024 with more than 16 rows of x: 1 x 4096 x 4096 takes
// 5.8, 4.4, 3.6 and 3.7 us with 512, 1024, 2048 and 4096 in all, 32 x 12288 x 4096 13.0, 10.3, 11.3 and 11.7. Both have 32 steps
// of 128 k: with other numbers the shares are uneven (few()).
int few_split(int M, int N, int K) {
  const int tiles = ceil_div(N, 16), steps = ceil_div(K, 128);
  int kw = 1;
  while (kw < kFewWaves && tiles * kw < (M <= 16 ? 2048 : 1024) && 2 * kw <= steps) kw *= 2;
  return kw;
}
// Up to 48 rows run this way, as far as x fits: x in 4 bits, weights that no cache holds, 32 x 12288 x 4096 takes 11.5 us (tiles
// 16.9), 32 x 4096 x 2048 5.6 (7.4), 48 x 4096 x 2560 7.4 (8.6), 48 x 2048 x 1024 4.6 (4.7), 48 x 12288 x 1536 7.1 (6.9); 64 x
// 2048 x 1024 would take 5.4 (4.7). Many columns of a short K are faster as tiles before that: 20, 32 and 48 x 32000 x 2048 10.8,
// 11.5 and 12.6 (11.6, 11.7 and 11.8). What does not fit runs as tiles: 16 x 4096 x 14336 14.9 us, 32 x 5120 x 5120 11.2,
// 48 x 4096 x 4096 10.8, for 5.0, 2.3 and 1.5 of bytes.
constexpr int kFewRows = 48;
bool few_fits(int M, int N, int K) { return M <= kFewRows && few_lds_bytes(M, K, few_split(M, N, K)) <= kLds; }

template <class X>
hipError_t few(const Mx4GemmArgs& a, hipStream_t s) {
  const int kw = few_split(a.M, a.N, a.K), groups = ceil_div(ceil_div(a.N, 16), kFewWaves / kw), share = ceil_div(ceil_div(a.K, 128), kw);
  // No slot's steps in two 16-byte pieces of scales, for which the last waves of a tile may have less or nothing: of 40 steps in
  // eight shares five take 8 each (16 x 5120 x 5120: 8.6 us).
  const int per = share <= 2 ? share : ceil_div(share, kFewSteps) * kFewSteps;
  const int lds = static_cast<int>(few_lds_bytes(a.M, a.K, kw));
  const dim3 grid(std::min(groups, 256 * (kLds / lds))), block(64 * kFewWaves);
  if (a.M <= 16) hipLaunchKernelGGL((mx4_few_kernel<X, 1>), grid, block, lds, s, a, kw, per);
  else if (a.M <= 32) hipLaunchKernelGGL((mx4_few_kernel<X, 2>), grid, block, lds, s, a, kw, per);
  else hipLaunchKernelGGL((mx4_few_kernel<X, 3>), grid, block, lds, s, a, kw, per);
  return hipGetLastError();
}

// ---- many rows: a workgroup of 2 x WN waves takes 32 FM rows of x and 16 FN WN of w, a wave 16 FM and 16 FN
//
// Pairs of stages of 128 k pass through a ring of D pairs in LDS, by direct loads: a row's 128 bytes at a time, a cache line, its
// eight 16-byte blocks swapped so that a fragment's reads meet every bank once. (Stages of 64 bytes a row came twice from L2.) A
// stage's fragments are read, and a later pair loaded, between the products of the one before, an instruction or two behind each
// product, which is as many as a product hides; so nothing waits for LDS behind a barrier, of which there is one to a pair. x's
// fragments but the last kTwice are read over the ones that were just multiplied; those and w's have two places, so that the last
// read of a stage is well before its barrier.
//
// Scales come for two pairs at a time: a row's 16 bytes, transposed as 4 x 4 on their way, so that a lane's dword holds the four
// stages' scales of its block, of which the product's operand selects the byte.
//
// Fragment j of w holds rows 64 (j / 4) + 16 (r / 4) + 4 (j % 4) + r % 4: the outputs of a lane's four neighbouring fragments
// are then 16 neighbours of a row.
//
// 8192 x 8192 x 8192 takes 265 us, 4.1 PFLOP/s. The clock falls to 1.77 of 2.4 GHz under it, at which the matrix units are busy for
// 53 % of the cycles: waves wait for loads and barriers a quarter of their time. Under the same instructions alone it falls to 1.6
// GHz, and they are busy for 93 %: 6.0 to 6.6 PFLOP/s.
//
// The swap of a row's blocks: row r of a fragment, by lane r (and as swap_of, for rows of 128 bytes).
__device__ __forceinline__ int x_swap(int row) { return row >> 1 & 7; }
__device__ __forceinline__ int w_swap(int row) { return (row >> 3 & 6) | (row >> 1 & 1); }
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

// Columns of a split's sums in the workspace.
__host__ __device__ __forceinline__ int split_cols(int N) { return (N + 15) / 16 * 16; }

constexpr int kGroup = 8;  // tiles of x that take turns over a tile of w

template <int FM, int FN, int WN, int D, bool TAIL>
__global__ __launch_bounds__(128 * WN, 2) void mx4_tile_kernel(Mx4GemmArgs a, int mt, int nt, int splits) {
  constexpr int kWaves = 2 * WN, BM = 32 * FM, BN = 16 * FN * WN, L = (BM + BN) / 8 / kWaves, XL = BM / 8 / kWaves;
  constexpr int SL = (BM + BN + 64 * kWaves - 1) / (64 * kWaves);
  static_assert(BM % (8 * kWaves) == 0 && BN % (8 * kWaves) == 0 && BM % 64 == 0 && FN % 4 == 0 && D >= 2 && D <= 4, "whole loads; scales as far ahead as the ring");
  constexpr int kPair = (BM + BN) * 128, kScales = SL * kWaves * 1024;
  constexpr int kTwice = 1, kOnce = FM - kTwice, kSlots = FM * FN;
  __shared__ __align__(1024) char lds[D * kPair + 3 * kScales];  // the ring, scales transposed, scales as they come
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int wm = wave & 1, wn = wave >> 1;
  // consecutive tiles of an XCD: kGroup tiles of x by all of w's
  const int number = xcd_block(blockIdx.x, gridDim.x), split = number / (mt * nt), id = number - split * mt * nt;
  const int per = kGroup * nt, first = id / per * kGroup, deep = min(kGroup, mt - first);
  const int m0 = (first + id % per % deep) * BM, n0 = id % per / deep * BN;
  // stages by fours, the workgroup's share of them; what is behind K counts for nothing
  const int all_blocks = a.K / 32, each_split = ceil_div(ceil_div(all_blocks, 16), splits), start = split * each_split;
  const int blocks = min(all_blocks - 16 * start, 16 * each_split), pieces = ceil_div(blocks, 16), pairs = 2 * pieces;

  const char* const xb = a.x.values + m0 * a.x.ld_values + 256 * start;
  const char* const wb = a.w.values + n0 * a.w.ld_values + 256 * start;
  const uint8_t* const xsb = a.x.scales + m0 * a.x.ld_scales + 16 * start;
  const uint8_t* const wsb = a.w.scales + n0 * a.w.ld_scales + 16 * start;
  uint32_t off[L], soff[SL];
  int chunk[L];
#pragma unroll
  for (int u = 0; u < L; ++u) {  // 8 rows to a load, x's first
    const int row = 8 * (wave + kWaves * u) + lane / 8, mine = u < XL ? row : row - BM;
    chunk[u] = (lane & 7) ^ (u < XL ? x_swap(mine) : w_swap(mine));
    off[u] = u < XL ? min(mine, a.M - 1 - m0) * static_cast<uint32_t>(a.x.ld_values) : min(mine, a.N - 1 - n0) * static_cast<uint32_t>(a.w.ld_values);
    if (!TAIL) off[u] += 16 * chunk[u];
  }
#pragma unroll
  for (int u = 0; u < SL; ++u) {
    const int row = min(64 * (wave + kWaves * u) + lane, BM + BN - 1), mine = row < BM ? row : w_scale_row(row - BM);
    soff[u] = row < BM ? min(mine, a.M - 1 - m0) * static_cast<uint32_t>(a.x.ld_scales) : min(mine, a.N - 1 - n0) * static_cast<uint32_t>(a.w.ld_scales);
  }
  const uint32_t ring = lds_addr(lds);
  // load u of a pair of stages
  auto issue_one = [&](int pair, uint32_t dst, int u) __attribute__((always_inline)) {
    const char* base = u < XL ? xb : wb;
    if constexpr (TAIL) {  // behind K: the row's first block, whose scales are taken for 0
      const int block = 8 * pair + chunk[u];
      ring_load16(base, off[u] + (block < blocks ? 16 * block : 0), dst + 1024 * kWaves * u);
    } else {
      ring_load16(base + 128 * pair, off[u], dst + 1024 * kWaves * u);
    }
  };
  auto pair_at = [&](int slot) __attribute__((always_inline)) { return __builtin_amdgcn_readfirstlane(ring + kPair * slot + 1024 * wave); };
  auto issue_scales = [&](int piece) __attribute__((always_inline)) {
    const int from = min(piece, pieces - 1);
    const uint32_t dst = __builtin_amdgcn_readfirstlane(ring + D * kPair + kScales * (1 + (piece & 1)) + 1024 * wave);
#pragma unroll
    for (int u = 0; u < SL; ++u) ring_load16((64 * (wave + kWaves * u) < BM ? xsb : wsb) + 16 * from, soff[u], dst + 1024 * kWaves * u);
  };
  // a thread's own loads of scales
  char* const done = lds + D * kPair + 16 * threadIdx.x;
  auto transpose_scales = [&](int piece) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < SL; ++u) {
      uint4 v = *reinterpret_cast<const uint4*>(done + kScales * (1 + (piece & 1)) + 1024 * kWaves * u);
      if constexpr (TAIL) {
        uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int left = blocks - 16 * piece - 4 * k;
          w[k] = left >= 4 ? w[k] : left <= 0 ? 0 : w[k] & ((1u << 8 * left) - 1);
        }
        v = make_uint4(w[0], w[1], w[2], w[3]);
      }
      *reinterpret_cast<uint4*>(done + 1024 * kWaves * u) = transposed(v);
    }
  };
  // the wave's fragments in a stage and their scales
  // (of the pair's first stage; the second's are 64 bytes up or down)
  const uint32_t x_at = 128 * (wm * (BM / 2) + r) + 16 * (g ^ x_swap(r));
  const uint32_t w_at = 128 * (BM + wn * (16 * FN) + 16 * (r / 4) + r % 4) + 16 * (g ^ w_swap(16 * (r / 4) + r % 4));
  const char* const xs_at = lds + D * kPair + 16 * (wm * (BM / 2) + r) + 4 * g;
  const char* const ws_at = lds + D * kPair + 16 * (BM + wn * (16 * FN) + r) + 4 * g;
  struct Fragments {
    uint4 w[FN], x[kTwice];
  };
  uint4 x[kOnce];
  int xs[FM], ws[FN];
  auto read_w = [&](uint32_t at, int j) __attribute__((always_inline)) {
    return *reinterpret_cast<const uint4*>(lds + at + 128 * (64 * (j / 4) + 4 * (j % 4)));
  };
  auto read_x = [&](uint32_t at, int i) __attribute__((always_inline)) { return *reinterpret_cast<const uint4*>(lds + at + 2048 * i); };
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
  for (int d = 0; d < D; ++d) {
#pragma unroll
    for (int u = 0; u < L; ++u) issue_one(min(d, pairs - 1), pair_at(d), u);
    if (d == 0) issue_scales(1);
  }
  wait_vmcnt<(D - 1) * L>();
  asm volatile("" ::: "memory");
  transpose_scales(0);
  wait_lgkm0();
  barrier();
  Fragments f0, f1;
#pragma unroll
  for (int j = 0; j < FN; ++j) f0.w[j] = read_w(w_at, j);
#pragma unroll
  for (int i = 0; i < FM; ++i) (i < kOnce ? x[i] : f0.x[i - kOnce]) = read_x(x_at, i);
#pragma unroll
  for (int i = 0; i < FM; ++i) xs[i] = read_xs(i);
#pragma unroll
  for (int j = 0; j < FN; ++j) ws[j] = read_ws(j);
  wait_lgkm0();
  barrier();
  int slot = 0;  // of stage st's pair
  // Multiplies stage st's fragments, st % 4 = S, and reads the next one's (behind the last stage: of whatever is there, not used).
  auto step = [&](auto s_, int st, Fragments& now, Fragments& next) __attribute__((always_inline)) {
    constexpr int S = decltype(s_)::value;
    constexpr bool second = S & 1;  // the pair's fragments are all read: the pair that is a ring ahead, or the last again, takes its slot
    const int after = !second ? slot : slot + 1 == D ? 0 : slot + 1;
    const uint32_t xa = kPair * after + (second ? x_at : x_at ^ 64), wa = kPair * after + (second ? w_at : w_at ^ 64);
    const int ahead = min((st >> 1) + D, pairs - 1);
    const uint32_t dst = pair_at(slot);
    if constexpr (S == 1) issue_scales((st >> 2) + 2);
    issue_fence();
    each<kSlots>([&](auto t_) __attribute__((always_inline)) {
      constexpr int t = decltype(t_)::value, i = t / FN, j = t % FN;
      c[i][j] = mfma_fp4_scale<S>(now.w[j], ws[j], i < kOnce ? x[i < kOnce ? i : 0] : now.x[i < kOnce ? 0 : i - kOnce], xs[i], c[i][j]);
      each<L>([&](auto u) __attribute__((always_inline)) {
        if constexpr (second && decltype(u)::value * kSlots / L == t) issue_one(ahead, dst, decltype(u)::value);
      });
      if constexpr (t % FN == 0 && t > 0 && t / FN <= kOnce) x[t / FN - 1] = read_x(xa, t / FN - 1);
      each<FN + kTwice>([&](auto k_) __attribute__((always_inline)) {
        constexpr int k = decltype(k_)::value;
        if constexpr (k * (kOnce * FN) / (FN + kTwice) + 1 == t) {
          if constexpr (k < FN) next.w[k] = read_w(wa, k);
          else next.x[k - FN] = read_x(xa, FM - kTwice + k - FN);
        }
      });
      if constexpr (S == 2 && t == 2) transpose_scales((st >> 2) + 1);
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
    if constexpr (!second) {
      wait_vmcnt<(D - 2) * L>();
      barrier();
    }
    slot = after;
  };
  hold(0);
  int st = 0;
  do {
    step(Int<0>{}, st, f0, f1);
    step(Int<1>{}, st + 1, f1, f0);
    step(Int<2>{}, st + 2, f0, f1);
    step(Int<3>{}, st + 3, f1, f0);
  } while ((st += 4) < 2 * pairs);
  wait_vmcnt<0>();  // the ring's last loads, before its room gets another use
  barrier();

  // the lane again where it is wanted, so that nothing of it is kept over the stages
  const auto thread_again = []() __attribute__((always_inline)) {
    int t = threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
  };
  const int nw = n0 + wn * (16 * FN), mw = m0 + wm * (BM / 2);
  // 16 neighbours to a lane, 64 to a row, eight of them within `cols` or none; 32-bit offsets
  const auto store_rows = [&](auto out_, auto bias_, char* y, int64_t ldy, int cols) __attribute__((always_inline)) {
    constexpr int out = decltype(out_)::value, e = out == 0 ? 4 : 2;
    char* const tile = y + mw * ldy + static_cast<int64_t>(nw) * e;
    const float* const bias = a.bias + nw;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int thread = thread_again(), col = thread & 15, part = thread >> 4 & 3, m = 16 * i + col;
      const uint32_t at = m * static_cast<uint32_t>(ldy) + 16 * part * e;
#pragma unroll
      for (int j = 0; j < FN; j += 2) {
        const int n = 64 * (j / 4) + 4 * (j % 4);
        v4f v = c[i][j], z = c[i][j + 1];
        const bool in = nw + 16 * part + n < cols;
        if constexpr (decltype(bias_)::value) {
          const float* at_bias = bias + (in ? 16 * part + n : -nw);
          const float4 b = *reinterpret_cast<const float4*>(at_bias), d = *reinterpret_cast<const float4*>(at_bias + 4);
          v += v4f{b.x, b.y, b.z, b.w};
          z += v4f{d.x, d.y, d.z, d.w};
        }
        if (in && mw + m < a.M) {
          if constexpr (out == 0) {
            *reinterpret_cast<v4f*>(tile + (at + 4 * n)) = v;
            *reinterpret_cast<v4f*>(tile + (at + 4 * n + 16)) = z;
          } else {
            *reinterpret_cast<uint4*>(tile + (at + 2 * n)) = make_uint4(pair(out, v[0], v[1]), pair(out, v[2], v[3]), pair(out, z[0], z[1]), pair(out, z[2], z[3]));
          }
        }
      }
      hold(i + 1);
      issue_fence();
    }
  };
  if (splits > 1) {
    const int64_t ld = 4ll * split_cols(a.N);
    store_rows(Int<0>{}, Int<0>{}, a.work + split * a.M * ld, ld, split_cols(a.N));
    return;
  }
  if (a.wide_rows && a.N % 8 == 0) {
    const auto of = [&](auto out) __attribute__((always_inline)) {
      if (a.bias) store_rows(out, Int<1>{}, a.y, a.ldy, a.N);
      else store_rows(out, Int<0>{}, a.y, a.ldy, a.N);
    };
    if (a.out == 0) of(Int<0>{});
    else if (a.out == 1) of(Int<1>{});
    else of(Int<3>{});
    return;
  }
  if (a.wide_store) {  // four neighbours of a row are aligned (64 x 300 x 512: 4.7 us, through LDS 7.3)
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int thread = thread_again(), m = mw + 16 * i + (thread & 15), n = nw + (thread & 48);
#pragma unroll
      for (int j = 0; j < FN; ++j)
        if (m < a.M && n + 4 * j < a.N) store_outputs(a, m, n + 4 * j, c[i][j]);
      hold(i + 1);
      issue_fence();
    }
    return;
  }
  // rows that are not aligned: 16 at a time through the wave's own part of the ring, then a column to a lane (3335 x 1373 x 14208
  // in whole tiles: 92 us, and 109 with one element after the other)
  static_assert(FN == 4, "a column of a wave's to each lane");
  constexpr int kPitch = 68, kAtOnce = FM > 4 ? 8 : 16;
  static_assert(kWaves * 16 * kPitch * 4 <= D * kPair, "a wave's 16 rows fit");
  float* mine = reinterpret_cast<float*>(lds) + wave * 16 * kPitch;
  const auto store_columns = [&](auto out_) __attribute__((always_inline)) {
    constexpr int out = decltype(out_)::value;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int thread = thread_again(), col = thread & 15, part = thread >> 4 & 3, lane = thread & 63;
      const int n = nw + lane, first = __builtin_amdgcn_readfirstlane(mw) + 16 * i;
#pragma unroll
      for (int j = 0; j < FN; ++j) *reinterpret_cast<v4f*>(mine + col * kPitch + 16 * part + 4 * j) = c[i][j];
      hold(i + 1);
      wait_lgkm0();
      issue_fence();
      const float bias = a.bias ? a.bias[min(n, a.N - 1)] : 0.0f;
#pragma unroll 1
      for (int r0 = 0; r0 < 16 && first + r0 < a.M; r0 += kAtOnce) {
        float y[kAtOnce];
#pragma unroll
        for (int r = 0; r < kAtOnce; ++r) y[r] = mine[(r0 + r) * kPitch + lane] + bias;
#pragma unroll
        for (int r = 0; r < kAtOnce; ++r) {
          const int m = first + r0 + r;
          char* to = a.y + m * a.ldy;
          if (m < a.M && n < a.N) {
            if constexpr (out == 0) reinterpret_cast<float*>(to)[n] = y[r];
            else reinterpret_cast<uint16_t*>(to)[n] = static_cast<uint16_t>(pair(out, y[r], 0.0f));
          }
        }
      }
      wait_lgkm0();
      issue_fence();
    }
  };
  if (a.out == 0) store_columns(Int<0>{});
  else if (a.out == 1) store_columns(Int<1>{});
  else store_columns(Int<3>{});
}

// The splits' sums in order: four neighbours to a thread, which pass 32 bits in no shape that is split (tile_choice).
__global__ __launch_bounds__(256) void mx4_join_kernel(Mx4GemmArgs a, int splits) {
  const int cols = split_cols(a.N), quads = cols / 4;
  const uint32_t i = blockIdx.x * 256 + threadIdx.x, all = static_cast<uint32_t>(a.M) * quads;
  if (i >= all) return;
  const int m = i / quads, n = (i - m * quads) * 4;
  const v4f* from = reinterpret_cast<const v4f*>(a.work) + i;
  v4f y = from[0];
#pragma unroll 4
  for (int k = 1; k < splits; ++k) y += from[static_cast<int64_t>(k) * all];
  if (n < a.N) store_outputs(a, m, n, y);
}

template <int FM, int FN, int WN, int D>
hipError_t tiles(const Mx4GemmArgs& a, hipStream_t s, int splits = 1) {
  const int mt = ceil_div(a.M, 32 * FM), nt = ceil_div(a.N, 16 * FN * WN);
  const dim3 grid(mt * nt * splits), block(128 * WN);
  if (a.K % 512) hipLaunchKernelGGL((mx4_tile_kernel<FM, FN, WN, D, true>), grid, block, 0, s, a, mt, nt, splits);
  else hipLaunchKernelGGL((mx4_tile_kernel<FM, FN, WN, D, false>), grid, block, 0, s, a, mt, nt, splits);
  if (splits > 1) {
    const int64_t quads = static_cast<int64_t>(a.M) * (split_cols(a.N) / 4);
    hipLaunchKernelGGL(mx4_join_kernel, dim3(static_cast<uint32_t>((quads + 255) / 256)), dim3(256), 0, s, a, splits);
  }
  return hipGetLastError();
}

// Tiles of 256 x 256, 128 x 128 or 64 x 128, and parts of K, by what they would take, in ns: a start, the stages in rounds that
// fill the card, of which the last may leave CUs to fewer workgroups, and a second launch that joins the parts. A stage's times
// are of 8192 x 8192 x 8192 (265, 353 and 464 us) and, a workgroup to a CU or less, of 64 x 4096 x 4096 (23.6, 10.8 and 8.8 us),
// whose weights a cache held. 2011 x 12288 x 4096 takes 67, 72 and 92 us with such weights, 71, 77 and 110 with weights that none
// holds. In eight parts 100 x 1024 x 8192 takes 10 us for 17.9 (64 x 128 tiles), in two 64 x 4096 x 4096 10.4 for 8.8, which is why
// the join counts. Where few workgroups wait for memory the times are too short, and parts would be better than the rule has it:
// 64 x 4096 x 4096 takes 12.0 us whole and 11.5 in two, 128 x 8192 x 8192 30.3 and 23.4 (21.4 and 19.2 out of a cache). (Whole
// rounds of columns first and the rest in smaller tiles, by a second launch, took 75, 86 and 90 us where the rule took 75, 83 and
// 102 on the same card, for 2011 x 12288 x 4096, 5000 x 5000 x 5120 and 3000 x 11008 x 4096.)
struct TileChoice {
  int kind, splits;
};
TileChoice tile_choice(int M, int N, int K) {
  const struct {
    int m, n, slots, full, one, none;  // workgroups at a time; ns of a stage with all of them, with one to a CU, with few
  } kinds[] = {{256, 256, 256, 1030, 1030, 650}, {128, 128, 512, 690, 400, 310}, {64, 128, 512, 450, 260, 200}};
  const int pieces = ceil_div(K, 512);
  double best = 1e30;
  TileChoice choice{0, 1};
  for (int i = 0; i < 3; ++i) {
    const auto& k = kinds[i];
    const int64_t tiles = static_cast<int64_t>(ceil_div(M, k.m)) * ceil_div(N, k.n);
    for (int want = 1; want <= 32 && want <= pieces; want *= 2) {
      const int each = ceil_div(pieces, want), splits = ceil_div(pieces, each);
      const double bytes = 8.0 * splits * M * split_cols(N);
      if (splits > 1 && (tiles * splits > 1024 || bytes > 128e6)) continue;
      const int64_t all = tiles * splits, left = all % k.slots;
      const double last = left > 256 ? k.full : all > left ? k.one : k.none + (k.one - k.none) * left / 256.0;
      const double ns = 4.0 * each * (all / k.slots * k.full + (left ? last : 0)) + (splits > 1 ? 2500 + bytes / 3000 : 0);
      if (ns < best) best = ns, choice = {i, splits};
    }
  }
  return choice;
}

}  // namespace

hipError_t launch_mx4_quant(const Mx4QuantArgs& a, hipStream_t s) {
  const dim3 grid(ceil_div(a.pad_blocks * 4, 256), std::min(a.M, 65535), ceil_div(a.M, 65535)), block(256);
  if (a.dtype == 0) hipLaunchKernelGGL(mx4_quant_kernel<XFp32>, grid, block, 0, s, a);
  else if (a.dtype == 1) hipLaunchKernelGGL(mx4_quant_kernel<XBf16>, grid, block, 0, s, a);
  else hipLaunchKernelGGL(mx4_quant_kernel<XFp16>, grid, block, 0, s, a);
  return hipGetLastError();
}

// Whether few rows are quantised by every workgroup itself rather than by a launch before: 1 x 4096 x 4096 then takes 3.8 us for
// 5.2, 16 x 4096 x 4096 6.1 for 7.0; from 2^17 elements on it is the same (2 x 2048 x 65536, 32 x 1024 x 8192).
bool mx4_quantises(int M, int N, int K) { return few_fits(M, N, K) && static_cast<int64_t>(M) * K <= 1 << 17; }

int64_t mx4_parts_bytes(int M, int N, int K) {
  if (few_fits(M, N, K)) return 0;
  const int splits = tile_choice(M, N, K).splits;
  return splits > 1 ? 4ll * splits * M * split_cols(N) : 0;
}

hipError_t launch_mx4_gemm(const Mx4GemmArgs& a, hipStream_t s) {
  if (a.dtype >= 0) return a.dtype == 0 ? few<XFp32>(a, s) : a.dtype == 1 ? few<XBf16>(a, s) : few<XFp16>(a, s);
  if (few_fits(a.M, a.N, a.K)) return few<Codes>(a, s);
  const TileChoice c = tile_choice(a.M, a.N, a.K);
  return c.kind == 0 ? tiles<8, 4, 4, 2>(a, s, c.splits) : c.kind == 1 ? tiles<4, 4, 2, 2>(a, s, c.splits) : tiles<2, 4, 2, 2>(a, s, c.splits);
}

}  // namespace tars
