// The norm of queries and keys for each head and their rotation by position, in one pass over the rows; the keys, and the
// values, may go straight to their pages of a key / value cache.
//
// For a head's hd elements x of the row at position p:  u = x gamma / sqrt(mean(x^2) + eps)  (u = x without a gamma), and with
// h = rot / 2 and the table's row p = [cos(0 .. h - 1), sin(0 .. h - 1)]:  y[i] = u[i] cos_i - u[i + h] sin_i,
// y[i + h] = u[i + h] cos_i + u[i] sin_i for i < h, y = u behind rot. All of it fp32, rounded once where it is stored: to the
// rows' type, or as kv_append does to e4m3.
//
// hd / 16 lanes take a head, two chunks of 8 elements each: chunk j and the one it is rotated with, rot / 16 chunks on, or two
// of the elements that are not rotated. So a rotation stays in a lane, and a norm crosses 4, 8 or 16 neighbours. Memory bounds it:
// 127 MB of 6 prompts' rows take 24 us (5.3 TB/s), 90 MB into an e4m3 cache 19, with fp64 quotients beside.
#include "paged_device.h"
#include "wave_reduce.h"

namespace tars {
namespace {

constexpr int kThreads = 256;

template <int L>
__device__ __forceinline__ float lanes_sum(float x) {
  x += __int_as_float(dpp<kDppQuadXor1>(__float_as_int(x)));
  x += __int_as_float(dpp<kDppQuadXor2>(__float_as_int(x)));
  if constexpr (L >= 8) x += __int_as_float(dpp<kDppRowHalfMirror>(__float_as_int(x)));
  if constexpr (L >= 16) x += __int_as_float(dpp<kDppRowMirror>(__float_as_int(x)));
  return x;
}

// 1 / sqrt(x), to a step of fp32; the instruction takes subnormal numbers for 0.
__device__ __forceinline__ float inverse_root(float x) {
  const bool low = x < 0x1p-96f;
  return __builtin_amdgcn_rsqf(low ? x * 0x1p96f : x) * (low ? 0x1p48f : 1.0f);
}

template <class T>
__device__ __forceinline__ void widen(uint4 v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = T::wide(w[i] & 0xFFFFu);
    x[2 * i + 1] = T::wide(w[i] >> 16);
  }
}
template <class T>
__device__ __forceinline__ uint4 narrow(const float (&x)[8]) {
  return make_uint4(T::pair(x[0], x[1]), T::pair(x[2], x[3]), T::pair(x[4], x[5]), T::pair(x[6], x[7]));
}
// Eight e4m3 values x / scale: the quotient as kv_append forms it, saturating at 448, NaN kept.
__device__ __forceinline__ uint2 narrow_e4m3(const float (&x)[8], double inv) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    f[i] = static_cast<float>(x[i] * inv);
    f[i] = f[i] != f[i] ? f[i] : fminf(fmaxf(f[i], -448.0f), 448.0f);
  }
  uint32_t lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false), hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[4], f[5], 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[6], f[7], hi, true);
  return make_uint2(lo, hi);
}

// A wave takes 64 / L heads of one row (all of a row's, in turn, took 37.2 us where this takes 32.8, for 4096 rows of 72 heads of
// 128, and 4.6 for 3.5 with 512 rows of 24). Heads: the queries', the keys' and, into a cache, the values'.
template <class T, int L, bool STORE, bool E4M3>
__global__ __launch_bounds__(kThreads) void qk_rope_kernel(QkRopeArgs a, int waves_per_row) {
  const int item = __builtin_amdgcn_readfirstlane((blockIdx.x * kThreads + threadIdx.x) / 64);
  const int row = item / waves_per_row, part = item - row * waves_per_row;
  const KvSeqs& s = a.seqs;
  if (row >= s.rows) return;
  int b = row, i = 0, n = 1;
  if (s.starts) {
    b = seq_of_row(s, row);
    if (b >= s.seqs) return;
    const RowSpan span = seq_rows(s.starts, b, s.rows);
    i = row - span.first;
    n = span.n;
    if (i < 0 || i >= n) return;
  }
  const int p = seq_len(s.lens, b, s.cap) - n + i;
  if (p < 0 || p >= a.positions) return;
  const int lane = threadIdx.x & 63, j = lane % L, turning = a.rot / 16;
  // the lane's two chunks
  const bool turns = j < turning;
  const int c0 = turns ? j : 2 * j, c1 = turns ? j + turning : 2 * j + 1;
  float cs[8], sn[8];
  if (turns) {
    const float* t = a.tab + static_cast<int64_t>(p) * a.rot + 8 * j;
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      *reinterpret_cast<float4*>(cs + e) = *reinterpret_cast<const float4*>(t + e);
      *reinterpret_cast<float4*>(sn + e) = *reinterpret_cast<const float4*>(t + a.rot / 2 + e);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) cs[e] = 1, sn[e] = 0;
  }
  char* kd = nullptr;
  char* vd = nullptr;
  if constexpr (STORE) {
    const int page = s.table[b * s.ld_table + (p >> a.pool.page_shift)];
    if (page >= 0 && page < a.pool.pages) {
      const int slot = p & ((1 << a.pool.page_shift) - 1);
      kd = a.pool.k + page * a.pool.k_page + slot * a.pool.k_slot;
      vd = a.pool.v + page * a.pool.v_page + slot * a.pool.v_slot;
    }
  }
  const int all = a.heads + (STORE ? 2 : 1) * a.kv_heads;
  const int h = part * (64 / L) + lane / L;
  if (h >= all) return;
  const int kind = h < a.heads ? 0 : h < a.heads + a.kv_heads ? 1 : 2;  // query, key, value
  const int hh = kind == 0 ? h : kind == 1 ? h - a.heads : h - a.heads - a.kv_heads;
  const char* x = (kind == 0 ? a.q + row * a.ldq : kind == 1 ? a.k + row * a.ldk : a.v + row * a.ldv) + hh * (32 * L);
  const uint4 r0 = *reinterpret_cast<const uint4*>(x + 16 * c0), r1 = *reinterpret_cast<const uint4*>(x + 16 * c1);
  float x0[8], x1[8];
  widen<T>(r0, x0);
  widen<T>(r1, x1);
  const float* gamma = kind == 0 ? a.qgamma : kind == 1 ? a.kgamma : nullptr;
  float sum = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) sum += x0[e] * x0[e] + x1[e] * x1[e];
  sum = lanes_sum<L>(sum);
  if (gamma) {
    const float k = inverse_root(sum * (1.0f / (16 * L)) + a.eps);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x0[e] = x0[e] * k * gamma[8 * c0 + e];
      x1[e] = x1[e] * k * gamma[8 * c1 + e];
    }
  }
  if (kind != 2 && turns) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float y0 = x0[e] * cs[e] - x1[e] * sn[e], y1 = x1[e] * cs[e] + x0[e] * sn[e];
      x0[e] = y0;
      x1[e] = y1;
    }
  }
  if (kind == 0 || !STORE) {
    char* y = (kind == 0 ? a.yq + row * a.ldyq : a.yk + row * a.ldyk) + hh * (32 * L);
    *reinterpret_cast<uint4*>(y + 16 * c0) = narrow<T>(x0);
    *reinterpret_cast<uint4*>(y + 16 * c1) = narrow<T>(x1);
  } else if (kd) {
    char* y = kind == 1 ? kd + hh * a.pool.k_head : vd + hh * a.pool.v_head;
    if constexpr (E4M3) {
      const float* sc = kind == 1 ? a.pool.kscale : a.pool.vscale;
      const double inv = sc ? 1.0 / sc[hh] : 1.0;
      *reinterpret_cast<uint2*>(y + 8 * c0) = narrow_e4m3(x0, inv);
      *reinterpret_cast<uint2*>(y + 8 * c1) = narrow_e4m3(x1, inv);
    } else {  // a value keeps its bits
      *reinterpret_cast<uint4*>(y + 16 * c0) = kind == 1 ? narrow<T>(x0) : r0;
      *reinterpret_cast<uint4*>(y + 16 * c1) = kind == 1 ? narrow<T>(x1) : r1;
    }
  }
}

template <class T, bool STORE, bool E4M3>
hipError_t go(const QkRopeArgs& a, hipStream_t s) {
  const int l = a.hd / 16, all = a.heads + (STORE ? 2 : 1) * a.kv_heads;
  const int per_row = ceil_div(all, 64 / l);
  // waves: at most 2^35 / 1024 elements' and one for each of 2^22 rows, and so below 2^32 threads
  const dim3 grid(ceil_div(a.seqs.rows * per_row, kThreads / 64)), block(kThreads);
  if (l == 4) hipLaunchKernelGGL((qk_rope_kernel<T, 4, STORE, E4M3>), grid, block, 0, s, a, per_row);
  else if (l == 8) hipLaunchKernelGGL((qk_rope_kernel<T, 8, STORE, E4M3>), grid, block, 0, s, a, per_row);
  else hipLaunchKernelGGL((qk_rope_kernel<T, 16, STORE, E4M3>), grid, block, 0, s, a, per_row);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_qk_rope(const QkRopeArgs& a, hipStream_t s) {
  if (!a.v) return a.dtype == KV_BF16 ? go<Bf16, false, false>(a, s) : go<Fp16, false, false>(a, s);
  if (a.pool.dtype == KV_E4M3) return a.dtype == KV_BF16 ? go<Bf16, true, true>(a, s) : go<Fp16, true, true>(a, s);
  return a.dtype == KV_BF16 ? go<Bf16, true, false>(a, s) : go<Fp16, true, false>(a, s);
}

}  // namespace tars
