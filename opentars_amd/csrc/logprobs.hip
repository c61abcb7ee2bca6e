// Log probabilities of given tokens, the entropy and the top alternatives of rows of logits x, in one pass over them.
//
// With m the largest logit, S = sum e^(x - m) and T = sum (x - m) e^(x - m):  ln p = x - m - ln S,  H = ln S - T / S.
// Each lane keeps its own m, S and T and moves them to a new maximum m' once for each group of loads, by f = e^(m - m'):
// S' = f S, T' = f (T + (m - m') S); lanes, waves and parts of a row are joined by the same rule, in order. A logit of
// -infinity adds nothing; NaN and +infinity make S NaN, and with it every result of the row.
//
// The top alternatives are kept for each wave as a sorted list of 64-bit keys, one to a lane: the logit's bits in an order that
// whole numbers keep (NaN last), above the place counted down, so that equal logits are in order of their places and no two keys
// are equal. A logit below the list's last is passed by with one comparison; the first group of loads is filtered by the top-th
// largest of the lanes' maxima.
#include <algorithm>

#include "kernels.h"
#include "paged_index.h"

namespace tars {
namespace {

constexpr int kWaves = 4, kLoads = 4, kLanes = 64;
constexpr float kLog2e = 1.44269504f, kFar = -1e4f;  // e^kFar is 0 in fp32

struct Sums {
  float m, s, t;
  static __device__ __forceinline__ Sums none() { return {-3.402823466e38f, 0, 0}; }
  __device__ __forceinline__ void move(float to) {
    const float d = fmaxf(m - to, kFar), f = __builtin_amdgcn_exp2f(d * kLog2e);
    t = f * (t + d * s);
    s *= f;
    m = to;
  }
  __device__ __forceinline__ void add(float x) {
    const float d = x - m, e = __builtin_amdgcn_exp2f(d * kLog2e);
    s += e;
    t += fmaxf(d, kFar) * e;
  }
  __device__ __forceinline__ void join(Sums o) {
    const float to = fmaxf(m, o.m);
    move(to);
    o.move(to);
    s += o.s;
    t += o.t;
  }
};

using Key = unsigned long long;
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);  // -0 is 0
  return x != x ? 0xFFFFFFFFu : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o); }
__device__ __forceinline__ Key key_of(float x, uint32_t at) { return static_cast<Key>(ordered(x)) << 32 | static_cast<uint32_t>(~at); }
__device__ __forceinline__ Key lane_key(Key k, int lane) {
  return static_cast<Key>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(k >> 32), lane))) << 32 |
         static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(k), lane));
}

// A wave's largest keys, lane i the i-th; 0 where there is none.
struct List {
  Key mine = 0, last = 0;  // last: the top-th, or a bound below which nothing counts
  __device__ __forceinline__ void take(Key k, bool in, int top) {
    const int lane = threadIdx.x & 63;
    uint64_t todo = __ballot(in && k > last);
    while (todo) {
      const Key c = lane_key(k, __builtin_ctzll(todo));
      const int at = __popcll(__ballot(mine > c));
      const Key up = static_cast<Key>(static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(mine >> 32), 0x138, 0xF, 0xF, false))) << 32 |
                     static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(mine), 0x138, 0xF, 0xF, false));  // the lane before's
      mine = lane < at ? mine : lane == at ? c : up;
      const Key end = lane_key(mine, top - 1);
      last = end > last ? end : last;
      todo &= todo - 1;
      todo &= __ballot(k > last);
    }
  }
};

// The n-th largest of the lanes' values.
__device__ __forceinline__ uint32_t nth_of(uint32_t x, int n) {
  uint32_t v = 0;
#pragma unroll 1
  for (uint32_t bit = 0x80000000u; bit; bit >>= 1)
    if (__popcll(__ballot(x >= (v | bit))) >= n) v |= bit;
  return v;
}

struct XF32 {
  static constexpr int kEach = 4;  // logits in 16 bytes
  static __device__ __forceinline__ float at(const uint32_t* w, int e) { return __uint_as_float(w[e]); }
  static __device__ __forceinline__ float one(const char* p) { return *reinterpret_cast<const float*>(p); }
};
struct XBf16 {
  static constexpr int kEach = 8;
  static __device__ __forceinline__ float at(const uint32_t* w, int e) {
    return __uint_as_float(e & 1 ? w[e / 2] & 0xFFFF0000u : w[e / 2] << 16);
  }
  static __device__ __forceinline__ float one(const char* p) {
    return __uint_as_float(static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(p)) << 16);
  }
};
struct XF16 {
  static constexpr int kEach = 8;
  static __device__ __forceinline__ float at(const uint32_t* w, int e) {
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[e / 2] >> (16 * (e & 1)))));
  }
  static __device__ __forceinline__ float one(const char* p) { return static_cast<float>(*reinterpret_cast<const _Float16*>(p)); }
};

__device__ __forceinline__ Sums over_wave(Sums a) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    a.join({__shfl_xor(a.m, d), __shfl_xor(a.s, d), __shfl_xor(a.t, d)});
  }
  return a;
}

struct Shared {
  Key keys[kWaves][kLanes];
  Key top[kLanes];
  Sums sums[kWaves];
};

// The waves' lists as one in sh.top: a key's place is its own list's and the number of larger ones in each other. The waves' sums joined.
__device__ __forceinline__ Sums over_workgroup(Shared& sh, Sums a, Key mine, int top) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  a = over_wave(a);
  if (lane == 0) sh.sums[wave] = a;
  if (top) {
    sh.keys[wave][lane] = mine;
    if (wave == 0) sh.top[lane] = 0;
  }
  __syncthreads();
  if (top && lane < top) {
    int place = lane;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) {
      const Key* other = sh.keys[(wave + w) % kWaves];
      int n = 0;  // the first ones are larger
#pragma unroll
      for (int step = 32; step; step /= 2)
        if (other[n + step - 1] > mine) n += step;
      if (n == 63 && other[63] > mine) n = 64;
      place += n;
    }
    if (mine && place < top) sh.top[place] = mine;
  }
  Sums all = sh.sums[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) all.join(sh.sums[w]);
  __syncthreads();
  return all;
}

template <class X>
__device__ __forceinline__ void answer(const LogprobArgs& a, const Shared& sh, Sums all, int row) {
  const bool none = all.s == 0;
  const double log_s = none ? 0.0 : ::log(static_cast<double>(all.s));  // once a row: in 64 bits
  const auto lp = [&](float x) { return none ? -INFINITY : static_cast<float>(static_cast<double>(x) - all.m - log_s); };
  if (threadIdx.x == 0) {
    const float h = none ? 0.0f : static_cast<float>(log_s - static_cast<double>(all.t) / all.s);
    a.entropy[row] = h < 0 ? 0.0f : h;
  }
  if (static_cast<int>(threadIdx.x) < a.top) {
    const Key k = sh.top[threadIdx.x];
    a.top_values[static_cast<int64_t>(row) * a.top + threadIdx.x] = lp(value_of(static_cast<uint32_t>(k >> 32)));
    a.top_ids[static_cast<int64_t>(row) * a.top + threadIdx.x] = static_cast<int32_t>(~static_cast<uint32_t>(k));
  }
  const char* tokens = static_cast<const char*>(a.tokens) + row * a.ld_tokens;
  for (int i = threadIdx.x; i < a.given; i += blockDim.x) {
    const int64_t t = a.wide_tokens ? reinterpret_cast<const int64_t*>(tokens)[i] : reinterpret_cast<const int32_t*>(tokens)[i];
    const bool in = t >= 0 && t < a.vocab;
    a.logprobs[static_cast<int64_t>(row) * a.given + i] =
        in ? lp(X::one(a.x + row * a.ld + t * (16 / X::kEach))) : -INFINITY;
  }
}

__device__ __forceinline__ char* part_at(const LogprobArgs& a, int row, int part) {
  return static_cast<char*>(a.work) + (static_cast<int64_t>(row) * a.parts + part) * logprobs_part_bytes(a.top);
}

template <class X, bool TOP>
__global__ __launch_bounds__(64 * kWaves) void logprobs_kernel(LogprobArgs a) {
  __shared__ Shared sh;
  constexpr int kEach = X::kEach, kSize = 16 / kEach;
  const int row = blockIdx.y + blockIdx.z * 65535, part = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (row >= a.rows) return;
  const char* x = a.x + row * a.ld;
  // whole 16-byte pieces from `head` logits on; the few before and behind them are one wave's extra load
  const int head = min(static_cast<int>(-reinterpret_cast<uintptr_t>(x) % 16) / kSize, a.vocab);
  const int pieces = (a.vocab - head) / kEach, tail = a.vocab - head - pieces * kEach;
  const char* body = x + head * kSize;
  const int share = ceil_div(ceil_div(pieces, a.parts * kWaves), 64) * 64;
  const int p0 = min(pieces, (part * kWaves + wave) * share), p1 = min(pieces, p0 + share);
  Sums sums = Sums::none();
  List list;
  if (part == 0 && wave == 0 && head + tail > 0) {
    const bool in = lane < head + tail;
    const int at = lane < head ? lane : a.vocab - tail + lane - head;
    const float v = in ? X::one(x + static_cast<int64_t>(at) * kSize) : -INFINITY;
    if (in) {
      sums.move(fmaxf(sums.m, v));
      sums.add(v);
    }
    if constexpr (TOP) list.take(key_of(v, at), in, a.top);
  }
  bool first = true;
  for (int p = p0; p < p1; p += 64 * kLoads) {
    uint32_t w[kLoads][4];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int q = p + 64 * i + lane;
      const uint4 v = *reinterpret_cast<const uint4*>(body + 16ll * min(q, p1 - 1));
      w[i][0] = v.x;
      w[i][1] = v.y;
      w[i][2] = v.z;
      w[i][3] = v.w;
    }
    float v[kLoads][kEach], most = -INFINITY;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const bool in = p + 64 * i + lane < p1;
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        v[i][e] = in ? X::at(w[i], e) : -INFINITY;
        most = fmaxf(most, v[i][e]);
      }
    }
    sums.move(fmaxf(sums.m, most));
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
#pragma unroll
      for (int e = 0; e < kEach; ++e) sums.add(v[i][e]);
    if constexpr (TOP) {
      if (first) {  // at least `top` logits reach the top-th largest maximum, where that many lanes have one
        const uint32_t bound = nth_of(p + lane < p1 ? ordered(most) : 0, a.top);
        if (bound) {
          const Key below = (static_cast<Key>(bound) << 32) - 1;
          list.last = below > list.last ? below : list.last;
        }
        first = false;
      }
      const float least = value_of(static_cast<uint32_t>(list.last >> 32));
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int q = p + 64 * i + lane;
#pragma unroll
        for (int e = 0; e < kEach; ++e)
          if (__ballot(list.last == 0 || !(v[i][e] < least))) list.take(key_of(v[i][e], head + q * kEach + e), q < p1, a.top);
      }
    }
  }
  const Sums all = over_workgroup(sh, sums, list.mine, TOP ? a.top : 0);
  if (a.parts == 1) {
    answer<X>(a, sh, all, row);
    return;
  }
  char* to = part_at(a, row, part);
  if (threadIdx.x == 0) *reinterpret_cast<float4*>(to) = make_float4(all.m, all.s, all.t, 0);
  if (static_cast<int>(threadIdx.x) < a.top) reinterpret_cast<Key*>(to + 16)[threadIdx.x] = sh.top[threadIdx.x];
}

template <class X>
__global__ __launch_bounds__(64 * kWaves) void logprobs_join_kernel(LogprobArgs a) {
  __shared__ Shared sh;
  const int row = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Sums sums = Sums::none();
  for (int p = threadIdx.x; p < a.parts; p += 64 * kWaves) {
    const float4 v = *reinterpret_cast<const float4*>(part_at(a, row, p));
    sums.join({v.x, v.y, v.z});
  }
  List list;
  if (a.top)
    for (int i = 64 * wave; i < a.parts * a.top; i += 64 * kWaves) {
      const int at = i + lane, k = at / a.parts;  // the parts' largest first
      const bool in = at < a.parts * a.top;
      const Key key = in ? reinterpret_cast<const Key*>(part_at(a, row, at - k * a.parts) + 16)[k] : 0;
      list.take(key, in, a.top);
    }
  const Sums all = over_workgroup(sh, sums, list.mine, a.top);
  answer<X>(a, sh, all, row);
}

template <class X>
hipError_t go(const LogprobArgs& a, hipStream_t s) {
  const dim3 grid(a.parts, std::min(a.rows, 65535), ceil_div(a.rows, 65535)), block(64 * kWaves);
  if (a.top) hipLaunchKernelGGL((logprobs_kernel<X, true>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((logprobs_kernel<X, false>), grid, block, 0, s, a);
  if (a.parts > 1) hipLaunchKernelGGL(logprobs_join_kernel<X>, dim3(a.rows), block, 0, s, a);
  return hipGetLastError();
}

}  // namespace

// Parts of a row: enough workgroups for the card where there are few rows, 16 KiB of logits each at least.
int logprobs_parts(int rows, int vocab, int dtype) {
  const int64_t bytes = static_cast<int64_t>(vocab) * (dtype == 0 ? 4 : 2);
  const int64_t most = std::max<int64_t>(1, bytes >> 14), want = std::max(1, 1024 / rows);
  return static_cast<int>(std::min(most, want));
}

hipError_t launch_logprobs(const LogprobArgs& a, hipStream_t s) {
  return a.dtype == 0 ? go<XF32>(a, s) : a.dtype == 1 ? go<XBf16>(a, s) : go<XF16>(a, s);
}

}  // namespace tars
