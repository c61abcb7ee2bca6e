// Log probabilities of given tokens, the entropy and the top alternatives of rows of logits x, in one pass over them.
//
// With m the largest logit, S = sum e^(x - m) and T = sum (x - m) e^(x - m):  ln p = x - m - ln S,  H = ln S - T / S.
// Each lane keeps its own m, S and T and moves them to a new maximum m' once for each group of loads, by f = e^(m - m'):
// S' = f S, T' = f (T + (m - m') S); lanes, waves and parts of a row are joined by the same rule, in order. A logit of
// -infinity adds nothing; NaN and +infinity make S NaN, and with it every result of the row.
//
// The top alternatives are found by 64-bit keys: the logit's bits in an order that whole numbers keep (NaN last), above the place
// counted down, so that equal logits are in order of their places and no two keys are equal. The pass over the logits only notes,
// to 16 bits, the largest of each group of a lane's loads. The top-th largest of the lanes' maxima is a bound that at least `top`
// logits reach, and little more than that do: the few groups that reach it are fetched again, and the logits above the bound go to
// their wave's list in LDS. A list that fills up is cut to its largest `top`, the last of which is the wave's new bound. A key's
// place among the largest is the number of larger ones, counted over all lists at the end.
//
// A workgroup takes a row, or a part of one where there are few; a second launch joins the parts. 2048 rows of 151936 bf16 logits
// take 123 us, 5.1 TB/s. Smaller calls are chains of latencies (waves wait for half of their time, three quarters in the join): of
// the 20 us of 61 rows with 20 alternatives the sums alone take 10.5, the bound, the second look and the ranking the rest, which
// hardly goes by the size: 200 rows take 17.8 us without alternatives and 25.7 with five, one row 6.2 and 12.0.
#include <algorithm>

#include "kernels.h"
#include "paged_index.h"
#include "wave_reduce.h"

namespace tars {
namespace {

constexpr int kWaves = 4, kLoads = 4, kLanes = 64;
constexpr int kGroups = 32;  // of a lane's loads, whose maxima are noted
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

constexpr int kAtOnce = 4;                     // keys of a lane that are offered together
constexpr int kRoom = (1 + kAtOnce) * kLanes;  // of a wave's list: 64 and what may be offered
constexpr int kAhead = 8;                      // keys that a count fetches at once: lists end in as many zeros
struct Shared {
  Key keys[kWaves][kRoom + kAhead];
  Key all[kWaves * kLanes + kAhead];
  Key top[kLanes];
  uint16_t group[kGroups][kWaves * kLanes];
  uint32_t most[kWaves][kLanes];
  Key bound;
  int equal;
  int n[kWaves];
  float sums[kWaves][3];
};

// A wave's list of keys above its bound.
struct List {
  Key* keys;  // kRoom of them in LDS
  Key last = 0;
  int n = 0, top;
  // At most kAtOnce times between two calls of cut().
  __device__ __forceinline__ void take(Key k, bool in) {
    const int lane = threadIdx.x & 63;
    const uint64_t who = __ballot(in && k > last);
    const int at = __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(who >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(who), 0));
    if (who >> lane & 1) keys[n + at] = k;
    n += __popcll(who);
  }
  // Where the list has more than 64, keeps the largest `top`.
  __device__ __forceinline__ void cut() {
    if (n <= kLanes) return;
    const int lane = threadIdx.x & 63;
    Key a[kRoom / kLanes];
    int place[kRoom / kLanes];
    if (lane < kAhead) keys[n + lane] = 0;
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < kRoom / kLanes; ++i) {
      place[i] = top;
      if (kLanes * i >= n) continue;
      a[i] = lane + kLanes * i < n ? keys[lane + kLanes * i] : 0;
      place[i] = a[i] ? 0 : top;
#pragma unroll 1
      for (int k = 0; k < n; k += kAhead) {
        Key c[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) c[j] = keys[k + j];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) place[i] += c[j] > a[i];
      }
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < kRoom / kLanes; ++i)
      if (place[i] < top) keys[place[i]] = a[i];
    __builtin_amdgcn_wave_barrier();
    n = min(n, top);
    const Key end = keys[top - 1];
    last = static_cast<Key>(static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(end >> 32)))) << 32 |
           static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(end)));
  }
};

struct XF32 {
  static constexpr int kEach = 4;  // logits in 16 bytes
  static constexpr bool kWhole = false;  // whether the upper 16 bits are all of a logit
  static __device__ __forceinline__ float at(const uint32_t* w, int e) { return __uint_as_float(w[e]); }
  static __device__ __forceinline__ float one(const char* p) { return *reinterpret_cast<const float*>(p); }
};
struct XBf16 {
  static constexpr int kEach = 8;
  static constexpr bool kWhole = true;
  static __device__ __forceinline__ float at(const uint32_t* w, int e) {
    return __uint_as_float(e & 1 ? w[e / 2] & 0xFFFF0000u : w[e / 2] << 16);
  }
  static __device__ __forceinline__ float one(const char* p) {
    return __uint_as_float(static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(p)) << 16);
  }
};
struct XF16 {
  static constexpr int kEach = 8;
  static constexpr bool kWhole = false;
  static __device__ __forceinline__ float at(const uint32_t* w, int e) {
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[e / 2] >> (16 * (e & 1)))));
  }
  static __device__ __forceinline__ float one(const char* p) { return static_cast<float>(*reinterpret_cast<const _Float16*>(p)); }
};

__device__ __forceinline__ Sums over_wave(Sums a) {
  const auto with = [&](auto other) { a.join({other(a.m), other(a.s), other(a.t)}); };
  with([](float x) { return __int_as_float(dpp<kDppQuadXor1>(__float_as_int(x))); });
  with([](float x) { return __int_as_float(dpp<kDppQuadXor2>(__float_as_int(x))); });
  with([](float x) { return __int_as_float(dpp<kDppRowHalfMirror>(__float_as_int(x))); });
  with([](float x) { return __int_as_float(dpp<kDppRowMirror>(__float_as_int(x))); });
  with([](float x) { return __shfl_xor(x, 16); });
  with([](float x) { return __shfl_xor(x, 32); });
  return a;
}

// Whether the upper 16 of a logit's `ordered` bits are all of it: a bfloat16, or -infinity, which is much of a masked row.
template <class X>
__device__ __forceinline__ bool whole(uint32_t upper) {
  return X::kWhole || upper == ordered(-INFINITY) >> 16;
}

// The workgroup's bound, for every wave: the top-th largest of the lanes' maxima, to 16 bits of their `ordered` values (0: a lane
// without one); where more lanes than that are equal by those bits, by their whole keys (place() is where a lane has its maximum
// first).
template <class X, class F>
__device__ __forceinline__ Key bound_of(Shared& sh, uint32_t most, int top, F place) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const bool mine = wave == static_cast<int>((blockIdx.x + blockIdx.y) & (kWaves - 1));  // one wave's work, another's in each workgroup
  sh.most[wave][lane] = most >> 16;
  __syncthreads();
  if (mine) {
    uint32_t x[kWaves], v = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) x[w] = sh.most[w][lane];
    int reach = 0;
#pragma unroll
    for (uint32_t bit = 0x8000u; bit; bit >>= 1) {
      int count = 0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) count += __popcll(__ballot(x[w] >= (v | bit)));
      if (count >= top) v |= bit, reach = count;
    }
    if (lane == 0) {
      sh.bound = static_cast<Key>(v) << 48;
      sh.equal = v != 0 && reach > top + 24;
    }
  }
  __syncthreads();
  Key b = sh.bound;
  if (sh.equal) {
    sh.keys[wave][lane] = most ? static_cast<Key>(most) << 32 | static_cast<uint32_t>(~place()) : 0;
    __syncthreads();
    Key k[kWaves];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) k[w] = sh.keys[w][lane];
    const auto search = [&](Key from, Key to) __attribute__((always_inline)) {
#pragma unroll 1
      for (Key bit = from; bit >= to; bit >>= 1) {
        int count = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) count += __popcll(__ballot(k[w] >= (b | bit)));
        if (count >= top) b |= bit;
      }
    };
    // the logit's lower bits where it has any, then the place's 24: the bits above those are ones in every key
    if (whole<X>(static_cast<uint32_t>(b >> 48))) b |= b >> 48 & 0x8000u ? 0 : Key{0xFFFF} << 32;
    else search(Key{1} << 47, Key{1} << 32);
    b |= 0xFF000000u;
    search(Key{1} << 23, 1);
    __syncthreads();  // before the lists take the keys' room
  }
  return b ? b - 1 : 0;
}

// The waves' lists as one in sh.top, the largest key first, 0 behind the last; their sums joined.
__device__ __forceinline__ Sums over_workgroup(Shared& sh, Sums a, List& list) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (list.top) list.cut();
  a = over_wave(a);
  if (lane == 0) {
    sh.sums[wave][0] = a.m;
    sh.sums[wave][1] = a.s;
    sh.sums[wave][2] = a.t;
    sh.n[wave] = list.n;
  }
  if (wave == 0) sh.top[lane] = 0;
  __syncthreads();
  if (list.top) {
    int first = 0, n = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      first += w < wave ? sh.n[w] : 0;
      n += sh.n[w];
    }
    if (lane < list.n) sh.all[first + lane] = list.keys[lane];
    if (wave == 0 && lane < kAhead) sh.all[n + lane] = 0;
    __syncthreads();
    const int t = threadIdx.x;
    if (64 * wave < n) {
      const Key mine = t < n ? sh.all[t] : 0;
      int place = 0;
#pragma unroll 1
      for (int k = 0; k < n; k += kAhead) {
        Key c[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) c[i] = sh.all[k + i];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) place += c[i] > mine;
      }
      if (mine && place < list.top) sh.top[place] = mine;
    }
  }
  Sums all{sh.sums[0][0], sh.sums[0][1], sh.sums[0][2]};
#pragma unroll
  for (int w = 1; w < kWaves; ++w) all.join({sh.sums[w][0], sh.sums[w][1], sh.sums[w][2]});
  __syncthreads();
  return all;
}

// The logit of the row's i-th given token; `in`: whether it has one.
struct Given {
  float x;
  bool in;
};
template <class X>
__device__ __forceinline__ Given given_at(const LogprobArgs& a, int row, int i) {
  if (i >= a.given) return {0, false};
  const char* tokens = static_cast<const char*>(a.tokens) + row * a.ld_tokens;
  const int64_t t = a.wide_tokens ? reinterpret_cast<const int64_t*>(tokens)[i] : reinterpret_cast<const int32_t*>(tokens)[i];
  const bool in = t >= 0 && t < a.vocab;
  return {in ? X::one(a.x + row * a.ld + t * (16 / X::kEach)) : 0.0f, in};
}

// The row's results; `first` is the thread's first given token, fetched before its value is needed.
template <class X>
__device__ __forceinline__ void answer(const LogprobArgs& a, const Shared& sh, Sums all, int row, Given first) {
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
  for (int i = threadIdx.x; i < a.given; i += blockDim.x) {
    a.logprobs[static_cast<int64_t>(row) * a.given + i] = first.in ? lp(first.x) : -INFINITY;
    first = given_at<X>(a, row, i + blockDim.x);
  }
}

__device__ __forceinline__ char* part_at(const LogprobArgs& a, int row, int part) {
  return static_cast<char*>(a.work) + (static_cast<int64_t>(row) * a.parts + part) * logprobs_part_bytes(a.top);
}

template <class X, bool TOP>
__global__ __launch_bounds__(64 * kWaves, 4) void logprobs_kernel(LogprobArgs a) {
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
  List list{sh.keys[wave]};
  list.top = TOP ? a.top : 0;
  // the logits around the pieces
  const bool edge = part == 0 && wave == 0 && lane < head + tail;
  const int edge_at = lane < head ? lane : a.vocab - tail + lane - head;
  const float edge_v = edge ? X::one(x + static_cast<int64_t>(edge_at) * kSize) : -INFINITY;
  if (edge) {
    sums.move(fmaxf(sums.m, edge_v));
    sums.add(edge_v);
  }
  const auto load = [&](int p, uint4 (&w)[kLoads]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) w[i] = *reinterpret_cast<const uint4*>(body + 16ll * min(p + 64 * i + lane, p1 - 1));
  };
  const auto unpack = [&](int p, const uint4 (&w)[kLoads], float (&v)[kLoads][kEach]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const uint32_t word[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
      for (int e = 0; e < kEach; ++e) v[i][e] = X::at(word, e);
    }
    if (p + 64 * kLoads > p1)
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
#pragma unroll
        for (int e = 0; e < kEach; ++e) v[i][e] = p + 64 * i + lane < p1 ? v[i][e] : -INFINITY;
  };
  const int steps = ceil_div(share, 64 * kLoads), stride = ceil_div(steps, kGroups);  // steps of a wave, and of a group
  float most = -INFINITY, in_group = -INFINITY;
  uint4 w[kLoads];
  if (p0 < p1) load(p0, w);
  int left = stride, group = 0;
  for (int p = p0; p < p1; p += 64 * kLoads) {
    float v[kLoads][kEach], here = -INFINITY;
    unpack(p, w, v);
    if (p + 64 * kLoads < p1) load(p + 64 * kLoads, w);
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
#pragma unroll
      for (int e = 0; e < kEach; ++e) here = fmaxf(here, v[i][e]);
    sums.move(fmaxf(sums.m, here));
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
#pragma unroll
      for (int e = 0; e < kEach; ++e) sums.add(v[i][e]);
    if constexpr (TOP) {
      in_group = fmaxf(in_group, here);
      if (--left == 0 || p + 64 * kLoads >= p1) {
        // a maximum passes NaN by; the sum does not
        sh.group[group][threadIdx.x] = static_cast<uint16_t>(sums.s != sums.s ? 0xFFFF : ordered(in_group) >> 16);
        most = fmaxf(most, in_group);
        in_group = -INFINITY;
        left = stride;
        ++group;
      }
    }
  }
  if constexpr (TOP) {
    const auto at_of = [&](int p, int i, int e) { return head + (p + 64 * i + lane) * kEach + e; };
    const bool any = p0 + lane < p1;
    list.last = bound_of<X>(sh, any ? ordered(most) : 0, a.top, [&]() {  // where the lane has its maximum first
      int at = a.vocab - 1;
#pragma unroll 1
      for (int p = p0; __ballot(any && at == a.vocab - 1) && p < p1; p += 64 * kLoads) {
        load(p, w);
        float v[kLoads][kEach];
        unpack(p, w, v);
#pragma unroll
        for (int i = kLoads; i-- > 0;)
#pragma unroll
          for (int e = kEach; e-- > 0;) at = v[i][e] == most && p + 64 * i + lane < p1 ? min(at, at_of(p, i, e)) : at;
      }
      return at;
    });
    list.take(key_of(edge_v, edge_at), edge);
    // The groups that reach the bound. Where its 16 bits are all of a logit, a group that equals them and lies behind the bound's
    // own place does not.
    const uint32_t line = static_cast<uint32_t>((list.last + 1) >> 48), least_at = ~static_cast<uint32_t>(list.last + 1);
    const bool all_bits = whole<X>(line);
    uint32_t groups = 0;
    for (int k = 0; k < group; ++k) {
      const uint32_t g = sh.group[k][threadIdx.x];
      const bool before = !all_bits || static_cast<uint32_t>(at_of(p0 + k * stride * 64 * kLoads, 0, 0)) <= least_at;
      groups |= static_cast<uint32_t>(g > line || (g == line && before)) << k;
    }
#pragma unroll 1
    for (uint32_t all = any ? groups : 0; __ballot(all != 0); all &= all - 1) {
      const int k = all ? __builtin_ctz(all) : 0;
#pragma unroll 1
      for (int j = 0; j < stride; ++j) {  // each lane its own group
        const int p = p0 + (k * stride + j) * 64 * kLoads;
        load(p, w);
        float v[kLoads][kEach];
        unpack(p, w, v);
        // a bit for each logit whose key may be the bound's next or above: of those equal to its logit only the places up to its own
        const Key next = list.last + 1;
        const float least = value_of(static_cast<uint32_t>(next >> 32));  // NaN at either end: all may be
        const int upto = static_cast<int>(min(~static_cast<uint32_t>(next), 0x7FFFFFFEu)) + 1;
        uint32_t may = 0;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          uint32_t up = 0, eq = 0;
#pragma unroll
          for (int e = 0; e < kEach; ++e) {
            up |= static_cast<uint32_t>(!(v[i][e] <= least)) << e;
            eq |= static_cast<uint32_t>(v[i][e] == least) << e;
          }
          const bool in = all != 0 && p + 64 * i + lane < p1;
          may |= in ? (up | (eq & ((1u << iclamp(upto - at_of(p, i, 0), 0, kEach)) - 1))) << (i * kEach) : 0;
        }
#pragma unroll 1
        while (__ballot(may != 0)) {
          list.cut();
#pragma unroll
          for (int u = 0; u < kAtOnce; ++u) {
            const int b = may ? __builtin_ctz(may) : 0, at = at_of(min(p + 64 * (b / kEach), p1 - 1 - lane), 0, 0) + b % kEach;
            const float again = X::one(x + static_cast<int64_t>(may ? at : 0) * kSize);
            list.take(key_of(again, at), may != 0);
            may &= may - 1;
          }
        }
      }
    }
  }
  const Given first = a.parts == 1 ? given_at<X>(a, row, threadIdx.x) : Given{0, false};
  const Sums all = over_workgroup(sh, sums, list);
  if (a.parts == 1) {
    answer<X>(a, sh, all, row, first);
    return;
  }
  char* to = part_at(a, row, part);
  if (threadIdx.x == 0) *reinterpret_cast<float4*>(to) = make_float4(all.m, all.s, all.t, 0);
  if (static_cast<int>(threadIdx.x) < a.top) reinterpret_cast<Key*>(to + 16)[threadIdx.x] = sh.top[threadIdx.x];
}

template <class X>
__global__ __launch_bounds__(64 * kWaves) void logprobs_join_kernel(LogprobArgs a) {
  __shared__ Shared sh;
  const int row = blockIdx.x, wave = threadIdx.x >> 6;
  const Given first = given_at<X>(a, row, threadIdx.x);
  Sums sums = Sums::none();
  for (int p = threadIdx.x; p < a.parts; p += 64 * kWaves) {
    const float4 v = *reinterpret_cast<const float4*>(part_at(a, row, p));
    sums.join({v.x, v.y, v.z});
  }
  List list{sh.keys[wave]};
  list.top = a.top;
  if (a.top) {
    const int n = a.parts * a.top;
    for (int base = 0; base < n; base += 64 * kWaves) {
      const int at = base + threadIdx.x, k = at / a.parts;  // the parts' largest first
      const bool in = at < n;
      const Key key = in ? reinterpret_cast<const Key*>(part_at(a, row, at - k * a.parts) + 16)[k] : 0;
      if (base == 0) list.last = bound_of<X>(sh, static_cast<uint32_t>(key >> 32), a.top, [&]() { return static_cast<int>(~static_cast<uint32_t>(key)); });
      list.cut();
      list.take(key, in);
    }
  }
  const Sums all = over_workgroup(sh, sums, list);
  answer<X>(a, sh, all, row, first);
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

// Parts of a row, by what they would take: the steps of 16 KiB that the workgroups of the fullest CU take, and half a one for each
// workgroup (0.62 us a step, 0.72 where there is one workgroup to a CU), and 6 us for the join and its launch. Measured with five alternatives: 64 and 128 rows of
// 151936 bf16 logits 18.4 and 22.1 us in four parts, 24.3 and 24.8 whole; 200 and 400 rows 25.2 and 35.3 us whole, 28 and 41 in
// parts; 100 rows of 32000 11.5 us whole, 13.5 in parts.
int logprobs_parts(int rows, int vocab, int dtype) {
  const int steps = ceil_div(std::max(1, vocab / (dtype == 0 ? 4 : 8)), 64 * kLoads * kWaves);
  int64_t best = 0;
  int parts = 1;
  for (int want = 1;; want = want & (want - 1) ? want / 3 * 4 : want == 1 ? 2 : want / 2 * 3) {
    const int each = ceil_div(steps, std::min(want, steps)), p = ceil_div(steps, each);
    const int64_t on_a_cu = (static_cast<int64_t>(rows) * p + 255) / 256, time = (2 * each + 1) * (on_a_cu == 1 ? 36 : 31 * on_a_cu) + (p > 1 ? 600 : 0);
    if (want == 1 || time < best) best = time, parts = p;
    if (want >= steps) return parts;
  }
}

hipError_t launch_logprobs(const LogprobArgs& a, hipStream_t s) {
  return a.dtype == 0 ? go<XF32>(a, s) : a.dtype == 1 ? go<XBf16>(a, s) : go<XF16>(a, s);
}

}  // namespace tars
