// Attention of one row per sequence over the paged cache, split over the caches' lengths and joined.
//
// Per sequence and K / V head the cache is read once for all the query heads that share it, 32 positions a step. Both
// products run on matrix instructions with the positions as rows, so that nothing passes through LDS on the way:
//   S^T = K Q^T   16 positions x 16 heads: lane l loads row l % 16 of K, 16 bytes of it, as the instruction wants it;
//   O^T += V^T P^T  lane l loads the rows of V at the very positions whose scores it holds (16 t + 4 (l / 16) + i of
//                 the step), hd / 16 columns of each: its block of 8 positions x hd / 16 columns, turned over by
//                 v_perm_b32 in its own registers, is V^T's operand for hd / 16 products, and its 8 numerators, in
//                 the order they left the softmax, are P^T's.
// The order of a product's inner index is free as long as both operands use it, which is all this needs. A numerator
// goes in as the sum of two values of q's type (its rounding and what that left), two products instead of one: next to
// the loads they are free, and the result is rounded once, at the end.
//
// The running maximum is kept per head; accumulators are rescaled only when it grows, which after a few steps is rare.
// Positions that the row does not see get a numerator of 0 and zeros for V (which may hold anything there). Only steps
// at the end of the cache, at the window's edges or with a page number outside the pool pay for that.
//
// The split is made on the device from the lengths: every workgroup adds up the steps of all sequences, sets the share
// C of a workgroup so that the shares fill the GPU, and finds its own (sequence, part) in the prefix sums. So one long
// cache fills the GPU as well as many short ones, whatever the batch's longest is. A sequence of one part is written
// at once; the parts of the others go to the workspace as (maximum, sum, unscaled output) in fp32 and a second launch
// joins them in order.
#include <algorithm>

#include "paged_device.h"

namespace tars {
namespace {

// Positions that a wave takes at a time: 16 for heads of 256, whose K and V rows fill the registers.
constexpr int step_of(int hd) { return hd == 256 ? 16 : 32; }
constexpr int kWaves = 4;
constexpr int kHeads = 16;       // query heads of a workgroup
constexpr int kSlots = 1536;     // workgroups that long work is dealt to: two rounds of the three on every CU
constexpr int kFew = 512;        // and short work, in shares of kLeast to kShort positions: one round
constexpr int kLeast = 64, kShort = 512;

// The sequences' steps dealt to workgroups: `slots` shares for each K / V head (and head tile).
struct Deal {
  int slots, few;        // workgroups for a K / V head and head tile, of long and of short work
  int least, most_few;   // steps
};
struct Part {
  int b, part, parts, first;     // the sequence, its part's number and count, the number of its first part among all
  int len;
  Steps steps;
};

template <int STEP>
__device__ __forceinline__ Steps steps_of(int len, int window, int sinks) {
  return visible_steps(len - 1, len - 1, len, window, sinks, STEP);
}

// The share C of a workgroup, the same in every wave.
template <int STEP>
__device__ __forceinline__ int share(const KvSeqs& s, int window, int sinks, const Deal& deal) {
  const int lane = threadIdx.x & 63;
  uint64_t mine = 0;
  for (int b = lane; b < s.seqs; b += 64) mine += steps_of<STEP>(seq_len(s.lens, b, s.cap), window, sinks).n();
  const uint64_t lo = group_sum<64>(static_cast<int>(mine & 0xFFFFFF)), hi = group_sum<64>(static_cast<int>(mine >> 24));
  const uint64_t total = lo + (hi << 24);
  // in units of 2^16 steps where the sum has more than 31 bits (a share too long is no harm)
  const int up = total < (1ull << 31) ? 0 : 16;
  const uint32_t units = static_cast<uint32_t>((total + (1ull << up) - 1) >> up);
  const auto per = [&](uint32_t slots) { return min((units + slots - 1) / slots, 1u << 25 >> up) << up; };
  const int c = max(static_cast<int>(per(deal.slots)), min(static_cast<int>(per(deal.few)), deal.most_few));
  return max(c, deal.least);  // no sequence has more than 2^25 steps
}

__device__ __forceinline__ int parts_of(int n, int c) { return max((n + c - 1) / c, 1); }

__device__ __forceinline__ int inclusive_sum(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);  // row_shr 1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // row_bcast 15 to rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // row_bcast 31 to rows 2 and 3
  return x;
}

// The part numbered idx among all (b < 0: none).
template <int STEP>
__device__ __forceinline__ Part find_part(const KvSeqs& s, int window, int sinks, int c, int idx) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int b0 = 0; b0 < s.seqs; b0 += 64) {
    const int b = b0 + lane;
    const int len = b < s.seqs ? seq_len(s.lens, b, s.cap) : 0;
    const int parts = b < s.seqs ? parts_of(steps_of<STEP>(len, window, sinks).n(), c) : 0;
    const int upto = before + inclusive_sum(parts);
    const uint64_t hit = __ballot(upto > idx);
    if (hit) {
      const int at = __builtin_ctzll(hit);
      Part p;
      p.b = b0 + at;
      p.len = __builtin_amdgcn_readlane(len, at);
      p.parts = __builtin_amdgcn_readlane(parts, at);
      p.first = __builtin_amdgcn_readlane(upto, at) - p.parts;
      p.part = idx - p.first;
      p.steps = steps_of<STEP>(p.len, window, sinks);
      return p;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }
  return {-1, 0, 0, 0, 0, {}};
}

__device__ __forceinline__ uint32_t perm(uint32_t hi, uint32_t lo, uint32_t sel) { return __builtin_amdgcn_perm(hi, lo, sel); }

template <class T>
__device__ __forceinline__ v4f mfma16(const uint32_t (&a)[4], const uint32_t (&b)[4], v4f c) {
  const uint4 x = make_uint4(a[0], a[1], a[2], a[3]), y = make_uint4(b[0], b[1], b[2], b[3]);
  return T::mfma_16x16x32(x, y, c);
}
template <class T>
__device__ __forceinline__ v4f mfma16(const uint32_t (&a)[2], const uint32_t (&b)[2], v4f c) {
  return T::mfma_16x16x16(make_uint2(a[0], a[1]), make_uint2(b[0], b[1]), c);
}

// N dwords from global memory, read once: a scalar base and a lane offset; past four, FAR bytes from one four to the next.
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
template <int FAR, int N>
__device__ __forceinline__ void load_dwords(uint32_t (&d)[N], const char* base, uint32_t off) {
  if constexpr (N == 1) {
    d[0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(base + off));
  } else if constexpr (N == 2) {
    const v2u v = __builtin_nontemporal_load(reinterpret_cast<const v2u*>(base + off));
    d[0] = v[0];
    d[1] = v[1];
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const v4u v = __builtin_nontemporal_load(reinterpret_cast<const v4u*>(base + off + FAR * (i / 4)));
#pragma unroll
      for (int j = 0; j < 4; ++j) d[i + j] = v[j];
    }
  }
}

__device__ __forceinline__ float max_over_groups(float x) {  // over lanes l % 16
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_over_groups(float x) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The two pages of a step and whether they are in the pool (bit t), the same in every lane.
struct Pages {
  int page[2];
  int ok;
};

// The workspace: (first part, parts) of every sequence, then every part's rows.
__host__ __device__ __forceinline__ int64_t head_bytes(int seqs) { return (8ll * seqs + 15) / 16 * 16; }
__device__ __forceinline__ float* parts_at(const PagedAttnArgs& a) { return a.work + head_bytes(a.seqs.seqs) / 4; }

template <class T, bool E4M3, int D>
__global__ __launch_bounds__(64 * kWaves, 2) void paged_decode_kernel(PagedAttnArgs a, Deal deal, int head_tiles) {
  constexpr int KS = D / 32;                        // products of a scores tile
  constexpr int E = D / 16;                         // columns of V per lane
  constexpr int KW = E4M3 ? 4 * KS / 2 : 4 * KS;    // dwords of a lane's K row part
  constexpr int VW = E4M3 ? E / 4 : E / 2;          // dwords of a lane's V row part
  constexpr int C = VW == 8 ? 8 : E;                // its neighbouring columns: two runs of 8 for 16-bit rows of 256
  constexpr int kPad = D + 4;
  constexpr int kStep = step_of(D), kTiles = kStep / 16, NK = kStep / 4;  // NK: positions of a lane
  __shared__ __attribute__((aligned(16))) float os[kWaves / 2][kHeads][kPad];
  __shared__ float ms[kWaves][kHeads], ls[kWaves][kHeads];
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = share<step_of(D)>(a.seqs, a.window, a.sinks, deal);
  const int columns = a.pool.kv_heads * head_tiles, number = blockIdx.x / columns, column = blockIdx.x % columns;
  const Part part = find_part<step_of(D)>(a.seqs, a.window, a.sinks, c, number);
  if (part.b < 0) return;
  const int h = column / head_tiles, tile = column % head_tiles;
  const int heads = min(a.group - tile * kHeads, kHeads);   // of this workgroup
  const int head0 = h * a.group + tile * kHeads;
  const int n = part.steps.n(), per = (n + part.parts - 1) / part.parts;
  const int t0 = part.part * per, t1 = min(n, t0 + per);
  const int lo = a.window == 0 ? 0 : max(part.len - a.window, 0);

  // Q^T: column = head. Heads of 256 keep it in LDS (every wave's own copy, 16 bytes of a lane at a time), where the
  // registers are needed for K and V.
  constexpr bool kQLds = D == 256;
  uint32_t qf[kQLds ? 1 : KS][4];
  const char* q = a.q + part.b * a.ldq + 2 * D * (head0 + min(col, heads - 1));
  char* qs = reinterpret_cast<char*>(os) + 1024 * KS * wave + 16 * lane;
  static_assert(!kQLds || 1024 * KS * kWaves <= sizeof(os), "Q's copies fit the rows that join the waves");
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    load_dwords<16>(qf[kQLds ? 0 : s], q, E4M3 ? 128 * (s / 2) + 16 * (s % 2) + 32 * g : 64 * s + 16 * g);
    if constexpr (kQLds) *reinterpret_cast<uint4*>(qs + 1024 * s) = make_uint4(qf[0][0], qf[0][1], qf[0][2], qf[0][3]);
  }
  const float sc = a.scale * 1.44269504f * (E4M3 && a.pool.kscale ? a.pool.kscale[h] : 1.0f);

  const int shift = a.pool.page_shift, mask = (1 << shift) - 1, last = (part.len - 1) >> shift;
  const __attribute__((address_space(4))) int32_t* table = reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(
      reinterpret_cast<uintptr_t>(a.seqs.table + part.b * a.seqs.ld_table));
  const uint32_t koff = col * static_cast<uint32_t>(a.pool.k_slot) + 16 * g;
  const uint32_t voff = 4 * g * static_cast<uint32_t>(a.pool.v_slot) + 4 * (VW < 4 ? VW : 4) * col;
  const char* kbase = a.pool.k + h * a.pool.k_head;
  const char* vbase = a.pool.v + h * a.pool.v_head;
  auto pages_of = [&](int i) {
    const int k0 = part.steps.at(i) * kStep;
    Pages p;
    p.page[0] = table[min(k0 >> shift, last)];
    p.page[1] = kTiles == 2 ? table[min((k0 + 16) >> shift, last)] : 0;
    return p;
  };
  auto check = [&](Pages& p) {
    p.ok = 0;
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      const bool in = static_cast<uint32_t>(p.page[t]) < static_cast<uint32_t>(a.pool.pages);
      p.ok |= in << t;
      p.page[t] = in ? p.page[t] : 0;
    }
  };
  uint32_t kf[kTiles][KW], vf[NK][VW];
  auto load_k = [&](int i, const Pages& p) {
    const int k0 = part.steps.at(i) * kStep;
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      const char* base = kbase + p.page[t] * a.pool.k_page + ((k0 + 16 * t) & mask) * a.pool.k_slot;
#pragma unroll
      for (int s = 0; s < KW / 4; ++s)
        load_dwords<16>(reinterpret_cast<uint32_t(&)[4]>(kf[t][4 * s]), base, koff + 64 * s);
    }
  };
  auto load_v = [&](int i, const Pages& p) {
    const int k0 = part.steps.at(i) * kStep;
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      const char* base = vbase + p.page[t] * a.pool.v_page + ((k0 + 16 * t) & mask) * a.pool.v_slot;
#pragma unroll
      for (int j = 0; j < 4; ++j) load_dwords<256>(vf[4 * t + j], base + j * a.pool.v_slot, voff);
    }
  };

  float m = -INFINITY, l = 0;
  v4f o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = v4f{0, 0, 0, 0};

  Pages cur, next;
  auto step = [&](int i, bool more) __attribute__((always_inline)) {
    const int k0 = part.steps.at(i) * kStep;
    v4f s[kTiles];
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      s[t] = v4f{0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        uint32_t f[4];
        if constexpr (E4M3) {
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const uint32_t x = kf[t][4 * (k / 2) + 2 * (k % 2) + w];
            f[2 * w] = T::template from_e4m3<false>(x);
            f[2 * w + 1] = T::template from_e4m3<true>(x);
          }
        } else {
#pragma unroll
          for (int w = 0; w < 4; ++w) f[w] = kf[t][4 * k + w];
        }
        if constexpr (kQLds) {
          const uint4 v = *reinterpret_cast<const uint4*>(qs + 1024 * k);
          const uint32_t qk[4] = {v.x, v.y, v.z, v.w};
          s[t] = mfma16<T>(f, qk, s[t]);
        } else {
          s[t] = mfma16<T>(f, qf[k], s[t]);
        }
      }
    }
    issue_fence();  // keeps the phases' registers apart
    if (more) load_k(i + kWaves, next);
    issue_fence();
    float x[NK];
#pragma unroll
    for (int j = 0; j < NK; ++j) x[j] = s[j >> 2][j & 3] * sc;
    const bool whole = k0 + kStep <= part.len && (k0 >= lo || k0 + kStep <= a.sinks) && cur.ok == (1 << kTiles) - 1;
    if (!whole) {
#pragma unroll
      for (int j = 0; j < NK; ++j) {
        const int p = k0 + 16 * (j >> 2) + 4 * g + (j & 3);
        const bool seen = p < part.len && (p >= lo || p < a.sinks) && (cur.ok >> (j >> 2) & 1);
        x[j] = seen ? x[j] : -INFINITY;
#pragma unroll
        for (int w = 0; w < VW; ++w) vf[j][w] = seen ? vf[j][w] : 0;
      }
    }
    float top = x[0];
#pragma unroll
    for (int j = 1; j < NK; ++j) top = fmaxf(top, x[j]);
    top = max_over_groups(top);
    if (__ballot(top > m)) {
      const float m2 = fmaxf(m, top);
      const float keep = __builtin_amdgcn_exp2f(m2 == -INFINITY ? 0.0f : m - m2);
      m = m2;
      l *= keep;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] *= keep;
    }
    const float base = m == -INFINITY ? 0.0f : m;     // nothing seen yet: every numerator is 0
    uint32_t hi[NK / 2], lo2[NK / 2];
#pragma unroll
    for (int w = 0; w < NK / 2; ++w) {
      const float p0 = __builtin_amdgcn_exp2f(x[2 * w] - base), p1 = __builtin_amdgcn_exp2f(x[2 * w + 1] - base);
      l += p0 + p1;
      hi[w] = T::pair(p0, p1);
      lo2[w] = T::pair(p0 - T::wide(hi[w] & 0xFFFFu), p1 - T::wide(hi[w] >> 16));
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      uint32_t f[NK / 2];
#pragma unroll
      for (int w = 0; w < NK / 2; ++w) {
        if constexpr (E4M3) {
          // columns e and e ^ 1 of a position are one pair
          const uint32_t x0 = (e & 2) ? T::template from_e4m3<true>(vf[2 * w][e >> 2]) : T::template from_e4m3<false>(vf[2 * w][e >> 2]);
          const uint32_t x1 = (e & 2) ? T::template from_e4m3<true>(vf[2 * w + 1][e >> 2]) : T::template from_e4m3<false>(vf[2 * w + 1][e >> 2]);
          f[w] = perm(x1, x0, (e & 1) ? 0x07060302u : 0x05040100u);
        } else {
          f[w] = perm(vf[2 * w + 1][e >> 1], vf[2 * w][e >> 1], (e & 1) ? 0x07060302u : 0x05040100u);
        }
      }
      o[e] = mfma16<T>(f, hi, o[e]);
      o[e] = mfma16<T>(f, lo2, o[e]);
    }
    issue_fence();
    if (more) load_v(i + kWaves, next);
    issue_fence();
  };

  if (t0 + wave < t1) {
    cur = pages_of(t0 + wave);
    check(cur);
    load_k(t0 + wave, cur);
    load_v(t0 + wave, cur);
    next = pages_of(min(t0 + wave + kWaves, t1 - 1));
    int i = t0 + wave;
    for (; i + kWaves < t1; i += kWaves) {
      check(next);
      Pages after = pages_of(min(i + 2 * kWaves, t1 - 1));
      step(i, true);
      cur = next;
      next = after;
    }
    step(i, false);
  }

  // The waves' parts in one: o[e][i] is head col's column (4 g + i) C + e % C of run e / C.
  l = sum_over_groups(l);
  if (g == 0) {
    ms[wave][col] = m;
    ls[wave][col] = l;
  }
  __syncthreads();
  float top = ms[0][col];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) top = fmaxf(top, ms[w][col]);
  const float keep = __builtin_amdgcn_exp2f(top == -INFINITY ? 0.0f : m - top);
  // the upper half of the waves leaves its rows in LDS, the lower half adds its own
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] *= keep;
  float* mine = &os[wave % (kWaves / 2)][col][4 * g * C];
#pragma unroll
  for (int turn = 1; turn >= 0; --turn) {
    if (wave / (kWaves / 2) == turn && col < heads) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < E; e += 4) {
          float4 y = make_float4(o[e][i], o[e + 1][i], o[e + 2][i], o[e + 3][i]);
          float4* at = reinterpret_cast<float4*>(mine + 16 * C * (e / C) + i * C + e % C);
          if (turn == 0) {
            const float4 v = *at;
            y = make_float4(y.x + v.x, y.y + v.y, y.z + v.z, y.w + v.w);
          }
          *at = y;
        }
    }
    __syncthreads();
  }
  if (column == 0 && part.part == 0 && a.work && threadIdx.x == 0)
    reinterpret_cast<int2*>(a.work)[part.b] = make_int2(part.first, part.parts);
  const float vs = E4M3 && a.pool.vscale ? a.pool.vscale[h] : 1.0f;
  for (int x = threadIdx.x; x < heads * (D / 4); x += 64 * kWaves) {
    const int hh = x / (D / 4), d = 4 * (x % (D / 4));
    float4 y = make_float4(0, 0, 0, 0);
    float t = ms[0][hh];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) t = fmaxf(t, ms[w][hh]);
    float sum = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (w < kWaves / 2) {
        const float4 v = *reinterpret_cast<const float4*>(&os[w][hh][d]);
        y.x += v.x;
        y.y += v.y;
        y.z += v.z;
        y.w += v.w;
      }
      sum += ls[w][hh] * __builtin_amdgcn_exp2f(t == -INFINITY ? 0.0f : ms[w][hh] - t);
    }
    if (part.parts == 1) {
      const float r = sum == 0 ? 0.0f : vs * __builtin_amdgcn_rcpf(sum);
      store4<T>(a.y + part.b * a.ldy, (head0 + hh) * D + d, a.out_f32, y.x * r, y.y * r, y.z * r, y.w * r);
    } else {
      const int64_t at = static_cast<int64_t>(number) * a.heads + head0 + hh;
      float* ws = parts_at(a) + at * (D + 4);
      *reinterpret_cast<float4*>(ws + d) = y;
      if (d == 0) *reinterpret_cast<float2*>(ws + D) = make_float2(t, sum);
    }
  }
}

// Joins the parts of a sequence: a workgroup per head, D / 4 lanes for a part's row.
template <class T, int D>
__global__ __launch_bounds__(64 * kWaves) void paged_join_kernel(PagedAttnArgs a) {
  constexpr int L = D / 4, R = 64 * kWaves / L;     // lanes of a row, rows at a time
  __shared__ float4 os[R][L];
  __shared__ float ms[R], ls[R];
  const int b = blockIdx.y, head = blockIdx.x, r = threadIdx.x / L, at = threadIdx.x % L, d = 4 * at;
  const int2 own = reinterpret_cast<const int2*>(a.work)[b];
  if (own.y <= 1) return;
  const float* ws = parts_at(a) + (static_cast<int64_t>(own.x) * a.heads + head) * (D + 4);
  const int64_t ld = static_cast<int64_t>(a.heads) * (D + 4);
  float4 y = make_float4(0, 0, 0, 0);
  float m = -INFINITY, sum = 0;
  auto add = [&](float m1, float l1, float4 v) {
    const float top = fmaxf(m, m1), base = top == -INFINITY ? 0.0f : top;
    const float k0 = __builtin_amdgcn_exp2f(m - base), k1 = __builtin_amdgcn_exp2f(m1 - base);
    m = top;
    y = make_float4(y.x * k0 + v.x * k1, y.y * k0 + v.y * k1, y.z * k0 + v.z * k1, y.w * k0 + v.w * k1);
    sum = sum * k0 + l1 * k1;
  };
#pragma unroll 4
  for (int p = r; p < own.y; p += R) {
    const float4 v = *reinterpret_cast<const float4*>(ws + p * ld + d);
    const float2 ml = *reinterpret_cast<const float2*>(ws + p * ld + D);
    add(ml.x, ml.y, v);
  }
  os[r][at] = y;
  if (at == 0) {
    ms[r] = m;
    ls[r] = sum;
  }
  __syncthreads();
  if (r) return;
#pragma unroll
  for (int i = 1; i < R; ++i) add(ms[i], ls[i], os[i][at]);
  const float vs = a.pool.vscale ? a.pool.vscale[head / a.group] : 1.0f;
  const float k = sum == 0 ? 0.0f : vs * __builtin_amdgcn_rcpf(sum);
  store4<T>(a.y + b * a.ldy, head * D + d, a.out_f32, y.x * k, y.y * k, y.z * k, y.w * k);
}

// The deal of a call and the most parts it can come to: the shares' and one more for each sequence, or every sequence
// at its longest in the smallest shares.
struct Plan {
  Deal deal;
  int64_t parts;
  bool split;
};
Plan plan(int kv_heads, int group, int hd, int seqs, int cap, int window, int sinks) {
  const int columns = kv_heads * ceil_div(group, kHeads);
  Plan p;
  const int step = step_of(hd);
  p.deal = {std::max(kSlots / columns, 1), std::max(kFew / columns, 1), kLeast / step, kShort / step};
  int64_t longest = ceil_div(cap, step);
  if (window > 0) longest = std::min<int64_t>(longest, window / step + 2 + ceil_div(std::min(sinks, cap), step));
  const int64_t most = (longest + p.deal.least - 1) / p.deal.least;
  p.split = most > 1;
  p.parts = std::min<int64_t>(int64_t{p.deal.slots} + seqs, most * seqs);
  return p;
}

template <class T, bool E4M3, int D>
hipError_t go(const PagedAttnArgs& a, hipStream_t s) {
  const int tiles = ceil_div(a.group, kHeads);
  const Plan p = plan(a.pool.kv_heads, a.group, D, a.seqs.seqs, a.seqs.cap, a.window, a.sinks);
  const dim3 grid(static_cast<uint32_t>(a.pool.kv_heads * tiles * p.parts)), block(64 * kWaves);
  hipLaunchKernelGGL((paged_decode_kernel<T, E4M3, D>), grid, block, 0, s, a, p.deal, tiles);
  if (p.split) hipLaunchKernelGGL((paged_join_kernel<T, D>), dim3(a.heads, a.seqs.seqs), block, 0, s, a);
  return hipGetLastError();
}

template <class T, bool E4M3>
hipError_t by_hd(const PagedAttnArgs& a, hipStream_t s) {
  return a.pool.hd == 64 ? go<T, E4M3, 64>(a, s) : a.pool.hd == 128 ? go<T, E4M3, 128>(a, s) : go<T, E4M3, 256>(a, s);
}

}  // namespace

int64_t paged_decode_workspace(int heads, int kv_heads, int hd, int seqs, int cap) {
  const Plan p = plan(kv_heads, heads / kv_heads, hd, seqs, cap, 0, 0);
  return p.split ? head_bytes(seqs) + p.parts * heads * (hd + 4) * 4 : 0;
}

hipError_t launch_paged_decode(const PagedAttnArgs& a, hipStream_t s) {
  const bool e4m3 = a.pool.dtype == KV_E4M3;
  if (a.dtype == KV_BF16) return e4m3 ? by_hd<Bf16, true>(a, s) : by_hd<Bf16, false>(a, s);
  return e4m3 ? by_hd<Fp16, true>(a, s) : by_hd<Fp16, false>(a, s);
}

}  // namespace tars
