// Attention of few rows per sequence over the paged cache, split over the caches' lengths and joined: decode, packed rows
// that come to 32 columns or fewer a sequence (a column is a row of one query head of a K / V head), and some over short
// caches.
//
// Per sequence and K / V head the cache is read once for the columns that share it, 16 or 32 of them, a step of 32
// positions at a time. Both products run on matrix instructions with the positions as rows, so that nothing passes
// through LDS on the way:
//   S^T = K Q^T   16 positions x 16 columns: lane l loads row l % 16 of K, 16 bytes of it, as the instruction wants it;
//   O^T += V^T P^T  lane l loads the rows of V at the very positions whose scores it holds (16 t + 4 (l / 16) + i of
//                 the step), hd / 16 columns of each: its block of 8 positions x hd / 16 columns, turned over by
//                 v_perm_b32 in its own registers, is V^T's operand for hd / 16 products, and its 8 numerators, in
//                 the order they left the softmax, are P^T's.
// The order of a product's inner index is free as long as both operands use it, which is all this needs. A numerator
// goes in as the sum of two values of q's type (its rounding and what that left), two products instead of one: next to
// the loads they are free, and the result is rounded once, at the end.
//
// The running maximum is kept per column; accumulators are rescaled only when it grows, which after a few steps is rare.
// Positions that a column does not see get a numerator of 0, and what nobody in the workgroup sees zeros for V (which may
// hold anything there). Where some columns see a position and others do not, its infinities and NaN are zeros in the
// product. Only steps at the rows' own positions, at the window's edges or with a page number outside the pool pay for that.
// Where one was found, or an output is not finite, the outputs that V's infinities and NaN reach are set to their sum at the
// end.
//
// The split is made on the device from the lengths: every workgroup adds up the steps of all sequences (those of a
// sequence once for each of its column tiles), sets the share C of a workgroup so that the shares fill the GPU, and finds
// its own (sequence, tile, part) in the prefix sums. So one long cache fills the GPU as well as many short ones, whatever
// the batch's longest is. A sequence of one part is written at once; the parts of the others go to the workspace as
// (maximum, sum, unscaled output) in fp32 and a second launch joins them in order.
//
// What bounds it: reading the cache once. Measured with 8 K / V heads of 128: three caches of 90k to 131k 231 us, 6.4 TB/s
// (a plain read of memory comes to 6.0 to 6.4); 64 of up to 8k 174 to 180 us, 5.7 TB/s; 32 of 9k to 17k in e4m3 with
// 64 query heads 162 us, 5.4 TB/s, the widening of K and V beside the loads; 16 of 3k to 16k with five rows each (32
// columns, two workgroups on a CU instead of three) 134 us, 4.8 TB/s. Short work is bound by the chain launch -> lengths
// -> page numbers -> K and V -> second launch: one cache of 2k 10.8 us, of 300 9.1 us; 100 windows of 512, one K / V
// head of 256, 20.2 us.
#include <algorithm>

#include "paged_device.h"

namespace tars {
namespace {

// Positions that a wave takes at a time: 16 for heads of 256, whose K and V rows fill the registers.
constexpr int step_of(int hd) { return hd == 256 ? 16 : 32; }
constexpr int kWaves = 4;
// Long work is dealt to two rounds of three workgroups on every CU, of two with 32 columns (kSlots for each): 64 caches of
// up to 8k 174 us and three of 110k 231 us (in 1024 workgroups 175 and 246, in 2048 173 and 234). Heads of 256, of which a
// CU holds two, take the same: 172 and 235 us (in 1024: 176 and 225). Short work, shares of up to kShort positions, is
// dealt to two workgroups on a CU: 100 windows of 512 13.9 us (16.4 with one, which is better for one long cache: 8k 15.0
// and 13.1). A share has a step for each wave at least: one cache of 4k 10.9 us (12.8 with half of that).
constexpr int kSlots = 512, kFew = 512, kShort = 512;
// Caches that may have up to kAlone steps, by the table's width or the window, are not split, which spares the second launch:
// one of 120 positions 7.3 us (8.7 in a table for 8192), of 300 9.1 us (9.8), of 480 10.4 us (10.2; the host's work is 3 us
// less), 32 of up to 480 14.8 us (18.0); of 600, whose 19 steps are split, 10.3 us (11.4).
constexpr int kAlone = 16;

struct Deal {
  int slots, few;        // workgroups for a K / V head, of long and of short work
  int least, most_few;   // steps
};
// A sequence's rows and steps, and its column tiles of `wide` columns.
struct Work {
  int len, first, rows, tiles;
  Steps steps;
};
struct Part {
  int b, tile, part, parts;
  int first;             // the number of the sequence's first part among all
  Work work;
};

template <int STEP>
__device__ __forceinline__ Work work_of(const PagedAttnArgs& a, int b, int wide) {  // wide: a constant; of no sequence: no rows
  Work w{0, 0, 0, 0, {0, 0, 0}};
  if (b >= a.seqs.seqs) return w;
  w.len = seq_len(a.seqs.lens, b, a.seqs.cap);
  const RowSpan r = a.seqs.starts ? seq_rows(a.seqs.starts, b, a.seqs.rows) : RowSpan{b, 1};
  w.first = r.first;
  w.rows = r.n;
  w.tiles = static_cast<uint32_t>(r.n * a.group + wide - 1) / static_cast<uint32_t>(wide);
  w.steps = visible_steps(w.len - r.n, w.len - 1, w.len, a.window, a.sinks, STEP);
  return w;
}

// The share C of a workgroup for `total` steps.
__device__ __forceinline__ int share_of(uint64_t total, const Deal& deal) {
  // in units of 2^20 steps where the sum has more than 31 bits (a share too long is no harm; no sequence has more than
  // 2^26 steps)
  const int up = total < (1ull << 31) ? 0 : 20;
  const uint32_t units = static_cast<uint32_t>((total + (1ull << up) - 1) >> up);
  const auto per = [&](uint32_t slots) { return min((units + slots - 1) / slots, 1u << 26 >> up) << up; };
  const int c = max(static_cast<int>(per(deal.slots)), min(static_cast<int>(per(deal.few)), deal.most_few));
  return max(c, deal.least);
}
__device__ __forceinline__ uint64_t steps_of(const Work& w) { return static_cast<uint64_t>(w.steps.n()) * w.tiles; }
__device__ __forceinline__ uint64_t wave_sum(uint64_t x) {
  const auto sum = [&](int from) -> uint64_t { return group_sum<64>(static_cast<int>(x >> from & 0xFFFFF)); };
  return sum(0) + (sum(20) << 20) + (sum(40) << 40);
}
__device__ __forceinline__ int parts_of(const Work& w, int c) { return max((w.steps.n() + c - 1) / c, 1); }

// The part numbered idx of the wave's 64 sequences from b0 on, w a lane's, whose parts end at `upto`.
__device__ __forceinline__ Part pick(const Work& w, int parts, int upto, int b0, int idx) {
  const int at = __builtin_ctzll(__ballot(upto > idx));
  const auto of = [&](int x) { return __builtin_amdgcn_readlane(x, at); };
  Part p;
  p.b = __builtin_amdgcn_readfirstlane(b0 + at);
  p.parts = of(parts);
  p.work = {of(w.len), of(w.first), of(w.rows), of(w.tiles), {of(w.steps.a), of(w.steps.b0), of(w.steps.b1)}};
  p.first = of(upto) - p.parts * p.work.tiles;
  // clamped, for starts that do not ascend: their sums may be anything
  const int part = p.work.tiles == 1 ? idx - p.first : (idx - p.first) / p.work.tiles;
  p.part = iclamp(part, 0, p.parts - 1);
  p.tile = iclamp(idx - p.first - part * p.work.tiles, 0, p.work.tiles - 1);
  return p;
}

// The part numbered idx among all (b < 0: none), the same in every wave: a sequence's tiles side by side, then its next
// part. Up to 64 sequences are every wave's, a lane to each; of more, each wave takes its 64 in turn (250k positions of one
// K / V head of 128 in 64 caches 28.7 us, in 1024 39 us, in 4096 92 us; 54 and 181 us where every wave went through all).
template <int STEP>
__device__ __forceinline__ Part find_part(const PagedAttnArgs& a, int wide, const Deal& deal, int idx) {
  const Part none{-1, 0, 0, 0, 0, {0, 0, 0, 0, {0, 0, 0}}};
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (a.seqs.seqs <= 64) {
    const Work w = work_of<STEP>(a, lane, wide);
    const int c = share_of(wave_sum(steps_of(w)), deal);
    const int parts = parts_of(w, c), upto = inclusive_sum(parts * w.tiles);
    return idx < __builtin_amdgcn_readlane(upto, 63) ? pick(w, parts, upto, 0, idx) : none;
  }
  __shared__ uint64_t sums[kWaves];
  __shared__ int counts[2][kWaves];
  __shared__ Part found;
  uint64_t mine = 0;
  for (int b0 = 64 * wave; b0 < a.seqs.seqs; b0 += 64 * kWaves) mine += steps_of(work_of<STEP>(a, b0 + lane, wide));
  mine = wave_sum(mine);
  if (lane == 0) sums[wave] = mine;
  __syncthreads();
  uint64_t total = 0;
#pragma unroll
  for (int x = 0; x < kWaves; ++x) total += sums[x];
  const int c = share_of(total, deal);
  int before = 0;
  for (int b0 = 0, turn = 0; b0 < a.seqs.seqs; b0 += 64 * kWaves, turn ^= 1) {
    const Work w = work_of<STEP>(a, b0 + 64 * wave + lane, wide);
    const int parts = parts_of(w, c), own = inclusive_sum(parts * w.tiles);
    if (lane == 63) counts[turn][wave] = own;
    __syncthreads();
    // the wave whose parts hold it, alike in all of them whatever the counts (starts that do not ascend)
    int upto = before, start = 0, owner = -1;
#pragma unroll
    for (int x = 0; x < kWaves; ++x) {
      const int n = counts[turn][x];
      if (owner < 0 && upto <= idx && idx < upto + n) {
        owner = x;
        start = upto;
      }
      upto += n;
    }
    before = upto;
    owner = __builtin_amdgcn_readfirstlane(owner);
    if (owner >= 0) {
      if (wave == owner) {
        const Part p = pick(w, parts, start + own, b0 + 64 * wave, idx);
        if (lane == 0) found = p;
      }
      __syncthreads();
      Part p;
      for (int x = 0; x < static_cast<int>(sizeof(Part) / 4); ++x)
        reinterpret_cast<int*>(&p)[x] = __builtin_amdgcn_readfirstlane(reinterpret_cast<const int*>(&found)[x]);
      return p;
    }
  }
  return none;
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

// The pages of a step's blocks of 16 positions and whether they are in the pool (bit t), the same in every lane.
struct Pages {
  int page[2];
  int ok;
};

// The workspace: (first part, parts) of every sequence, then every part's columns for every K / V head.
__host__ __device__ __forceinline__ int64_t head_bytes(int seqs) { return (8ll * seqs + 15) / 16 * 16; }
__device__ __forceinline__ float* parts_at(const PagedAttnArgs& a) { return a.work + head_bytes(a.seqs.seqs) / 4; }

// CT: column tiles of 16.
template <class T, bool E4M3, int D, int CT>
__global__ __launch_bounds__(64 * kWaves, 2) void paged_rows_kernel(PagedAttnArgs a, Deal deal) {
  constexpr int KS = D / 32;                        // products of a scores tile
  constexpr int E = D / 16;                         // columns of V per lane
  constexpr int KW = E4M3 ? 4 * KS / 2 : 4 * KS;    // dwords of a lane's K row part
  constexpr int VW = E4M3 ? E / 4 : E / 2;          // dwords of a lane's V row part
  constexpr int C = VW == 8 ? 8 : E;                // its neighbouring columns: two runs of 8 for 16-bit rows of 256
  constexpr int kStep = step_of(D), kTiles = kStep / 16, NK = kStep / 4;  // NK: positions of a lane
  constexpr int kWide = 16 * CT;
  __shared__ __attribute__((aligned(16))) float os[kWaves / 2][kWide][D + 4];
  __shared__ float ms[kWaves][kWide], ls[kWaves][kWide];
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int number = blockIdx.x / a.pool.kv_heads, h = blockIdx.x % a.pool.kv_heads;
  const Part part = find_part<kStep>(a, kWide, deal, number);
  if (part.b < 0) return;
  const Steps steps = part.work.steps;
  const int len = part.work.len, p0 = len - part.work.rows;       // the first row's position
  const int c0 = part.tile * kWide, cols = min(part.work.rows * a.group - c0, kWide);
  const int n = steps.n(), per = (n + part.parts - 1) / part.parts;
  const int t0 = min(part.part * per, n), t1 = min(n, t0 + per);
  // positions of the workgroup's first and last column, and of this lane's
  const auto token_of = [&](int x) { return part.work.rows == 1 ? 0 : x / a.group; };
  const int plo = p0 + token_of(c0), phi = p0 + token_of(c0 + cols - 1);
  int at[CT];
#pragma unroll
  for (int u = 0; u < CT; ++u) at[u] = p0 + token_of(c0 + min(16 * u + col, cols - 1));

  // Q^T. Heads of 256 keep it in LDS (every wave's own copy, 16 bytes of a lane at a time), where the registers are needed
  // for K and V.
  constexpr bool kQLds = D == 256;
  static_assert(!kQLds || CT == 1, "one tile of columns");
  uint32_t qf[CT][kQLds ? 1 : KS][4];
  char* qs = reinterpret_cast<char*>(os) + 1024 * KS * wave + 16 * lane;
  static_assert(!kQLds || 1024 * KS * kWaves <= sizeof(os), "Q's copies fit the rows that join the waves");
#pragma unroll
  for (int u = 0; u < CT; ++u) {
    const int x = c0 + min(16 * u + col, cols - 1), token = token_of(x);
    const char* q = a.q + (part.work.first + token) * a.ldq + 2 * D * (h * a.group + x - token * a.group);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      load_dwords<16>(qf[u][kQLds ? 0 : s], q, E4M3 ? 128 * (s / 2) + 16 * (s % 2) + 32 * g : 64 * s + 16 * g);
      if constexpr (kQLds) *reinterpret_cast<uint4*>(qs + 1024 * s) = make_uint4(qf[0][0][0], qf[0][0][1], qf[0][0][2], qf[0][0][3]);
    }
  }
  const float sc = score_scale(a, h);

  const int shift = a.pool.page_shift, mask = (1 << shift) - 1, last = max(len - 1, 0) >> shift;
  const __attribute__((address_space(4))) int32_t* table = reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(
      reinterpret_cast<uintptr_t>(a.seqs.table + part.b * a.seqs.ld_table));
  const uint32_t koff = col * static_cast<uint32_t>(a.pool.k_slot) + 16 * g;
  const uint32_t voff = 4 * g * static_cast<uint32_t>(a.pool.v_slot) + 4 * (VW < 4 ? VW : 4) * col;
  const char* kbase = a.pool.k + h * a.pool.k_head;
  const char* vbase = a.pool.v + h * a.pool.v_head;
  auto pages_of = [&](int i) {
    const int k0 = steps.at(i) * kStep;
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
    const int k0 = steps.at(i) * kStep;
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      const char* base = kbase + p.page[t] * a.pool.k_page + ((k0 + 16 * t) & mask) * a.pool.k_slot;
#pragma unroll
      for (int s = 0; s < KW / 4; ++s)
        load_dwords<16>(reinterpret_cast<uint32_t(&)[4]>(kf[t][4 * s]), base, koff + 64 * s);
    }
  };
  auto load_v = [&](int i, const Pages& p) {
    const int k0 = steps.at(i) * kStep;
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      const char* base = vbase + p.page[t] * a.pool.v_page + ((k0 + 16 * t) & mask) * a.pool.v_slot;
#pragma unroll
      for (int j = 0; j < 4; ++j) load_dwords<256>(vf[4 * t + j], base + j * a.pool.v_slot, voff);
    }
  };
  // Whether every column sees all of step i.
  auto is_whole = [&](int i, int ok) {
    const int k0 = steps.at(i) * kStep;
    return k0 + kStep - 1 <= plo && (a.window == 0 || k0 > phi - a.window || k0 + kStep <= a.sinks) && ok == (1 << kTiles) - 1;
  };

  float m[CT], l[CT];
  v4f o[CT][E];
#pragma unroll
  for (int u = 0; u < CT; ++u) {
    m[u] = -INFINITY;
    l[u] = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) o[u][e] = v4f{0, 0, 0, 0};
  }
  bool spoiled = false;

  Pages cur, next;
  auto step = [&](int i, bool more) __attribute__((always_inline)) {
    v4f s[CT][kTiles];
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
#pragma unroll
      for (int u = 0; u < CT; ++u) s[u][t] = v4f{0, 0, 0, 0};
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
          s[0][t] = mfma16<T>(f, qk, s[0][t]);
        } else {
#pragma unroll
          for (int u = 0; u < CT; ++u) s[u][t] = mfma16<T>(f, qf[u][k], s[u][t]);
        }
      }
    }
    issue_fence();  // keeps the phases' registers apart
    if (more) load_k(i + kWaves, next);
    issue_fence();
    float x[CT][NK];
#pragma unroll
    for (int u = 0; u < CT; ++u)
#pragma unroll
      for (int j = 0; j < NK; ++j) x[u][j] = s[u][j >> 2][j & 3];
    if (!is_whole(i, cur.ok)) {
      const int k0 = steps.at(i) * kStep;
#pragma unroll
      for (int j = 0; j < NK; ++j) {
        const int p = k0 + 16 * (j >> 2) + 4 * g + (j & 3);
        const bool in = cur.ok >> (j >> 2) & 1;
#pragma unroll
        for (int u = 0; u < CT; ++u) x[u][j] = in && sees(at[u], p, a.window, a.sinks) ? x[u][j] : -INFINITY;
        // seen by some column: by the last, or by the first or its own row where that has a window
        const bool some = in && p <= phi && sees(max(plo, p), p, a.window, a.sinks);
#pragma unroll
        for (int w = 0; w < VW; ++w) vf[j][w] = some ? vf[j][w] : 0;
      }
      if (plo != phi) {
        uint32_t bad = 0;
#pragma unroll
        for (int j = 0; j < NK; ++j)
#pragma unroll
          for (int w = 0; w < VW; ++w) {
            const uint32_t out = E4M3 ? nan_e4m3(vf[j][w]) : not_finite<T>(vf[j][w]);
            bad |= out;
            vf[j][w] &= ~out;
            asm volatile("" : "+v"(bad), "+v"(vf[j][w]));  // one mask at a time in the registers
          }
        spoiled |= bad != 0;
      }
    }
    uint32_t hi[CT][NK / 2], lo[CT][NK / 2];
#pragma unroll
    for (int u = 0; u < CT; ++u) {
      float top = x[u][0];
#pragma unroll
      for (int j = 1; j < NK; ++j) top = fmaxf(top, x[u][j]);
      top = over_row<16>(top, [](float y, float z) { return fmaxf(y, z); });
      // by column, not for the wave as a whole: the compiler then scales in place
      if (top > m[u]) {
        const float keep = __builtin_amdgcn_exp2f((m[u] - top) * sc);
        m[u] = top;
        l[u] *= keep;
#pragma unroll
        for (int e = 0; e < E; ++e) o[u][e] *= keep;
      }
      const float base = m[u] == -INFINITY ? 0.0f : m[u];   // nothing seen yet: every numerator is 0
#pragma unroll
      for (int w = 0; w < NK / 2; ++w) {
        const float y = __builtin_amdgcn_exp2f((x[u][2 * w] - base) * sc), z = __builtin_amdgcn_exp2f((x[u][2 * w + 1] - base) * sc);
        l[u] += y + z;
        hi[u][w] = T::pair(y, z);
        lo[u][w] = T::pair(y - T::wide(hi[u][w] & 0xFFFFu), z - T::wide(hi[u][w] >> 16));
      }
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
#pragma unroll
      for (int u = 0; u < CT; ++u) {
        o[u][e] = mfma16<T>(f, hi[u], o[u][e]);
        o[u][e] = mfma16<T>(f, lo[u], o[u][e]);
      }
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

  // V's infinities and NaN in whole steps met the numerators, second halves of 0 or less among them: the outputs they reached
  // are not finite, and are put right at the end.
#pragma unroll
  for (int u = 0; u < CT; ++u) spoiled |= not_all_finite(o[u]);

  // The waves' parts in one: o[u][e][i] is column 16 u + col's (4 g + i) C + e % C of run e / C.
#pragma unroll
  for (int u = 0; u < CT; ++u) {
    l[u] = over_row<16>(l[u], [](float y, float z) { return y + z; });
    if (g == 0) {
      ms[wave][16 * u + col] = m[u];
      ls[wave][16 * u + col] = l[u];
    }
  }
  const int any = __syncthreads_or(spoiled);
#pragma unroll
  for (int u = 0; u < CT; ++u) {
    float top = ms[0][16 * u + col];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = fmaxf(top, ms[w][16 * u + col]);
    const float keep = __builtin_amdgcn_exp2f(top == -INFINITY ? 0.0f : (m[u] - top) * sc);
#pragma unroll
    for (int e = 0; e < E; ++e) o[u][e] *= keep;
  }
  // the upper half of the waves leaves its columns in LDS, the lower half adds its own
#pragma unroll
  for (int turn = 1; turn >= 0; --turn) {
    if (wave / (kWaves / 2) == turn) {
#pragma unroll
      for (int u = 0; u < CT; ++u) {
        float* mine = &os[wave % (kWaves / 2)][16 * u + col][4 * g * C];
        if (16 * u + col < cols) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < E; e += 4) {
              float4 y = make_float4(o[u][e][i], o[u][e + 1][i], o[u][e + 2][i], o[u][e + 3][i]);
              float4* to = reinterpret_cast<float4*>(mine + 16 * C * (e / C) + i * C + e % C);
              if (turn == 0) {
                const float4 v = *to;
                y = make_float4(y.x + v.x, y.y + v.y, y.z + v.z, y.w + v.w);
              }
              *to = y;
            }
        }
      }
    }
    __syncthreads();
  }
  if (h == 0 && part.part == 0 && part.tile == 0 && a.work && threadIdx.x == 0)
    reinterpret_cast<int2*>(a.work)[part.b] = make_int2(part.first, part.parts);
  float* ws = parts_at(a) + (static_cast<int64_t>(number) * a.pool.kv_heads + h) * kWide * (D + 4);
  const float vs = E4M3 && a.pool.vscale ? a.pool.vscale[h] : 1.0f;
  for (int x = threadIdx.x; x < cols * (D / 4); x += 64 * kWaves) {
    const int cc = x / (D / 4), d = 4 * (x % (D / 4));
    float4 y = make_float4(0, 0, 0, 0);
    float top = ms[0][cc];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = fmaxf(top, ms[w][cc]);
    float sum = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (w < kWaves / 2) {
        const float4 v = *reinterpret_cast<const float4*>(&os[w][cc][d]);
        y.x += v.x;
        y.y += v.y;
        y.z += v.z;
        y.w += v.w;
      }
      sum += ls[w][cc] * __builtin_amdgcn_exp2f(top == -INFINITY ? 0.0f : (ms[w][cc] - top) * sc);
    }
    if (part.parts == 1) {
      const float r = sum == 0 ? 0.0f : vs * __builtin_amdgcn_rcpf(sum);
      const int token = token_of(c0 + cc), head = h * a.group + c0 + cc - token * a.group;
      store4<T>(a.y + (part.work.first + token) * a.ldy, head * D + d, a.out_f32, y.x * r, y.y * r, y.z * r, y.w * r);
    } else {
      float* to = ws + cc * (D + 4);
      *reinterpret_cast<float4*>(to + d) = y;
      if (d == 0) *reinterpret_cast<float2*>(to + D) = make_float2(top, sum);
    }
  }
  if (!any) return;
  __syncthreads();
  const auto sound = [&](int x) {
    float sum = 0;
    for (int w = 0; w < kWaves; ++w) sum += ls[w][x - c0];
    return part.parts > 1 || sum < INFINITY;
  };
  set_unfinite<T, E4M3, D, kStep>(
      a, part.b, h, len, [&](int i) { return steps.at(i); }, t0, t1, p0, part.work.first, c0, cols,
      [&](int x) { return part.parts > 1 ? ws + (x - c0) * (D + 4) : nullptr; }, sound);
}

// Joins the parts of a row, of `all`: a workgroup per row and head, D / 4 lanes for a part's row.
template <class T, int D, int CT>
__global__ __launch_bounds__(64 * kWaves) void paged_rows_join_kernel(PagedAttnArgs a, int all) {
  constexpr int L = D / 4, R = 64 * kWaves / L, kWide = 16 * CT;  // lanes of a row, rows at a time
  __shared__ float4 os[R][L];
  __shared__ float ms[R], ls[R];
  const int row = blockIdx.x, head = blockIdx.y, r = threadIdx.x / L, at = threadIdx.x % L, d = 4 * at;
  int b = row, token = 0, tiles = ceil_div(a.group, kWide);
  if (a.seqs.starts) {
    b = seq_of_row(a.seqs, row);
    if (b >= a.seqs.seqs) return;
    const RowSpan span = seq_rows(a.seqs.starts, b, a.seqs.rows);
    token = row - span.first;
    if (token < 0 || token >= span.n) return;
    tiles = ceil_div(span.n * a.group, kWide);
  }
  const int2 own = reinterpret_cast<const int2*>(a.work)[b];
  if (own.y <= 1) return;
  const int h = head / a.group, x = token * a.group + head - h * a.group;
  // Within the workspace: with starts that do not ascend nobody may have written the sequence's numbers, or not all its parts.
  const int first = own.x + x / kWide, n = min(own.y, (all - 1 - first) / tiles + 1);
  if (own.x < 0 || first < 0 || first >= all) return;
  const int64_t ld = static_cast<int64_t>(tiles) * a.pool.kv_heads * kWide * (D + 4);
  const float* ws = parts_at(a) + ((static_cast<int64_t>(first) * a.pool.kv_heads + h) * kWide + x % kWide) * (D + 4);
  float4 y = make_float4(0, 0, 0, 0);
  float m = -INFINITY, sum = 0;
  const float sc = score_scale(a, h);
  auto add = [&](float m1, float l1, float4 v) {
    const float top = fmaxf(m, m1), base = top == -INFINITY ? 0.0f : top;
    const float k0 = __builtin_amdgcn_exp2f((m - base) * sc), k1 = __builtin_amdgcn_exp2f((m1 - base) * sc);
    m = top;
    y = make_float4(y.x * k0 + v.x * k1, y.y * k0 + v.y * k1, y.z * k0 + v.z * k1, y.w * k0 + v.w * k1);
    sum = sum * k0 + l1 * k1;
  };
#pragma unroll 4
  for (int p = r; p < n; p += R) {
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
  join_unfinite(y, n, [&](int p) { return *reinterpret_cast<const float4*>(ws + p * ld + d); });
  const float vs = a.pool.vscale ? a.pool.vscale[h] : 1.0f;
  const float k = sum == 0 ? 0.0f : vs * __builtin_amdgcn_rcpf(sum);
  store4<T>(a.y + row * a.ldy, head * D + d, a.out_f32, y.x * k, y.y * k, y.z * k, y.w * k);
}

// Column tiles of a workgroup, the deal, and the most parts it can come to: the shares' and one more for each column tile
// of each sequence, or everyone's at the longest in the smallest shares.
// 32 columns where a sequence has more than 16 on average: five rows of four query heads over 16 caches 134 us, and 206 in
// tiles of 16, which read the cache twice. 16 columns leave room for a third workgroup on a CU; heads of 256 for no more.
struct Plan {
  int wide;
  Deal deal;
  int64_t parts;
  bool split;
};
Plan plan(int kv_heads, int group, int hd, int rows, int seqs, int cap, bool one_each, int window, int sinks) {
  const int step = step_of(hd);
  Plan p;
  p.wide = hd != 256 && static_cast<int64_t>(rows) * group > 16ll * seqs ? 32 : 16;
  p.deal = {std::max(kSlots * (p.wide == 32 ? 2 : 3) / kv_heads, 1), std::max(kFew / kv_heads, 1), kWaves, kShort / step};
  int64_t longest = ceil_div(cap, step);
  if (window > 0 && one_each)
    longest = std::min<int64_t>(longest, window / step + 2 + ceil_div(std::min(sinks, cap), step));
  if (longest <= kAlone) p.deal.least = std::max<int>(longest, p.deal.least);
  const int64_t most = (longest + p.deal.least - 1) / p.deal.least;
  p.split = most > 1;
  const int64_t tiles = rows == seqs ? int64_t{seqs} * ceil_div(group, p.wide) : static_cast<int64_t>(rows) * group / p.wide + seqs;
  p.parts = std::min(p.deal.slots + tiles, most * tiles);
  return p;
}

template <class T, bool E4M3, int D, int CT>
hipError_t run(const PagedAttnArgs& a, const Plan& p, hipStream_t s) {
  const dim3 block(64 * kWaves);
  hipLaunchKernelGGL((paged_rows_kernel<T, E4M3, D, CT>), dim3(static_cast<uint32_t>(a.pool.kv_heads * p.parts)), block, 0, s, a, p.deal);
  if (p.split) hipLaunchKernelGGL((paged_rows_join_kernel<T, D, CT>), dim3(a.seqs.rows, a.heads), block, 0, s, a, static_cast<int>(p.parts));
  return hipGetLastError();
}

template <class T, bool E4M3>
hipError_t go(const PagedAttnArgs& a, hipStream_t s) {
  const Plan p = plan(a.pool.kv_heads, a.group, a.pool.hd, a.seqs.rows, a.seqs.seqs, a.seqs.cap, a.seqs.starts == nullptr, a.window,
                      a.sinks);
  if (a.pool.hd == 256) return run<T, E4M3, 256, 1>(a, p, s);
  if (a.pool.hd == 128) return p.wide == 32 ? run<T, E4M3, 128, 2>(a, p, s) : run<T, E4M3, 128, 1>(a, p, s);
  return p.wide == 32 ? run<T, E4M3, 64, 2>(a, p, s) : run<T, E4M3, 64, 1>(a, p, s);
}

}  // namespace

int64_t paged_rows_workspace(int heads, int kv_heads, int hd, int rows, int seqs, int cap) {
  const Plan p = plan(kv_heads, heads / kv_heads, hd, rows, seqs, cap, false, 0, 0);
  return p.split ? head_bytes(seqs) + p.parts * kv_heads * p.wide * (hd + 4) * 4 : 0;
}

hipError_t launch_paged_rows(const PagedAttnArgs& a, hipStream_t s) {
  const bool e4m3 = a.pool.dtype == KV_E4M3;
  if (a.dtype == KV_BF16) return e4m3 ? go<Bf16, true>(a, s) : go<Bf16, false>(a, s);
  return e4m3 ? go<Fp16, true>(a, s) : go<Fp16, false>(a, s);
}

}  // namespace tars
