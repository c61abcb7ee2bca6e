// Attention of packed prompt rows over the paged cache.
//
// The rows of one sequence that read one K / V head (its query heads' rows of every new token, token after token) are
// the columns of two matrix products, 32 to a wave:  S^T = K Q^T  and  O^T += V^T P^T.  A lane then holds scores of one
// row only: the running maximum and sum need one exchange between lane halves, and the numerators leave the softmax in
// the registers and order in which P^T's operand wants them (any order of a product's inner index will do, as long as
// V's operand has the same). K and V tiles of 64 positions pass through LDS, two tiles deep, loaded while the tile
// before is computed: 16-bit pools by direct loads whose 16-byte chunks are permuted within a row so that the reads of
// 32 rows' same chunk (K) and the transposing reads of 4 rows x 64 bytes (V) meet every bank once; e4m3 pools through
// registers, widened on the way.
//
// The scores come out of the product with the running maximum already taken off: it is the product's initial value. It
// is moved (and the sum and output rescaled) only when a score passes it by more than 2^kSlack, so the numerators lie
// in [0, 2^kSlack] and are rounded to q's type for the second product.
//
// Tiles at a row's own position, at a window's edge or with a page number outside the pool mask their scores. There a
// hidden position may hold anything: the tile of V is searched for infinities and NaN; if it has any, they are added to
// the rows that see them and zeroed before the product.
//
// A workgroup's rows are NW * 32; the last rows of a sequence, which see most, start first. With few rows their tiles
// are split over workgroups and joined by a second launch.
#include <algorithm>

#include "paged_device.h"

namespace tars {
namespace {

constexpr int tile_of(int hd) { return hd == 256 ? 32 : 64; }  // positions of a tile
constexpr float kLog2e = 1.44269504f;
constexpr float kSlack = 6.0f;

struct Tile {
  int b, first, rows, len;         // the sequence, its first row, its rows, its length
  int r0;                          // the first of the workgroup's rows among rows * group
};

// The workgroup's rows: `number` counts M-row tiles over the sequences; within one the last comes first.
__device__ __forceinline__ int inclusive_sum(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);  // row_shr 1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // row_bcast 15 to rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // row_bcast 31 to rows 2 and 3
  return x;
}

template <int M>
__device__ __forceinline__ Tile find_tile(const KvSeqs& s, int group, int number) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int b0 = 0; b0 < s.seqs; b0 += 64) {
    const int b = b0 + lane;
    RowSpan r{0, 0};
    if (b < s.seqs) r = seq_rows(s.starts, b, s.rows);
    const int tiles = ceil_div(r.n * group, M);
    const int upto = before + inclusive_sum(tiles);
    const uint64_t hit = __ballot(upto > number);
    if (hit) {
      const int at = __builtin_ctzll(hit);
      Tile t;
      t.b = __builtin_amdgcn_readfirstlane(b0 + at);
      t.first = __builtin_amdgcn_readlane(r.first, at);
      t.rows = __builtin_amdgcn_readlane(r.n, at);
      t.r0 = (__builtin_amdgcn_readlane(upto, at) - 1 - number) * M;
      t.len = __builtin_amdgcn_readfirstlane(seq_len(s.lens, t.b, s.cap));
      return t;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }
  return {-1, 0, 0, 0, 0};
}

template <int D>
__device__ __forceinline__ Steps steps_of(const Tile& t, int m, const PagedAttnArgs& a) {
  const int p0 = t.len - t.rows;
  return visible_steps(p0 + t.r0 / a.group, p0 + (min(t.r0 + m, t.rows * a.group) - 1) / a.group, t.len, a.window, a.sinks,
                       tile_of(D));
}

// Tiles of a part, and the parts of n tiles.
__device__ __forceinline__ int parts_of(int n, int splits, int least) { return max(min(splits, n / least), 1); }

// Byte offset of 16-byte chunk c of row k in a tile.
template <int D>
__device__ __forceinline__ int k_at(int k, int c) {
  return k * 2 * D + ((c ^ (D == 64 ? (k >> 1) & 7 : k & 15)) << 4);
}
template <int D>
__device__ __forceinline__ int v_at(int k, int c) {
  return k * 2 * D + ((c ^ (D == 64 ? (k & 2) << 1 : (k & 3) << 2)) << 4);
}

template <class T>
__device__ __forceinline__ uint32_t not_finite(uint32_t x) {  // 0xFFFF in each half that is infinite or NaN
  const uint32_t e = T::kExponent;
  return ((x & e) == e ? 0xFFFFu : 0) | ((x >> 16 & e) == e ? 0xFFFF0000u : 0);
}

template <class T, bool E4M3, int D, int NW>
__global__ __launch_bounds__(64 * NW, D == 256 ? 1 : 2) void paged_prompt_kernel(PagedAttnArgs a, int splits, int least) {
  constexpr int M = 32 * NW, KS = D / 16, NT = D / 32;
  constexpr int kTile = tile_of(D), kBlocks = kTile / 16, kHalves = kTile / 32;
  constexpr int kBytes = kTile * D * 2;                 // a tile of K or V
  __shared__ __attribute__((aligned(1024))) char lds[2][2][kBytes];  // [stage][K, V]
  __shared__ int flags[2];
  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = blockIdx.x % a.pool.kv_heads, rest = blockIdx.x / a.pool.kv_heads, split = rest % splits;
  const Tile tile = find_tile<M>(a.seqs, a.group, rest / splits);
  if (tile.b < 0) return;
  const Steps steps = steps_of<D>(tile, M, a);
  const int n = steps.n(), parts = parts_of(n, splits, least);
  if (split >= parts) return;
  const int per = ceil_div(n, parts), t0 = min(split * per, n), t1 = min(t0 + per, n);

  // the rows of this wave: row r of the sequence's rows * group is token r / group, query head r % group
  const int total = tile.rows * a.group, w0 = tile.r0 + 32 * wave, r = min(w0 + col, total - 1);
  const int token = r / a.group, head = h * a.group + r - token * a.group;
  const int p0 = tile.len - tile.rows, p = p0 + token;
  const int plo = p0 + tile.r0 / a.group, phi = p0 + (min(tile.r0 + M, total) - 1) / a.group;
  const bool mine = w0 < total;
  const int wlo = __builtin_amdgcn_readfirstlane(p), whi = __builtin_amdgcn_readlane(p, 31);

  uint4 qf[KS];
  const char* q = a.q + (tile.first + token) * a.ldq + 2 * D * head + 16 * half;
#pragma unroll
  for (int s = 0; s < KS; ++s) qf[s] = *reinterpret_cast<const uint4*>(q + 32 * s);
  const float sc = a.scale * kLog2e * (E4M3 && a.pool.kscale ? a.pool.kscale[h] : 1.0f);

  const int shift = a.pool.page_shift, mask = (1 << shift) - 1, last = max(tile.len - 1, 0) >> shift;
  const __attribute__((address_space(4))) int32_t* table = reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(
      reinterpret_cast<uintptr_t>(a.seqs.table + tile.b * a.seqs.ld_table));
  const char* kbase = a.pool.k + h * a.pool.k_head;
  const char* vbase = a.pool.v + h * a.pool.v_head;

  // the pages of a tile's four blocks of 16 positions; the ones outside the pool are read as page 0 and masked
  struct Pages {
    int p0, p1, p2, p3, ok;
    __device__ __forceinline__ int of(int block) const {
      const int x0 = p0, x1 = p1, x2 = p2, x3 = p3;
      const int even = block & 2 ? x2 : x0, odd = block & 2 ? x3 : x1;
      return block & 1 ? odd : even;
    }
  };
  auto pages_of = [&](int i) {
    const int k0 = steps.at(i) * kTile;
    return Pages{table[min(k0 >> shift, last)], table[min((k0 + 16) >> shift, last)], table[min((k0 + 32) >> shift, last)],
                 table[min((k0 + 48) >> shift, last)], 0};
  };
  auto in_pool = [&](int& page, int bit) {
    const bool in = static_cast<uint32_t>(page) < static_cast<uint32_t>(a.pool.pages);
    page = in ? page : 0;
    return in ? bit : 0;
  };
  auto check = [&](Pages g) {
    int p0 = g.p0, p1 = g.p1, p2 = g.p2, p3 = g.p3;
    const int ok = in_pool(p0, 1) | in_pool(p1, 2) | (kBlocks > 2 ? in_pool(p2, 4) | in_pool(p3, 8) : 0);
    return Pages{p0, p1, p2, p3, ok};
  };

  // Loading a tile. 16-bit: a load instruction moves 1 KiB = kRows rows, lane l the 16 bytes at 16 l.
  constexpr int kRows = 512 / D, kLoads = kTile / kRows;                    // of one of K, V
  constexpr int kHold = E4M3 ? kTile * D / 16 / (64 * NW) : 1;              // e4m3: 16-byte loads of a thread
  uint4 hold[2][kHold];
  auto load = [&](int i, Pages g, int stage) __attribute__((always_inline)) {
    const int k0 = steps.at(i) * kTile;
    if constexpr (E4M3) {
#pragma unroll
      for (int x = 0; x < kHold; ++x) {
        const int at = x * 64 * NW + threadIdx.x, k = at / (D / 16), c = at % (D / 16), page = g.of(k >> 4);
        const int64_t slot = (k0 + k) & mask;
        hold[0][x] = *reinterpret_cast<const uint4*>(kbase + page * a.pool.k_page + slot * a.pool.k_slot + 16 * c);
        hold[1][x] = *reinterpret_cast<const uint4*>(vbase + page * a.pool.v_page + slot * a.pool.v_slot + 16 * c);
      }
    } else {
#pragma unroll
      for (int x = 0; x < 2 * kLoads / NW; ++x) {
        const int j = wave + NW * (x % (kLoads / NW)), kk = j * kRows;
        const bool is_v = x >= kLoads / NW;
        const int k = lane / (D / 8), c = lane % (D / 8);                   // within the instruction's rows
        const int page = g.of(kk >> 4);
        const int64_t slot = (k0 + kk) & mask;
        const int swz = is_v ? v_at<D>(kk + k, c) : k_at<D>(kk + k, c);
        const uint32_t off = k * static_cast<uint32_t>(is_v ? a.pool.v_slot : a.pool.k_slot) + (swz & (2 * D - 1));
        const char* base = is_v ? vbase + page * a.pool.v_page + slot * a.pool.v_slot
                                : kbase + page * a.pool.k_page + slot * a.pool.k_slot;
        ring_load16(base, off, lds_addr(lds[stage][is_v]) + 1024 * j);
      }
    }
  };
  auto land = [&](int stage) __attribute__((always_inline)) {  // e4m3: the held rows widened into the stage
    if constexpr (E4M3) {
#pragma unroll
      for (int x = 0; x < kHold; ++x) {
        const int at = x * 64 * NW + threadIdx.x, k = at / (D / 16), c = at % (D / 16);
#pragma unroll
        for (int is_v = 0; is_v < 2; ++is_v) {
          const uint32_t w[4] = {hold[is_v][x].x, hold[is_v][x].y, hold[is_v][x].z, hold[is_v][x].w};
          uint32_t f[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            f[2 * i] = T::template from_e4m3<false>(w[i]);
            f[2 * i + 1] = T::template from_e4m3<true>(w[i]);
          }
          char* to = lds[stage][is_v];
          *reinterpret_cast<uint4*>(to + (is_v ? v_at<D>(k, 2 * c) : k_at<D>(k, 2 * c))) = make_uint4(f[0], f[1], f[2], f[3]);
          *reinterpret_cast<uint4*>(to + (is_v ? v_at<D>(k, 2 * c + 1) : k_at<D>(k, 2 * c + 1))) = make_uint4(f[4], f[5], f[6], f[7]);
        }
      }
    }
  };
  auto meet = [&]() {
    asm volatile("" : : : "memory");
    wait_lgkm0();
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
  };

  // m: the maximum taken off, in units of the raw scores; bound: a score (with m taken off) above it moves m
  float l = 0, bound = -INFINITY;
  v16f minus, o[NT];
#pragma unroll
  for (int i = 0; i < 16; ++i) minus[i] = 0;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[t][i] = 0;
  const float slack = kSlack * __builtin_amdgcn_rcpf(sc);
  // lane offsets of the reads: row col, chunk 2 s + half of K; V's transposing read of 4 rows x 16 columns
  const int vrow = 4 * half + ((lane & 15) >> 2), vchunk = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1), vbyte = (lane & 1) * 8;

  auto compute = [&](int i, int ok, int stage) __attribute__((always_inline)) {
    const int k0 = steps.at(i) * kTile;
    const char* kt = lds[stage][0];
    char* vt = lds[stage][1];
    const bool whole = k0 + kTile - 1 <= plo && (a.window == 0 || k0 > phi - a.window || k0 + kTile <= a.sinks) && ok == (1 << kBlocks) - 1;
    if (!whole) {
      // hidden positions may hold anything: 16 bytes of V's tile per thread and turn
      uint32_t bad = 0;
      for (int x = threadIdx.x; x < kBytes / 16; x += 64 * NW) {
        const uint4 v = *reinterpret_cast<const uint4*>(vt + 16 * x);
        bad |= not_finite<T>(v.x) | not_finite<T>(v.y) | not_finite<T>(v.z) | not_finite<T>(v.w);
      }
      if (bad) flags[i & 1] = 1;
      meet();
      const bool any = __builtin_amdgcn_readfirstlane(flags[i & 1]) != 0;
      if (threadIdx.x == 0) flags[(i & 1) ^ 1] = 0;
      if (any) {
        for (int k = 0; k < kTile; ++k) {
          const int j = k0 + k;
          const bool seen = sees(p, j, a.window, a.sinks) && (ok >> (k >> 4) & 1);
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const int d = 32 * t + 8 * (e >> 2) + 4 * half + (e & 3);
              const uint32_t v = *reinterpret_cast<const uint16_t*>(vt + v_at<D>(k, d >> 3) + 2 * (d & 7));
              o[t][e] += seen && not_finite<T>(v) ? T::wide(v) : 0.0f;
            }
        }
        meet();
        for (int x = threadIdx.x; x < kBytes / 16; x += 64 * NW) {
          uint4 v = *reinterpret_cast<uint4*>(vt + 16 * x);
          v.x &= ~not_finite<T>(v.x);
          v.y &= ~not_finite<T>(v.y);
          v.z &= ~not_finite<T>(v.z);
          v.w &= ~not_finite<T>(v.w);
          *reinterpret_cast<uint4*>(vt + 16 * x) = v;
        }
        meet();
      }
    }
    if (!mine || k0 > whi || (a.window != 0 && k0 + kTile - 1 <= wlo - a.window && k0 >= a.sinks)) return;  // nothing seen
    v16f s[kHalves];
#pragma unroll
    for (int t = 0; t < kHalves; ++t) {
      s[t] = minus;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const uint4 f = *reinterpret_cast<const uint4*>(kt + k_at<D>(32 * t + col, 2 * k + half));
        s[t] = T::mfma_32x32x16(f, qf[k], s[t]);
      }
    }
    if (!whole) {
#pragma unroll
      for (int t = 0; t < kHalves; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int k = 32 * t + 8 * (e >> 2) + 4 * half + (e & 3);
          const bool seen = sees(p, k0 + k, a.window, a.sinks) && (ok >> (k >> 4) & 1);
          s[t][e] = seen ? s[t][e] : -INFINITY;
        }
    }
    float top = s[0][0];
#pragma unroll
    for (int e = 1; e < kTile / 2; ++e) top = fmaxf(top, s[e >> 4][e & 15]);
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
    top = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
    if (__ballot(top > bound)) {
      const bool up = top > bound;
      // the first scores that a row sees set m from nothing: its sum and output are 0 (or not finite) then
      const float by = up ? top : 0.0f, keep = bound == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(-by * sc);
      l *= keep;
      bound = up ? slack : bound;
#pragma unroll
      for (int e = 0; e < 16; ++e) minus[e] -= by;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[t][e] *= keep;
#pragma unroll
      for (int e = 0; e < kTile / 2; ++e) s[e >> 4][e & 15] -= by;
    }
    uint32_t pf[kTile / 4];
#pragma unroll
    for (int e = 0; e < kTile / 4; ++e) {
      const float x = __builtin_amdgcn_exp2f(s[e >> 3][2 * e & 15] * sc), y = __builtin_amdgcn_exp2f(s[e >> 3][(2 * e & 15) + 1] * sc);
      l += x + y;
      pf[e] = T::pair(x, y);
    }
#pragma unroll
    for (int k = 0; k < kBlocks; ++k) {
      const uint4 pk = make_uint4(pf[4 * k], pf[4 * k + 1], pf[4 * k + 2], pf[4 * k + 3]);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        uint32_t f[4];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const char* at = vt + v_at<D>(16 * k + 8 * x + vrow, 4 * t + vchunk) + vbyte;
          const v4s v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)(at));
          const uint2 w = __builtin_bit_cast(uint2, v);
          f[2 * x] = w.x;
          f[2 * x + 1] = w.y;
        }
        o[t] = T::mfma_32x32x16(make_uint4(f[0], f[1], f[2], f[3]), pk, o[t]);
      }
    }
  };

  if (threadIdx.x < 2) flags[threadIdx.x] = 0;
  if (t0 < t1) {
    Pages cur = pages_of(t0), next = pages_of(min(t0 + 1, t1 - 1));
    cur = check(cur);
    load(t0, cur, 0);
    if constexpr (E4M3) land(0);
    for (int i = t0; i < t1; ++i) {
      const int stage = (i - t0) & 1;
      if constexpr (!E4M3) wait_vmcnt<0>();
      meet();
      next = check(next);
      if (i + 1 < t1) load(i + 1, next, stage ^ 1);
      const Pages after = pages_of(min(i + 2, t1 - 1));
      compute(i, cur.ok, stage);
      if constexpr (E4M3) {
        if (i + 1 < t1) land(stage ^ 1);
      }
      cur = next;
      next = after;
    }
  }

  // row r: columns 32 t + 8 (e / 4) + 4 half + e % 4
  const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
  l = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
  if (w0 + col >= total) return;
  if (parts == 1) {
    const float vs = E4M3 && a.pool.vscale ? a.pool.vscale[h] : 1.0f;
    const float k = l == 0 ? 0.0f : vs * __builtin_amdgcn_rcpf(l);
    char* y = a.y + (tile.first + token) * a.ldy;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        store4<T>(y, head * D + 32 * t + 2 * e + 4 * half, a.out_f32, o[t][e] * k, o[t][e + 1] * k, o[t][e + 2] * k, o[t][e + 3] * k);
  } else {
    float* ws = a.work + ((static_cast<int64_t>(split) * a.seqs.rows + tile.first + token) * a.heads + head) * (D + 4);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *reinterpret_cast<float4*>(ws + 32 * t + 2 * e + 4 * half) = make_float4(o[t][e], o[t][e + 1], o[t][e + 2], o[t][e + 3]);
    // the maximum in the exponent's units; none seen: the sum is 0 and the maximum counts for nothing
    if (half == 0) *reinterpret_cast<float2*>(ws + D) = make_float2(l == 0 ? -INFINITY : -minus[0] * sc, l);
  }
}

// Joins the parts of rows whose tiles were split: a workgroup per row and 4 heads, D / 4 lanes of a wave for a head's
// row, the wave's other lanes for other parts.
template <class T, int D, int M>
__global__ __launch_bounds__(256) void paged_prompt_join_kernel(PagedAttnArgs a, int splits, int least) {
  constexpr int L = D / 4, R = 64 / L;
  const int row = blockIdx.x, lane = threadIdx.x & 63;
  const int head = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = seq_of_row(a.seqs, row);
  if (b >= a.seqs.seqs || head >= a.heads) return;
  const RowSpan span = seq_rows(a.seqs.starts, b, a.seqs.rows);
  if (row < span.first || row >= span.first + span.n) return;
  const int h = head / a.group, r = (row - span.first) * a.group + head % a.group;
  const Tile tile{b, span.first, span.n, seq_len(a.seqs.lens, b, a.seqs.cap), r / M * M};
  const int parts = parts_of(steps_of<D>(tile, M, a).n(), splits, least);
  if (parts == 1) return;
  const int64_t ld = static_cast<int64_t>(a.seqs.rows) * a.heads * (D + 4);
  const float* ws = a.work + (static_cast<int64_t>(row) * a.heads + head) * (D + 4);
  float top = -INFINITY;
  for (int i = lane; i < parts; i += 64) top = fmaxf(top, ws[i * ld + D]);
#pragma unroll
  for (int i = 1; i < 64; i *= 2) top = fmaxf(top, __shfl_xor(top, i));
  const float base = top == -INFINITY ? 0.0f : top;
  const int d = 4 * (lane % L);
  float4 y = make_float4(0, 0, 0, 0);
  float sum = 0;
#pragma unroll 4
  for (int i = lane / L; i < parts; i += R) {
    const float4 v = *reinterpret_cast<const float4*>(ws + i * ld + d);
    const float2 ml = *reinterpret_cast<const float2*>(ws + i * ld + D);
    const float w = __builtin_amdgcn_exp2f(ml.x - base);
    y.x += w * v.x;
    y.y += w * v.y;
    y.z += w * v.z;
    y.w += w * v.w;
    sum += w * ml.y;
  }
#pragma unroll
  for (int i = L; i < 64; i *= 2) {
    y.x += __shfl_xor(y.x, i);
    y.y += __shfl_xor(y.y, i);
    y.z += __shfl_xor(y.z, i);
    y.w += __shfl_xor(y.w, i);
    sum += __shfl_xor(sum, i);
  }
  const float vs = a.pool.vscale ? a.pool.vscale[h] : 1.0f;
  const float k = sum == 0 ? 0.0f : vs * __builtin_amdgcn_rcpf(sum);
  if (lane < L) store4<T>(a.y + row * a.ldy, head * D + d, a.out_f32, y.x * k, y.y * k, y.z * k, y.w * k);
}

struct Plan {
  int waves, splits;
  int64_t tiles;
};
constexpr int kLeast = 4;          // tiles of a part at least
Plan plan(int heads, int kv_heads, int hd, int rows, int seqs, int cap) {
  const int group = heads / kv_heads;
  Plan p;
  p.waves = 4;
  if (hd != 256 && (static_cast<int64_t>(rows) * heads) / 256 >= 512) p.waves = 8;
  const int m = 32 * p.waves;
  p.tiles = (static_cast<int64_t>(rows) * group + m - 1) / m + seqs;
  const int64_t wgs = std::max<int64_t>((static_cast<int64_t>(rows) * group + m - 1) / m, std::min(rows, seqs)) * kv_heads;
  const int64_t most = std::max(ceil_div(cap, tile_of(hd)) / kLeast, 1);
  p.splits = static_cast<int>(std::clamp<int64_t>(512 / wgs, 1, std::min<int64_t>(most, 64)));
  return p;
}

template <class T, bool E4M3, int D, int NW>
hipError_t run(const PagedAttnArgs& a, const Plan& p, hipStream_t s) {
  const dim3 grid(static_cast<uint32_t>(p.tiles * p.splits * a.pool.kv_heads));
  hipLaunchKernelGGL((paged_prompt_kernel<T, E4M3, D, NW>), grid, dim3(64 * NW), 0, s, a, p.splits, kLeast);
  if (p.splits > 1)
    hipLaunchKernelGGL((paged_prompt_join_kernel<T, D, 32 * NW>), dim3(a.seqs.rows, ceil_div(a.heads, 4)), dim3(256), 0, s, a,
                       p.splits, kLeast);
  return hipGetLastError();
}

template <class T, bool E4M3>
hipError_t go(const PagedAttnArgs& a, hipStream_t s) {
  const Plan p = plan(a.heads, a.pool.kv_heads, a.pool.hd, a.seqs.rows, a.seqs.seqs, a.seqs.cap);
  if (a.pool.hd == 256) return run<T, E4M3, 256, 4>(a, p, s);
  if (a.pool.hd == 128) return p.waves == 8 ? run<T, E4M3, 128, 8>(a, p, s) : run<T, E4M3, 128, 4>(a, p, s);
  return p.waves == 8 ? run<T, E4M3, 64, 8>(a, p, s) : run<T, E4M3, 64, 4>(a, p, s);
}

}  // namespace

int64_t paged_workspace(int heads, int kv_heads, int hd, int rows, int seqs, int cap, bool decode) {
  if (decode) return paged_decode_workspace(heads, kv_heads, hd, seqs, cap);
  const Plan p = plan(heads, kv_heads, hd, rows, seqs, cap);
  return p.splits > 1 ? int64_t{4} * p.splits * rows * heads * (hd + 4) : 0;
}

hipError_t launch_paged_attention(const PagedAttnArgs& a, hipStream_t s) {
  const bool e4m3 = a.pool.dtype == KV_E4M3;
  if (a.dtype == KV_BF16) return e4m3 ? go<Bf16, true>(a, s) : go<Bf16, false>(a, s);
  return e4m3 ? go<Fp16, true>(a, s) : go<Fp16, false>(a, s);
}

}  // namespace tars
