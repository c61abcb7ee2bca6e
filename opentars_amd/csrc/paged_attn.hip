// Attention of packed prompt rows over the paged cache.
//
// The rows of one sequence that read one K / V head (its query heads' rows of every new token, token after token) are
// the columns of two matrix products, 32 to a wave:  S^T = K Q^T  and  O^T += V^T P^T.  A lane then holds scores of one
// row only: the running maximum and sum need one exchange between lane halves, and the numerators leave the softmax in
// the registers and order in which P^T's operand wants them (any order of a product's inner index will do, as long as
// V's operand has the same). K and V tiles of 64 positions pass through LDS, two tiles deep, loaded while the tile
// before is computed: 16-bit pools by direct loads whose 16-byte chunks are permuted within a row so that the reads of
// 32 rows' same chunk (K) and the transposing reads of 4 rows x 64 bytes (V) meet every bank once; e4m3 pools by direct
// loads of the bytes as they are, which the wave that loaded them widens into the tile's place a tile later.
//
// The scores come out of the product with the running maximum already taken off: it is the product's initial value. It
// is moved (and the sum and output rescaled) only when a score passes it by more than kSlack powers of two, so the
// numerators lie in [0, 2^kSlack]. They are rounded to q's type for the second product, whose operands they are: each is
// off by half a step at most, so an output by no more than half a step of the largest |V| it sees. Their sum is of the
// unrounded values, in fp32.
//
// Tiles at a row's own position, at a window's edge or with a page number outside the pool mask their scores. There a
// hidden position may hold anything: the tile of V is searched for infinities and NaN, which are zeros in the product. Where
// one was found, or an output is not finite, the outputs that V's infinities and NaN reach are set to their sum at the end.
//
// A workgroup has 128 rows, a wave 32 (16 for heads of 256); the last rows of a sequence, which see most, start first.
// With few rows their tiles are split over workgroups and joined by a second launch.
//
// What bounds it: the matrix units within the power limit. 8192 rows of 32 heads of 128, causal: 530 to 560 us from card to
// card, 0.98 to 1.04 PF/s (1.25 with zeros for data; the library's bf16 product of 8192 x 8192 x 8192 runs at 1.23 to 1.35); 2000 rows behind 14000 of
// 16 heads 268 us, 0.92 PF/s; heads of 256, 16 of them, 619 us, 0.89 PF/s, the reads of K and V from LDS beside the
// products, and 748 us over an e4m3 pool, whose widening adds to them. Few workgroups are bound by their number: two
// chunks of 2000 to 3001 rows, heads of 256 with a window of 1024 in e4m3, 316 on 256 CUs, 126 us; 400 rows of 16 heads
// of 64, seven tiles one after another, 12.6 us.
#include <algorithm>

#include "paged_device.h"

namespace tars {
namespace {

constexpr int tile_of(int hd) { return hd == 256 ? 32 : 64; }  // positions of a tile
constexpr float kSlack = 6.0f;     // numerators up to 64: their sums and products stay far from fp16's and fp32's limits
constexpr int kRowsWg = 128;       // rows of a workgroup

struct Tile {
  int b, first, rows, len;         // the sequence, its first row, its rows, its length
  int r0;                          // the first of the workgroup's rows among rows * group
};

// The workgroup's rows: `number` counts kRowsWg-row tiles over the sequences; within one the last comes first.
__device__ __forceinline__ Tile find_tile(const KvSeqs& s, int group, int number) {
  Tile t{-1, 0, 0, 0, 0};
  const int b = count_first(s.seqs, [&](int i) { return tile_first(s.starts, i + 1, s.rows, group, kRowsWg) <= number; });
  if (b >= s.seqs) return t;
  const RowSpan r = seq_rows(s.starts, b, s.rows);
  // among its tiles, also for starts that do not ascend
  const int tiles = ceil_div(r.n * group, kRowsWg), at = number - tile_first(s.starts, b, s.rows, group, kRowsWg);
  if (at < 0 || at >= tiles) return t;
  return {b, r.first, r.n, seq_len(s.lens, b, s.cap), (tiles - 1 - at) * kRowsWg};
}

// The same with the tiles of all sequences, 64 at most, in the order of their length: in steps of `step` positions up to
// the last row, no more than a window holds. A lane to a sequence; the length of tile `number` is found by bisection.
__device__ __forceinline__ Tile find_longest(const PagedAttnArgs& a, int number, int step) {
  const KvSeqs& s = a.seqs;
  const int b = threadIdx.x & 63, most = a.window == 0 ? INT32_MAX : a.window / step + kRowsWg / a.group / step + 3;
  RowSpan r{0, 0};
  int len = 0;
  if (b < s.seqs) {
    r = seq_rows(s.starts, b, s.rows);
    len = seq_len(s.lens, b, s.cap);
  }
  const auto count = [&](int x) { return x > most ? 0 : tiles_behind(x, len - r.n, r.n, a.group, kRowsWg, step); };
  const auto sum = [](int x) { return __builtin_amdgcn_readfirstlane(group_sum<64>(x)); };
  if (number >= sum(count(0))) return {-1, 0, 0, 0, 0};
  int lo = 0, hi = __builtin_amdgcn_readfirstlane(group_max<64>(static_cast<uint32_t>(ceil_div(len, step)))) + 2;
  while (hi - lo > 1) {  // count(lo) > number >= count(hi)
    const int x = (lo + hi) / 2;
    if (sum(count(x)) > number) lo = x;
    else hi = x;
  }
  const int longer = count(lo + 1), alike = count(lo) - longer;
  const int upto = inclusive_sum(alike), at = number - sum(longer);
  const int hit = __builtin_ctzll(__ballot(upto > at));
  const auto of = [&](int x) { return __builtin_amdgcn_readlane(x, hit); };
  const int tile = of(ceil_div(r.n * a.group, kRowsWg) - longer - 1 - (at - (upto - alike)));
  return {__builtin_amdgcn_readfirstlane(hit), of(r.first), of(r.n), of(len), tile * kRowsWg};
}

template <int D>
__device__ __forceinline__ Steps steps_of(const Tile& t, int m, const PagedAttnArgs& a) {
  const int p0 = t.len - t.rows;
  return visible_steps(p0 + t.r0 / a.group, p0 + (min(t.r0 + m, t.rows * a.group) - 1) / a.group, t.len, a.window, a.sinks,
                       tile_of(D));
}

// Tiles of a part, and the parts of n tiles.
__device__ __forceinline__ int parts_of(int n, int splits, int least) { return max(min(splits, n / least), 1); }

// Rows of a wave, columns of its products. 32 read each operand of K and V half as often, and heads of 256 at 32 rows need
// 128 registers for the output alone: they take 16 rows, on twice the waves (8192 rows of 16 heads 619 us; at 32 rows,
// one wave to a SIMD, 933 us).
constexpr int wave_rows(int hd) { return hd == 256 ? 16 : 32; }
template <class T, int R>
struct Product;
template <class T>
struct Product<T, 32> {  // 32 x 32 x 16
  typedef v16f Acc;
  static __device__ __forceinline__ Acc go(uint4 a, uint4 b, Acc c) { return T::mfma_32x32x16(a, b, c); }
};
template <class T>
struct Product<T, 16> {  // 16 x 16 x 32
  typedef v4f Acc;
  static __device__ __forceinline__ Acc go(uint4 a, uint4 b, Acc c) { return T::mfma_16x16x32(a, b, c); }
};

// Byte offset of 16-byte chunk c of row k in a tile.
template <int D>
__device__ __forceinline__ int k_at(int k, int c) {
  return k * 2 * D + ((c ^ (D == 64 ? (k >> 1) & 7 : k & 15)) << 4);
}
template <int D>
__device__ __forceinline__ int v_at(int k, int c) {
  return k * 2 * D + ((c ^ (D == 64 ? (k & 2) << 1 : D == 128 ? (k & 3) << 2 : (k & 7) << 1)) << 4);
}

__device__ __forceinline__ uint32_t max_halves(uint32_t x, uint32_t y) {
  typedef uint16_t v2s __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(v2s, x), __builtin_bit_cast(v2s, y)));
}

template <class T, bool E4M3, int D>
__global__ __launch_bounds__(64 * kRowsWg / wave_rows(D), 2) void paged_prompt_kernel(PagedAttnArgs a, int splits, int least, bool sorted) {
  // R rows of a wave, N values of an accumulator; products of R x R x G, whose R positions make kHalves of a tile's scores,
  // NT of the columns, and whose G make KS of the columns and kSteps of the positions.
  constexpr int M = kRowsWg, R = wave_rows(D), kWaves = M / R, G = 512 / R, N = R * R / 64, KS = D / G, NT = D / R;
  constexpr int kTile = tile_of(D), kBlocks = kTile / 16, kHalves = kTile / R, kSteps = kTile / G;
  typedef Product<T, R> Mul;
  typedef typename Mul::Acc Acc;
  constexpr int kBytes = kTile * D * 2;                 // a tile of K or V
  // K's stages, V's, and for e4m3 what the loads bring: of K, of V
  __shared__ __attribute__((aligned(1024))) char lds[4 + E4M3][kBytes];
  bool spoiled = false;
  const int lane = threadIdx.x & 63, col = lane % R, part = lane / R;  // of N / 4 fours of positions, columns: 4 part + e
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = blockIdx.x % a.pool.kv_heads, rest = blockIdx.x / a.pool.kv_heads, split = rest % splits;
  const Tile tile = sorted ? find_longest(a, rest / splits, kTile) : find_tile(a.seqs, a.group, rest / splits);
  if (tile.b < 0) return;
  const Steps steps = steps_of<D>(tile, M, a);
  const int n = steps.n(), parts = parts_of(n, splits, least);
  if (split >= parts) return;
  const int per = ceil_div(n, parts), t0 = min(split * per, n), t1 = min(t0 + per, n);

  // the rows of this wave: row r of the sequence's rows * group is token r / group, query head r % group
  const int total = tile.rows * a.group, w0 = tile.r0 + R * wave, r = min(w0 + col, total - 1);
  const int token = r / a.group, head = h * a.group + r - token * a.group;
  const int p0 = tile.len - tile.rows, p = p0 + token;
  const int plo = p0 + tile.r0 / a.group, phi = p0 + (min(tile.r0 + M, total) - 1) / a.group;

  uint4 qf[KS];
  const char* q = a.q + (tile.first + token) * a.ldq + 2 * D * head + 16 * part;
#pragma unroll
  for (int s = 0; s < KS; ++s) qf[s] = *reinterpret_cast<const uint4*>(q + 2 * G * s);
  const float sc = score_scale(a, h);

  const int shift = a.pool.page_shift, mask = (1 << shift) - 1, last = max(tile.len - 1, 0) >> shift;
  const char* kbase = a.pool.k + h * a.pool.k_head;
  const char* vbase = a.pool.v + h * a.pool.v_head;

  // Where the blocks of 16 positions lie: lane x holds the addresses of block x % kBlocks of tile from + x / kBlocks, of
  // page 0 for a page number outside the pool, whose bit of `in` is 0. The loads go at most two tiles past the one
  // computed; the addresses move on by half their tiles, the page numbers asked for two tiles before.
  constexpr int kHeld = 64 / kBlocks, kMove = kHeld / 2;
  int from = 0, coming = 0;
  uint64_t k_held = 0, v_held = 0, in = 0;
  auto position_of = [&](int i) __attribute__((always_inline)) {
    return steps.at(min(i + lane / kBlocks, t1 - 1)) * kTile + 16 * (lane % kBlocks);
  };
  auto numbers = [&](int i) __attribute__((always_inline)) {
    return a.seqs.table[tile.b * a.seqs.ld_table + min(position_of(i) >> shift, last)];
  };
  auto hold = [&](int i, int number) __attribute__((always_inline)) {
    const bool good = static_cast<uint32_t>(number) < static_cast<uint32_t>(a.pool.pages);
    const int64_t page = good ? number : 0, slot = position_of(i) & mask;
    from = i;
    in = __ballot(good);
    k_held = reinterpret_cast<uint64_t>(kbase) + page * a.pool.k_page + slot * a.pool.k_slot;
    v_held = reinterpret_cast<uint64_t>(vbase) + page * a.pool.v_page + slot * a.pool.v_slot;
  };
  auto block_of = [&](uint64_t held, int i, int block) __attribute__((always_inline)) {
    const int x = (i - from) * kBlocks + block;
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(held), x);
    const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(held >> 32), x);
    return reinterpret_cast<const char*>(static_cast<uint64_t>(hi) << 32 | lo);
  };
  auto in_pool = [&](int i) __attribute__((always_inline)) {
    return static_cast<int>(in >> ((i - from) * kBlocks)) & ((1 << kBlocks) - 1);
  };

  // Loading a tile: a load instruction moves 1 KiB = kRows rows, lane l the 16 bytes at 16 l; a
  // wave's loads are kSpan rows apart. Rows of e4m3 come as they are and are widened into the stage by the wave that
  // loaded them, a tile later.
  constexpr int kRow = E4M3 ? D : 2 * D, kRows = 1024 / kRow, kSpan = kWaves * kRows, kTake = kTile / kSpan;
  constexpr int kSame = kSpan >= 16 ? 1 : 16 / kSpan;                        // loads with offsets of their own
  uint32_t k_off[kSame], v_off[kSame];
#pragma unroll
  for (int x = 0; x < kSame; ++x) {
    const int row = (wave * kRows + x * kSpan) % 16 + lane / (kRow / 16), c = lane % (kRow / 16);
    k_off[x] = row * static_cast<uint32_t>(a.pool.k_slot) + (E4M3 ? 16 * c : k_at<D>(row, c) & (2 * D - 1));
    v_off[x] = row * static_cast<uint32_t>(a.pool.v_slot) + (E4M3 ? 16 * c : v_at<D>(row, c) & (2 * D - 1));
  }
  const uint32_t stages = lds_addr(lds[0]) + 1024 * wave;
  // Piece x of K's (V's) tile to byte `to` of LDS; behind the last tile, of the last one again, to where nobody reads it.
  auto load = [&](int tile, uint32_t to, bool is_v, int x) __attribute__((always_inline)) {
    const char* at = block_of(is_v ? v_held : k_held, min(tile, t1 - 1), (wave * kRows + x * kSpan) >> 4);
    ring_load16_free(at, is_v ? v_off[x % kSame] : k_off[x % kSame], stages + to + 1024 * kWaves * x);
  };
  constexpr int kRaw = 4 * kBytes;                              // e4m3: where K arrives; V kBytes / 2 behind
  // What has arrived of K (and of V) into their stages; the arrival rows are free for the next loads then.
  auto widen = [&](int k_stage, int v_stage, bool with_v) __attribute__((always_inline)) {
    if constexpr (E4M3) {
      int thread = threadIdx.x;
      asm volatile("" : "+v"(thread) : : "memory");  // addresses formed here, rather than in registers all the way
      uint4 w[2][kTake];
#pragma unroll
      for (int v = 0; v < 1 + with_v; ++v)
#pragma unroll
        for (int x = 0; x < kTake; ++x)
          w[v][x] = *reinterpret_cast<const uint4*>(lds[0] + kRaw + v * (kBytes / 2) + 16 * (x * 64 * kWaves + thread));
#pragma unroll
      for (int v = 0; v < 1 + with_v; ++v)
#pragma unroll
        for (int x = 0; x < kTake; ++x) asm volatile("" : "+v"(w[v][x].x), "+v"(w[v][x].y), "+v"(w[v][x].z), "+v"(w[v][x].w));
#pragma unroll
      for (int v = 0; v < 1 + with_v; ++v)
#pragma unroll
        for (int x = 0; x < kTake; ++x) {
          const int at = x * 64 * kWaves + thread, k = at / (D / 16), c = at % (D / 16);
          const uint4 u = w[v][x];
          char* to = lds[v ? v_stage : k_stage];
          *reinterpret_cast<uint4*>(to + (v ? v_at<D>(k, 2 * c) : k_at<D>(k, 2 * c))) =
              make_uint4(T::template from_e4m3<false>(u.x), T::template from_e4m3<true>(u.x),
                         T::template from_e4m3<false>(u.y), T::template from_e4m3<true>(u.y));
          *reinterpret_cast<uint4*>(to + (v ? v_at<D>(k, 2 * c + 1) : k_at<D>(k, 2 * c + 1))) =
              make_uint4(T::template from_e4m3<false>(u.z), T::template from_e4m3<true>(u.z),
                         T::template from_e4m3<false>(u.w), T::template from_e4m3<true>(u.w));
        }
    }
  };
  auto meet = [&]() __attribute__((always_inline)) {
    asm volatile("" : : : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
  };

  // m: the maximum taken off, in units of the raw scores; bound: a score (with m taken off) above it moves m
  float l = 0, bound = -INFINITY;
  Acc minus, o[NT];
#pragma unroll
  for (int i = 0; i < N; ++i) minus[i] = 0;
#pragma unroll
  for (int t = 0; t < NT; ++t) o[t] = minus;
  const float slack = kSlack * __builtin_amdgcn_rcpf(sc);
  // Lane offsets of the reads, the permutation of the chunks included: row col, chunk `part` of K (product k's is that
  // offset with 2 G k turned over); V's transposing read of 4 rows x 16 columns (column tile t: with 2 R t turned over).
  const uint32_t k_lane = lds_addr(lds[0]) + k_at<D>(col, part);
  const uint32_t v_lane = lds_addr(lds[0]) + v_at<D>(4 * part + (lane % 16 >> 2), lane % R / 16 * 2 + (lane % 4 >> 1)) + lane % 2 * 8;
  Acc s0[kHalves], s1[kHalves];
  uint32_t pf[kTile * R / 128];

  // The steps [whole0, whole0 + wholes) are the ones that every row of the workgroup sees whole, their pages being in the
  // pool (with a window, the steps of the first tokens count as not whole).
  const int whole0 = steps.a + (a.window == 0 ? 0 : max(phi - a.window + kTile - steps.b0 * kTile, 0) / kTile);
  const int wholes = max(steps.a + (plo + 1) / kTile - steps.b0 - whole0, 0);
  auto is_whole = [&](int i) __attribute__((always_inline)) {
    return static_cast<uint32_t>(i - whole0) < static_cast<uint32_t>(wholes) && (~in == 0 || in_pool(i) == (1 << kBlocks) - 1);
  };
  // one operand of V^T: positions G k + (G / 2) x + 4 part + 0 .. 3 for x = 0, 1, column col of column tile t
  auto v_operand = [&](uint32_t vt, int k, int t) __attribute__((always_inline)) {
    typedef __attribute__((address_space(3))) v4s* P;
    const uint32_t at = (vt ^ (2 * R * t)) + 2 * G * k * D;
    const uint2 lo = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(at)));
    const uint2 hi = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(at + G * D)));
    return make_uint4(lo.x, lo.y, hi.x, hi.y);
  };
  auto numerators = [&](int k) __attribute__((always_inline)) {
    return make_uint4(pf[4 * k], pf[4 * k + 1], pf[4 * k + 2], pf[4 * k + 3]);
  };

  // Hidden positions of a tile that is not whole may hold anything: V's infinities and NaN become zeros (whichever wave
  // meets them), to be added at the end to the rows that see them.
  auto clean = [&](int i) __attribute__((always_inline)) {
    char* vt = lds[2 + (i & 1)];
    uint32_t bad = 0;
#pragma unroll 2
    for (int x = 0; x < kBytes / 1024; ++x) {
      const uint4 v = *reinterpret_cast<const uint4*>(vt + 1024 * x + 16 * lane);
      bad = max_halves(max_halves(bad, max_halves(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu)),
                       max_halves(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu));
    }
    if (__ballot(not_finite<T>(bad) != 0)) {
      spoiled = true;
#pragma unroll 1
      for (int x = lane; x < kBytes / 4; x += 64) {
        uint32_t* at = reinterpret_cast<uint32_t*>(vt) + x;
        *at &= ~not_finite<T>(*at);
      }
    }
  };
  // S^T = K Q^T, the maximum taken off: kQk products, whose operands are read kLead ahead.
  constexpr int kPv = kSteps * NT, kQk = KS * kHalves, kLead = D == 256 ? 8 : 4, kPairs = kTile * R / 128;
  auto k_operand = [&](uint32_t kt, int x) __attribute__((always_inline)) {
    typedef uint32_t v4u __attribute__((ext_vector_type(4)));
    const v4u v = *(__attribute__((address_space(3))) const v4u*)((kt ^ (2 * G * (x / kHalves))) + 2 * R * D * (x % kHalves));
    return make_uint4(v[0], v[1], v[2], v[3]);
  };
  auto score = [&](Acc (&s)[kHalves], int x, uint4 f) __attribute__((always_inline)) {
    s[x % kHalves] = Mul::go(f, qf[x / kHalves], x < kHalves ? minus : s[x % kHalves]);
  };
  // The softmax of tile i's scores s, and between its steps the products for the next tile's scores (behind the last
  // tile: of whatever the stage holds, not used).
  auto softmax_and_scores = [&](int i, bool whole, Acc (&s)[kHalves], Acc (&next)[kHalves]) __attribute__((always_inline)) {
    const uint32_t kt = k_lane + ((i + 1) & 1) * kBytes;
    if (!whole) {
      const int k0 = steps.at(i) * kTile, ok = in_pool(i);
#pragma unroll
      for (int t = 0; t < kHalves; ++t)
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const int k = R * t + (e >> 2) * (256 / R) + 4 * part + (e & 3);
          const bool seen = sees(p, k0 + k, a.window, a.sinks) && (ok >> (k >> 4) & 1);
          s[t][e] = seen ? s[t][e] : -INFINITY;
        }
    }
    issue_fence();
    uint4 f[kLead];
#pragma unroll
    for (int x = 0; x < kLead; ++x) f[x] = k_operand(kt, x);
    auto at = [&](Acc (&v)[kHalves], int e) __attribute__((always_inline)) -> float { return v[e / N][e % N]; };
    constexpr int kValues = kTile * R / 64;  // of a lane
    float top = at(s, 0);
#pragma unroll
    for (int x = 0; x < kQk; ++x) {
      score(next, x, f[x % kLead]);
      if (x + kLead < kQk) f[x % kLead] = k_operand(kt, x + kLead);
      constexpr int kTop = kHalves;  // the maximum: once every half's products are under way
      if (x == kTop - 1) {
#pragma unroll
        for (int e = 1; e < kValues / 2; ++e) top = fmaxf(top, at(s, e));
      } else if (x == kTop) {
#pragma unroll
        for (int e = kValues / 2; e < kValues; ++e) top = fmaxf(top, at(s, e));
        top = over_row<R>(top, [](float x, float y) { return fmaxf(x, y); });
        // By row, not for the wave as a whole: the compiler then scales the output in place, where it copied all of it on
        // the way past a uniform branch.
        if (top > bound) {
          // the first scores that a row sees set m from nothing: its sum and output are 0 (or not finite) then
          const float by = top, keep = bound == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(-by * sc);
          l *= keep;
          bound = slack;
#pragma unroll
          for (int e = 0; e < N; ++e) minus[e] -= by;
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < N; ++e) o[t][e] *= keep;
#pragma unroll
          for (int e = 0; e < kValues; ++e) {
            s[e / N][e % N] -= by;
            next[e / N][e % N] -= by;  // under way since the old maximum
          }
        }
      } else if (x > kTop) {
#pragma unroll
        for (int e = (x - kTop - 1) * kPairs / (kQk - kTop - 1); e < (x - kTop) * kPairs / (kQk - kTop - 1); ++e) {
          const float y = __builtin_amdgcn_exp2f(at(s, 2 * e) * sc), z = __builtin_amdgcn_exp2f(at(s, 2 * e + 1) * sc);
          l += y + z;
          pf[e] = T::pair(y, z);
          asm volatile("" : "+v"(pf[e]));  // here, not where it is used
        }
      }
      constexpr int kEvery = kQk / (2 * kTake);
      static_assert(kEvery > 0, "a load or none behind each product");
      if (!E4M3 && x % kEvery == kEvery - 1 && x / kEvery < 2 * kTake) {
        if (x / kEvery < kTake) load(i + 2, (i & 1) * kBytes, false, x / kEvery);
        else load(i + 1, (2 + ((i + 1) & 1)) * kBytes, true, x / kEvery - kTake);
      }
      issue_fence();
    }
  };
  // O^T += V^T P^T of tile i
  auto output = [&](int i) __attribute__((always_inline)) {
    const uint32_t vt = v_lane + (2 + (i & 1)) * kBytes;
    uint4 f[kLead];
    issue_fence();
#pragma unroll
    for (int x = 0; x < kLead; ++x) f[x] = v_operand(vt, x / NT, x % NT);
#pragma unroll
    for (int x = 0; x < kPv; ++x) {
      o[x % NT] = Mul::go(f[x % kLead], numerators(x / NT), o[x % NT]);
      if (x + kLead < kPv) f[x % kLead] = v_operand(vt, (x + kLead) / NT, (x + kLead) % NT);
      issue_fence();
    }
  };

  // A tile's softmax runs between the products for the next tile's scores: vector work that hides half the matrix work.
  // Its product with V is matrix work alone, next to which the SIMD runs the other workgroup's wave. Between the barriers
  // of tiles i - 1 and i K's tile i + 1 and V's tile i are read, K's i + 2 and V's i + 1 loaded, into the stages read
  // before.
  if (t0 < t1) {
    hold(t0, numbers(t0));
    auto arrive = [&](int k_tile, int v_tile) __attribute__((always_inline)) {  // e4m3
#pragma unroll
      for (int x = 0; x < kTake; ++x) load(k_tile, kRaw, false, x);
#pragma unroll
      for (int x = 0; x < kTake; ++x) load(v_tile, kRaw + kBytes / 2, true, x);
    };
    // K's tiles t0 and t0 + 1, V's tile t0
    if constexpr (E4M3) {
      arrive(t0, t0);
      wait_vmcnt<0>();
      widen(t0 & 1, 2 + (t0 & 1), true);
      arrive(t0 + 1, t0 + 1);
      wait_vmcnt<0>();
      widen((t0 + 1) & 1, 0, false);
      wait_lgkm0();
      arrive(t0 + 2, t0 + 1);
    } else {
#pragma unroll
      for (int x = 0; x < kTake; ++x) load(t0, (t0 & 1) * kBytes, false, x);
#pragma unroll
      for (int x = 0; x < kTake; ++x) load(t0 + 1, ((t0 + 1) & 1) * kBytes, false, x);
#pragma unroll
      for (int x = 0; x < kTake; ++x) load(t0, (2 + (t0 & 1)) * kBytes, true, x);
      wait_vmcnt<0>();
    }
    meet();
#pragma unroll
    for (int x = 0; x < kQk; ++x) score(s0, x, k_operand(k_lane + (t0 & 1) * kBytes, x));
    meet();
    auto turn = [&](int i, Acc (&s)[kHalves], Acc (&next)[kHalves]) __attribute__((always_inline)) {
      if (i - from == kMove - 2) coming = numbers(from + kMove);
      if (i - from == kMove) hold(i, coming);
      const bool whole = is_whole(i);
      if constexpr (E4M3) {
        wait_vmcnt<0>();
        widen(i & 1, 2 + ((i + 1) & 1), true);
        arrive(i + 3, i + 2);
      }
      softmax_and_scores(i, whole, s, next);
      if (!whole) clean(i);
      output(i);
      if constexpr (!E4M3) wait_vmcnt<0>();
      else wait_lgkm0();
      meet();
    };
    for (int i = t0;;) {
      turn(i, s0, s1);
      if (++i == t1) break;
      turn(i, s1, s0);
      if (++i == t1) break;
    }
    wait_vmcnt<0>();  // the loads behind the last tile, before the workgroup's LDS goes to another
  }

  l = over_row<R>(l, [](float x, float y) { return x + y; });
  int r_out = w0 + col;
  asm volatile("" : "+v"(r_out));  // the row's numbers again, rather than in registers all the way
  const int token_out = r_out / a.group, head_out = h * a.group + r_out - token_out * a.group;
  float* ws = a.work + static_cast<int64_t>(split) * a.seqs.rows * a.heads * (D + 4);
  if (r_out < total) {
    if (parts == 1) {
      const float vs = E4M3 && a.pool.vscale ? a.pool.vscale[h] : 1.0f;
      const float k = l == 0 ? 0.0f : vs * __builtin_amdgcn_rcpf(l);
      char* y = a.y + (tile.first + token_out) * a.ldy;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < N; e += 4)
          store4<T>(y, head_out * D + R * t + e * (64 / R) + 4 * part, a.out_f32, o[t][e] * k, o[t][e + 1] * k, o[t][e + 2] * k,
                    o[t][e + 3] * k, !E4M3);
    } else {
      float* at = ws + (static_cast<int64_t>(tile.first + token_out) * a.heads + head_out) * (D + 4);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < N; e += 4)
          *reinterpret_cast<float4*>(at + R * t + e * (64 / R) + 4 * part) = make_float4(o[t][e], o[t][e + 1], o[t][e + 2], o[t][e + 3]);
      // none seen: the sum is 0 and the maximum counts for nothing
      if (part == 0) *reinterpret_cast<float2*>(at + D) = make_float2(l == 0 ? -INFINITY : -minus[0], l);
    }
  }
  // In whole tiles V's infinities and NaN met the numerators, some of them rounded to 0: the outputs they reached are not finite.
  spoiled |= not_all_finite(o);
  __syncthreads();
  if (threadIdx.x == 0) *reinterpret_cast<volatile int*>(lds[0]) = 0;
  __syncthreads();
  if (spoiled) *reinterpret_cast<volatile int*>(lds[0]) = 1;
  __syncthreads();
  if (*reinterpret_cast<volatile int*>(lds[0]) == 0) return;

  float* sums = reinterpret_cast<float*>(lds[1]);
  sums[R * wave + col] = l;
  __syncthreads();
  const auto part_row = [&](int x) {
    const int t = x / a.group;
    return parts > 1 ? ws + (static_cast<int64_t>(tile.first + t) * a.heads + h * a.group + x - t * a.group) * (D + 4) : nullptr;
  };
  const auto sound = [&](int x) { return parts > 1 || sums[x - tile.r0] < INFINITY; };
  set_unfinite<T, E4M3, D, kTile>(
      a, tile.b, h, tile.len, [&](int i) { return steps.at(i); }, t0, t1, p0, tile.first, tile.r0, min(M, total - tile.r0), part_row, sound);
}

// Joins the parts of rows whose tiles were split: a workgroup per row and 4 heads, D / 4 lanes of a wave for a head's
// row, the wave's other lanes for other parts.
template <class T, int D>
__global__ __launch_bounds__(256) void paged_prompt_join_kernel(PagedAttnArgs a, int splits, int least) {
  constexpr int L = D / 4, R = 64 / L;
  const int row = blockIdx.x, lane = threadIdx.x & 63;
  const int head = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = seq_of_row(a.seqs, row);
  if (b >= a.seqs.seqs || head >= a.heads) return;
  const RowSpan span = seq_rows(a.seqs.starts, b, a.seqs.rows);
  if (row < span.first || row >= span.first + span.n) return;
  const int h = head / a.group, r = (row - span.first) * a.group + head % a.group;
  const Tile tile{b, span.first, span.n, seq_len(a.seqs.lens, b, a.seqs.cap), r / kRowsWg * kRowsWg};
  const int parts = parts_of(steps_of<D>(tile, kRowsWg, a).n(), splits, least);
  if (parts == 1) return;
  const int64_t ld = static_cast<int64_t>(a.seqs.rows) * a.heads * (D + 4);
  const float* ws = a.work + (static_cast<int64_t>(row) * a.heads + head) * (D + 4);
  float top = -INFINITY;
  for (int i = lane; i < parts; i += 64) top = fmaxf(top, ws[i * ld + D]);
#pragma unroll
  for (int i = 1; i < 64; i *= 2) top = fmaxf(top, __shfl_xor(top, i));
  const float base = top == -INFINITY ? 0.0f : top, sc = score_scale(a, h);
  const int d = 4 * (lane % L);
  float4 y = make_float4(0, 0, 0, 0);
  float sum = 0;
#pragma unroll 4
  for (int i = lane / L; i < parts; i += R) {
    const float4 v = *reinterpret_cast<const float4*>(ws + i * ld + d);
    const float2 ml = *reinterpret_cast<const float2*>(ws + i * ld + D);
    const float w = __builtin_amdgcn_exp2f((ml.x - base) * sc);
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
  join_unfinite(y, parts, [&](int p) { return *reinterpret_cast<const float4*>(ws + p * ld + d); });
  const float vs = a.pool.vscale ? a.pool.vscale[h] : 1.0f;
  const float k = sum == 0 ? 0.0f : vs * __builtin_amdgcn_rcpf(sum);
  if (lane < L) store4<T>(a.y + row * a.ldy, head * D + d, a.out_f32, y.x * k, y.y * k, y.z * k, y.w * k, !a.pool.vscale);
}

// Tiles start in the order of their length where more workgroups come than run at once, 512, and up to 64 sequences bring
// them: 11 prompts of 60 to 2000 rows 109 us (121 in the order of the sequences), with heads of 256 130 (156); 60 of up to
// 300 rows 69 (75), four of up to 4000 229 (230). The prompts of one sequence come last tile first in either order.
struct Plan {
  int splits;
  int64_t tiles;
  bool sorted;
};
// Few workgroups are split until there are up to 512, two on every CU, in parts of kLeast tiles or more: 256 rows of 16
// heads behind 30000 85 us (up to 256: 100, 1024: 108), 40 behind 3000 20.3 us (8 tiles: 23.1). Tables of up to 8 tiles are
// not split (480 rows of 16 heads of 64: 14.2 us in one, 18.7 in two). Past them the second launch pays the sooner the fewer
// workgroups there are: 16 of them (80 rows of 16 heads of 128) in 9 tiles 19.1 us and 21.5 in one part, in 24 20.9 and 38.4;
// 64 (480 rows) in 9 25.1 and 21.8, in 15 26.9 and 27.2; 120 (480 rows of 32 heads) in 11 33.8 and 23.9, in 24 as long: there
// the rule costs more than it gives. Of heads of 256, whose workgroups have twice the waves, a CU holds one: 128 rows of 16
// heads behind 8000 41 us (up to 512: 58), 256 behind 30000 175 us (193).
constexpr int resident(int hd) { return hd == 256 ? 256 : 512; }
constexpr int kLeast = 4;
Plan plan(int heads, int kv_heads, int hd, int rows, int seqs, int cap) {
  const int group = heads / kv_heads;
  const int64_t full = (static_cast<int64_t>(rows) * group + kRowsWg - 1) / kRowsWg;
  const int64_t wgs = std::max<int64_t>(full, std::min(rows, seqs)) * kv_heads;
  const int tiles = ceil_div(cap, tile_of(hd));
  const int64_t most = tiles <= 2 * kLeast ? 1 : tiles / kLeast;
  return {static_cast<int>(std::clamp<int64_t>(resident(hd) / wgs, 1, std::min<int64_t>(most, 64))), full + seqs, wgs > 512 && seqs > 1 && seqs <= 64};
}

template <class T, bool E4M3, int D>
hipError_t run(const PagedAttnArgs& a, hipStream_t s) {
  const Plan p = plan(a.heads, a.pool.kv_heads, D, a.seqs.rows, a.seqs.seqs, a.seqs.cap);
  const dim3 grid(static_cast<uint32_t>(p.tiles * p.splits * a.pool.kv_heads));
  hipLaunchKernelGGL((paged_prompt_kernel<T, E4M3, D>), grid, dim3(64 * kRowsWg / wave_rows(D)), 0, s, a, p.splits, kLeast, p.sorted);
  if (p.splits > 1)
    hipLaunchKernelGGL((paged_prompt_join_kernel<T, D>), dim3(a.seqs.rows, ceil_div(a.heads, 4)), dim3(256), 0, s, a, p.splits, kLeast);
  return hipGetLastError();
}

template <class T, bool E4M3>
hipError_t go(const PagedAttnArgs& a, hipStream_t s) {
  return a.pool.hd == 64 ? run<T, E4M3, 64>(a, s) : a.pool.hd == 128 ? run<T, E4M3, 128>(a, s) : run<T, E4M3, 256>(a, s);
}

}  // namespace

// Sequences of 32 columns or fewer on average go to the kernel for few rows: 16 caches of 3k to 16k with 20 columns 134 us
// and 148 here, with 32 143 and 150, with 64 233 and 157. So do rows that fill a quarter at most of a table for 257 to 512
// positions, where this kernel's tiles follow one another in few workgroups and that one has one for each 32 (16) columns: 20 to
// 77 rows behind 300 to 470, in four layouts of heads, 10.6 to 17.8 us there and 11.7 to 20.4 here, each of them faster there
// (77 behind 300, 16 heads of 64: 10.8 and 14.1; of 128: 13.6 and 17.7; 8 of 256: 15.2 and 19.0). The edges are not where the
// two kernels meet: 77 rows behind 200 in a table for 304 positions, more than a quarter of it, come here and take 13.2, 10.6
// there. 200 rows behind 300 (19.8 and 20.9 there), 77 behind 700 (15.7 and 16.9) and rows with no past (400: 12.6 and 14.9)
// are faster here.
constexpr int kShort = 256, kShortCap = 512, kShortWgs = 512;
static bool few_rows(int group, int kv_heads, int hd, int rows, int seqs, int cap) {
  const int64_t columns = static_cast<int64_t>(rows) * group;
  return columns <= 32ll * seqs || (cap > kShort && cap <= kShortCap && 4ll * rows <= static_cast<int64_t>(cap) * seqs &&
                                    (columns / (hd == 256 ? 16 : 32) + seqs) * kv_heads <= kShortWgs);
}

int64_t paged_workspace(int heads, int kv_heads, int hd, int rows, int seqs, int cap, bool decode) {
  if (decode || few_rows(heads / kv_heads, kv_heads, hd, rows, seqs, cap)) return paged_rows_workspace(heads, kv_heads, hd, rows, seqs, cap);
  const Plan p = plan(heads, kv_heads, hd, rows, seqs, cap);
  return p.splits > 1 ? int64_t{4} * p.splits * rows * heads * (hd + 4) : 0;
}

hipError_t launch_paged_attention(const PagedAttnArgs& a, hipStream_t s) {
  if (few_rows(a.group, a.pool.kv_heads, a.pool.hd, a.seqs.rows, a.seqs.seqs, a.seqs.cap)) return launch_paged_rows(a, s);
  const bool e4m3 = a.pool.dtype == KV_E4M3;
  if (a.dtype == KV_BF16) return e4m3 ? go<Bf16, true>(a, s) : go<Bf16, false>(a, s);
  return e4m3 ? go<Fp16, true>(a, s) : go<Fp16, false>(a, s);
}

}  // namespace tars
