// Storing new tokens' K and V rows in the pages of their sequences.
//
// Row i of a sequence with n new rows and length len (they included) goes to position p = len - n + i: page
// table[p / page], slot p % page, each K / V head's hd elements at its own stride. A pool of the rows' own type gets
// their bits; an e4m3 pool gets e4m3(x / scale[head]): the quotient rounded to fp32, then to nearest even at e4m3's
// 3 mantissa bits, saturating at +-448 (NaN stays NaN). The quotient is float(x * (1 / scale)) in fp64: x and scale
// have 24 bits at most, so x / scale is at least 2^-49 of itself away from every tie of fp32, and the fp64 product is
// within 2^-52 of it.
//
// Rows behind the last sequence, rows before position 0 and rows whose page number is not in the pool are not stored.
//
// A row goes to one, two or four waves of a workgroup, 16 bytes of it per lane, so that its place is worked out in scalar
// registers and narrow rows share a workgroup. Measured for 8192 rows: one K / V head of 64 4.5 us (7.7 with a workgroup
// to each row), two of 128 5.8 us (9.6), eight of 128 13.6 us, 4.9 TB/s. Four rows to a lane, their loads issued before
// the place is known, came to 4.0, 6.1 and 12.9 us, but 3 to 7 % slower for wider rows and e4m3 pools.
// What bounds it: HBM for prompts (e4m3 pools also the fp64 conversions, a tenth of the time), and for single tokens
// (2.3 us) the chain launch -> starts -> length -> page number -> store, with the row's own loads issued beside it.
#include "paged_device.h"

namespace tars {
namespace {

constexpr int kThreads = 256;

template <class T>
__device__ __forceinline__ uint32_t e4m3x4(uint32_t a, uint32_t b, double inv) {
  float f[4] = {T::wide(a & 0xFFFFu), T::wide(a >> 16), T::wide(b & 0xFFFFu), T::wide(b >> 16)};
#pragma unroll
  for (float& x : f) {
    x = static_cast<float>(x * inv);
    x = x != x ? x : fminf(fmaxf(x, -448.0f), 448.0f);  // past 448 the conversion gives NaN
  }
  const uint32_t lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], lo, true);
}

template <class T, bool E4M3, int LANES>
__global__ __launch_bounds__(kThreads) void kv_append_kernel(KvAppendArgs a) {
  const int row = LANES == kThreads ? blockIdx.x : __builtin_amdgcn_readfirstlane((blockIdx.x * kThreads + threadIdx.x) / LANES);
  const KvSeqs& s = a.seqs;
  if (row >= s.rows) return;
  int b = row, len, i = 0, n = 1;
  if (s.starts) {
    b = seq_of_row(s, row);
    if (b >= s.seqs) return;
    const RowSpan r = seq_rows(s.starts, b, s.rows);
    i = row - r.first;
    n = r.n;
    if (i < 0 || i >= n) return;
  }
  len = seq_len(s.lens, b, s.cap);
  const int p = len - n + i;
  if (p < 0) return;
  const int page = s.table[b * s.ld_table + (p >> a.pool.page_shift)];
  if (page < 0 || page >= a.pool.pages) return;
  const int slot = p & ((1 << a.pool.page_shift) - 1);
  const int hd = a.pool.hd, chunks = a.pool.kv_heads * hd / 8;  // 8 elements each
  const char* kr = a.k + static_cast<int64_t>(row) * a.ldk;
  const char* vr = a.v + static_cast<int64_t>(row) * a.ldv;
  char* kd = a.pool.k + page * a.pool.k_page + slot * a.pool.k_slot;
  char* vd = a.pool.v + page * a.pool.v_page + slot * a.pool.v_slot;
  for (int c = threadIdx.x % LANES; c < 2 * chunks; c += LANES) {
    const bool is_v = c >= chunks;
    const int e = 8 * (is_v ? c - chunks : c), h = e / hd, d = e - h * hd;
    const uint4 x = *reinterpret_cast<const uint4*>((is_v ? vr : kr) + 2 * e);
    char* dst = is_v ? vd + h * a.pool.v_head : kd + h * a.pool.k_head;
    if constexpr (E4M3) {
      const float* sc = is_v ? a.pool.vscale : a.pool.kscale;
      const double inv = sc ? 1.0 / sc[h] : 1.0;
      *reinterpret_cast<uint2*>(dst + d) = make_uint2(e4m3x4<T>(x.x, x.y, inv), e4m3x4<T>(x.z, x.w, inv));
    } else {
      *reinterpret_cast<uint4*>(dst + 2 * d) = x;
    }
  }
}

template <class T, bool E4M3>
void go(const KvAppendArgs& a, hipStream_t s) {
  const int rows = a.seqs.rows, chunks = a.pool.kv_heads * a.pool.hd / 4;
  const dim3 block(kThreads);
  if (chunks <= 64) hipLaunchKernelGGL((kv_append_kernel<T, E4M3, 64>), dim3(ceil_div(rows, 4)), block, 0, s, a);
  else if (chunks <= 128) hipLaunchKernelGGL((kv_append_kernel<T, E4M3, 128>), dim3(ceil_div(rows, 2)), block, 0, s, a);
  else hipLaunchKernelGGL((kv_append_kernel<T, E4M3, 256>), dim3(rows), block, 0, s, a);
}

}  // namespace

hipError_t launch_kv_append(const KvAppendArgs& a, hipStream_t s) {
  if (a.pool.dtype != KV_E4M3) go<Bf16, false>(a, s);
  else if (a.dtype == KV_BF16) go<Bf16, true>(a, s);
  else go<Fp16, true>(a, s);
  return hipGetLastError();
}

}  // namespace tars
