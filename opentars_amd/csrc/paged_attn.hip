// Attention over the paged key / value cache: y = softmax(scale q K^T) V over the positions a row sees, one pass with
// a running maximum m and sum l:
//   s_j = scale * kscale * (q . k_j),  m' = max(m, s_j),  l' = l e^(m - m') + e^(s_j - m'),
//   o' = o e^(m - m') + e^(s_j - m') v_j,  y = vscale * o / l.
// A wave per row and query head: lane = key for the scores, lane = column for P V. Every product and sum in fp32.
#include "paged_device.h"

namespace tars {
namespace {

constexpr int kWaves = 4;
constexpr float kLog2e = 1.44269504f;

__device__ __forceinline__ float e4m3_wide(uint32_t byte) {
  return Bf16::wide(Bf16::from_e4m3<false>(byte) & 0xFFFFu);
}

template <class T, bool E4M3>
__device__ __forceinline__ float element(const char* row, int d) {
  if constexpr (E4M3) return e4m3_wide(reinterpret_cast<const uint8_t*>(row)[d]);
  else return T::wide(reinterpret_cast<const uint16_t*>(row)[d]);
}

template <class T, bool E4M3, int D>
__global__ __launch_bounds__(64 * kWaves) void paged_rows_kernel(PagedAttnArgs a) {
  __shared__ float qs[kWaves][D];
  const KvSeqs& s = a.seqs;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int row = blockIdx.x, head = blockIdx.y * kWaves + wave;
  if (head >= a.heads) return;
  int b = row, p;
  if (s.starts) {
    b = seq_of_row(s, row);
    if (b >= s.seqs) return;
    const RowSpan r = seq_rows(s.starts, b, s.rows);
    if (row < r.first || row >= r.first + r.n) return;
    p = seq_len(s.lens, b, s.cap) - r.n + (row - r.first);
  } else {
    p = seq_len(s.lens, b, s.cap) - 1;
  }
  const int h = head / a.group;
  const float c = a.scale * kLog2e * (E4M3 && a.pool.kscale ? a.pool.kscale[h] : 1.0f);
  const uint16_t* q = reinterpret_cast<const uint16_t*>(a.q + row * a.ldq) + head * D;
  for (int d = lane; d < D; d += 64) qs[wave][d] = T::wide(q[d]);
  float m = -INFINITY, l = 0, o[D / 64] = {};
  const int lo = a.window == 0 ? 0 : max(p - a.window + 1, 0);
  const int mask = (1 << a.pool.page_shift) - 1;
  const int32_t* table = s.table + b * s.ld_table;
  for (int j0 = 0; j0 <= p; j0 += 64) {
    if (j0 + 63 < lo && j0 >= a.sinks) continue;
    const int j = j0 + lane;
    int page = -1;
    if (sees(p, j, a.window, a.sinks)) page = table[j >> a.pool.page_shift];
    const bool seen = page >= 0 && page < a.pool.pages;
    float x = -INFINITY;
    if (seen) {
      const char* k = a.pool.k + page * a.pool.k_page + h * a.pool.k_head + (j & mask) * a.pool.k_slot;
      float dot = 0;
      for (int d = 0; d < D; ++d) dot += qs[wave][d] * element<T, E4M3>(k, d);
      x = dot * c;
    }
    float top = x;
    for (int i = 32; i; i >>= 1) top = fmaxf(top, __shfl_xor(top, i));
    const float m2 = fmaxf(m, top);
    if (m2 == -INFINITY) continue;
    const float keep = __builtin_amdgcn_exp2f(m - m2), e = seen ? __builtin_amdgcn_exp2f(x - m2) : 0.0f;
    m = m2;
    float sum = e;
    for (int i = 32; i; i >>= 1) sum += __shfl_xor(sum, i);
    l = l * keep + sum;
    for (float& v : o) v *= keep;
    const uint64_t live = __ballot(seen);
    for (int i = 0; i < 64; ++i) {
      if (!(live >> i & 1)) continue;
      const float w = __shfl(e, i);
      const int pg = __shfl(page, i);
      const char* v = a.pool.v + pg * a.pool.v_page + h * a.pool.v_head + ((j0 + i) & mask) * a.pool.v_slot;
      for (int k = 0; k < D / 64; ++k) o[k] += w * element<T, E4M3>(v, 64 * k + lane);
    }
  }
  const float r = l == 0 ? 0.0f : (E4M3 && a.pool.vscale ? a.pool.vscale[h] : 1.0f) * __builtin_amdgcn_rcpf(l);
  char* y = a.y + row * a.ldy;
  for (int k = 0; k < D / 64; ++k) {
    const int e = head * D + 64 * k + lane;
    const float v = o[k] * r;
    if (a.out_f32) reinterpret_cast<float*>(y)[e] = v;
    else reinterpret_cast<uint16_t*>(y)[e] = static_cast<uint16_t>(T::pair(v, 0.0f));
  }
}

template <class T, bool E4M3>
hipError_t go(const PagedAttnArgs& a, hipStream_t s) {
  const dim3 grid(a.seqs.rows, ceil_div(a.heads, kWaves)), block(64 * kWaves);
  if (a.pool.hd == 64) hipLaunchKernelGGL((paged_rows_kernel<T, E4M3, 64>), grid, block, 0, s, a);
  else if (a.pool.hd == 128) hipLaunchKernelGGL((paged_rows_kernel<T, E4M3, 128>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((paged_rows_kernel<T, E4M3, 256>), grid, block, 0, s, a);
  return hipGetLastError();
}

}  // namespace

int64_t paged_workspace(int heads, int kv_heads, int hd, int, int seqs, int cap, bool decode) {
  return decode ? paged_decode_workspace(heads, kv_heads, hd, seqs, cap) : 0;
}

hipError_t launch_paged_attention(const PagedAttnArgs& a, hipStream_t s) {
  const bool e4m3 = a.pool.dtype == KV_E4M3;
  if (a.dtype == KV_BF16) return e4m3 ? go<Bf16, true>(a, s) : go<Bf16, false>(a, s);
  return e4m3 ? go<Fp16, true>(a, s) : go<Fp16, false>(a, s);
}

}  // namespace tars
