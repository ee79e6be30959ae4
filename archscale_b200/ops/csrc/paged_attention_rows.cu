// Attention of new tokens over a paged key-value cache (layout in paged.cuh), one CTA per query row: every type, head size and stride.
//
//   row (b, t, h):  o = Σ_j p_j v_j,  p = softmax over the visible j of scale · q·k_j,  visible: j ≤ pos, j ≥ pos − window, pos = lengths[b] − n + t
//   diff, row (b, t, pair):  a_i = Σ_j softmax_i(j) [v_1j | v_2j],  y = w · gain · (a_1 − λ a_2) / rms(a_1 − λ a_2)
//
// One pass over the keys with a running maximum and sum in 32 bits.  A warp takes every 16th key, its lanes every 32nd value of a row, so that loads
// are whole lines; the warps' parts meet in shared memory.  Keys and values are read once per query head: the cases that matter run
// paged_attention.cu, which reads them once for all heads and new tokens; this one takes what that one does not (fp32, head sizes and strides
// whose rows start off 4-byte boundaries, keys and values of different strides).
#include <cuda_fp8.h>

#include "paged.cuh"

namespace b200 {

constexpr int PR_WARPS = 16;
constexpr int PR_MAX = 8;                  // values of a row per lane: heads of up to 256

__device__ __forceinline__ float pr_value(const float* p) { return *p; }
__device__ __forceinline__ float pr_value(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float pr_value(const __nv_fp8_e4m3* p) { return static_cast<float>(*p); }
__device__ __forceinline__ void pr_put(float* p, float x) { *p = x; }
__device__ __forceinline__ void pr_put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ float pr_sum(float x) {
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// NB: softmax branches of a row, 2 for differential attention, whose values are the two heads side by side
template <class Cache, class Query, int NB>
__global__ void __launch_bounds__(PR_WARPS * 32) paged_rows_kernel(const PagedView c, const b200_paged_query a) {
  constexpr bool E8 = sizeof(Cache) == 1;
  __shared__ float s_top[NB][PR_WARPS], s_sum[NB][PR_WARPS], s_acc[NB][NB * PR_MAX * 32], s_red[PR_WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = c.dim;
  const int heads = a.H / NB;
  const int64_t row = blockIdx.x;
  const int h = static_cast<int>(row % heads), t = static_cast<int>(row / heads % a.T), b = static_cast<int>(row / heads / a.T);
  const int g = h / (a.H / c.groups) * NB;                             // (first) key head
  const int n = paged_new(c, b, a.T);
  int64_t first = 0, last = -1;                                        // visible keys
  if (t < n) {
    const int64_t pos = static_cast<int64_t>(c.lengths[b]) - n + t;
    last = min(pos, static_cast<int64_t>(c.table_cols) * c.page_size - 1);
    if (a.window >= 0) first = max(first, pos - a.window);
  }
  float q[NB][PR_MAX], acc[NB][NB][PR_MAX] = {}, top[NB], sum[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const Query* src = static_cast<const Query*>(a.q) + b * a.q_batch + t * a.q_token + (h * NB + i) * a.q_head;
#pragma unroll
    for (int e = 0; e < PR_MAX; ++e) q[i][e] = lane + 32 * e < D ? pr_value(src + lane + 32 * e) : 0.f;
    top[i] = -INFINITY; sum[i] = 0.f;
  }
  for (int64_t j = first + warp; j <= last; j += PR_WARPS) {
    const int page = paged_page(c, b, static_cast<int>(j) / c.page_size), slot = static_cast<int>(j) % c.page_size;
    if (page < 0) continue;
    float v[NB][PR_MAX];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const Cache* src = static_cast<const Cache*>(c.v) + page * c.v_page + (g + i) * c.v_group + slot * c.v_slot;
      const float s = E8 ? paged_pow2(c.vs[page * c.vs_page + (g + i) * c.vs_group + slot * c.vs_slot]) : 1.f;
#pragma unroll
      for (int e = 0; e < PR_MAX; ++e) v[i][e] = lane + 32 * e < D ? pr_value(src + lane + 32 * e) * s : 0.f;
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const Cache* src = static_cast<const Cache*>(c.k) + page * c.k_page + (g + i) * c.k_group + slot * c.k_slot;
      float x = 0.f;
#pragma unroll
      for (int e = 0; e < PR_MAX; ++e) if (lane + 32 * e < D) x = fmaf(q[i][e], pr_value(src + lane + 32 * e), x);
      x = pr_sum(x) * a.scale;
      if (E8) x *= paged_pow2(c.ks[page * c.ks_page + (g + i) * c.ks_group + slot * c.ks_slot]);
      if (x > top[i]) {
        const float f = top[i] == -INFINITY ? 0.f : expf(top[i] - x);
        sum[i] *= f;
#pragma unroll
        for (int m = 0; m < NB; ++m)
#pragma unroll
          for (int e = 0; e < PR_MAX; ++e) acc[i][m][e] *= f;
        top[i] = x;
      }
      const float p = x == -INFINITY ? 0.f : expf(x - top[i]);         // NaN stays NaN
      sum[i] += p;
#pragma unroll
      for (int m = 0; m < NB; ++m)
#pragma unroll
        for (int e = 0; e < PR_MAX; ++e) acc[i][m][e] = fmaf(p, v[m][e], acc[i][m][e]);
    }
  }
#pragma unroll
  for (int i = 0; i < NB; ++i) if (lane == 0) { s_top[i][warp] = top[i]; s_sum[i][warp] = sum[i]; }
  for (int i = threadIdx.x; i < NB * NB * PR_MAX * 32; i += blockDim.x) (&s_acc[0][0])[i] = 0.f;
  __syncthreads();
  float m_all[NB], l_all[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    m_all[i] = -INFINITY;
    for (int w = 0; w < PR_WARPS; ++w) m_all[i] = fmaxf(m_all[i], s_top[i][w]);
    l_all[i] = 0.f;
    for (int w = 0; w < PR_WARPS; ++w) l_all[i] += s_top[i][w] == -INFINITY ? s_sum[i][w] : s_sum[i][w] * expf(s_top[i][w] - m_all[i]);
  }
  for (int w = 0; w < PR_WARPS; ++w) {                                 // in a fixed order
    if (w == warp)
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const float f = top[i] == -INFINITY ? 1.f : expf(top[i] - m_all[i]);          // without a maximum the sums are 0, or NaN
#pragma unroll
        for (int m = 0; m < NB; ++m)
#pragma unroll
          for (int e = 0; e < PR_MAX; ++e) s_acc[i][(m * PR_MAX + e) * 32 + lane] += acc[i][m][e] * f;
      }
    __syncthreads();
  }
  // the row's softmax, its sink included, and its output; value i of the row is s_acc[.][i]
  float f[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    float m = m_all[i], l = l_all[i], keep = 1.f;
    if (NB == 1 && a.sink != nullptr && t < n) {
      const float s = paged_param(a.sink, a.sink_type, h), mm = fmaxf(m, s);
      keep = m == -INFINITY ? 0.f : expf(m - mm);
      l = (m == -INFINITY ? l : l * keep) + (s == -INFINITY ? 0.f : expf(s - mm));
      m = mm;
    }
    f[i] = l == 0.f ? 0.f : keep / l;                                  // a row that sees nothing is zero
    if (NB == 1 && a.lse != nullptr && threadIdx.x == 0) a.lse[(static_cast<int64_t>(b) * a.H + h) * a.T + t] = l == 0.f ? -INFINITY : m + logf(l);
  }
  const int i = threadIdx.x;                                           // NB · 256 ≤ the CTA's threads
  const int m = i / (PR_MAX * 32), d = i % (PR_MAX * 32);
  const bool mine = m < NB && d < D;
  Query* out = static_cast<Query*>(a.out) + (row * NB + m) * D + d;
  if constexpr (NB == 1) {
    if (mine) pr_put(out, s_acc[0][d] * f[0]);
  } else {
    const float y = mine ? s_acc[0][i] * f[0] - paged_param(a.lam, a.lam_type, 0) * (s_acc[1][i] * f[1]) : 0.f;
    const float part = pr_sum(y * y);
    if (lane == 0) s_red[warp] = part;
    __syncthreads();
    float total = 0.f;
    for (int w = 0; w < PR_WARPS; ++w) total += s_red[w];
    const float r = rsqrtf(total / (2 * D) + a.eps);
    if (mine) pr_put(out, t < n ? y * r * paged_param(a.w, a.w_type, m * D + d) * a.gain : 0.f);
  }
}

template <class Cache>
static int rows_as(const PagedView& c, const b200_paged_query& a, cudaStream_t st) {
  const int64_t rows = static_cast<int64_t>(a.B) * a.T * (a.H / (a.diff ? 2 : 1));
  if (rows > 0x7fffffffLL) return STATUS_BAD_ARG;
  const unsigned grid = static_cast<unsigned>(rows);
  if (a.type == 0) {
    if (a.diff) paged_rows_kernel<Cache, float, 2><<<grid, PR_WARPS * 32, 0, st>>>(c, a);
    else paged_rows_kernel<Cache, float, 1><<<grid, PR_WARPS * 32, 0, st>>>(c, a);
  } else {
    if (a.diff) paged_rows_kernel<Cache, __nv_bfloat16, 2><<<grid, PR_WARPS * 32, 0, st>>>(c, a);
    else paged_rows_kernel<Cache, __nv_bfloat16, 1><<<grid, PR_WARPS * 32, 0, st>>>(c, a);
  }
  return static_cast<int>(cudaGetLastError());
}

}  // namespace b200

extern "C" int b200_paged_attention_rows(const b200_paged_view* c, const b200_paged_query* a, cudaStream_t st) {
  using namespace b200;
  if (a->B <= 0 || a->T <= 0 || a->H <= 0) return 0;
  if (c->type == 0) return rows_as<float>(*c, *a, st);
  if (c->type == 1) return rows_as<__nv_bfloat16>(*c, *a, st);
  return rows_as<__nv_fp8_e4m3>(*c, *a, st);
}
