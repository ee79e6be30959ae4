// Product of e4m3 operands with one fp32 scale per block of 128 along K:
//
//   out[m, n] (+)= Σ_b  sa[m, b] · sb[n, b] · Σ_{k in block b} a[m, k] · b[n, k]   (+ bias[n])
//
// A scale belongs to one row (activations, gradients) or to 128 rows (weights); both operands are K-major.  The tensor cores take no
// fp32 scales, so the products of one block of K are accumulated in tensor memory (exact to fp32 rounding over 128 terms), read
// back, scaled and added to fp32 sums in registers.
//
// 128 × 128 tile per CTA, six stages of 32 KB; two accumulators in tensor memory, so that the products of a block run while the
// one before is read.  192 threads: warp 0 TMA, warp 1 MMA, warps 2..5 sums (thread = row of the tile, 128 sums each).
#include "api.h"
#include "sm100.cuh"

namespace b200 {

constexpr int FB_BM = 128, FB_BN = 128, FB_BK = 128, FB_STAGES = 6, FB_THREADS = 192;
constexpr int FB_A = FB_BM * FB_BK, FB_B = FB_BN * FB_BK, FB_STAGE = FB_A + FB_B;
constexpr int FB_SMEM = FB_STAGES * FB_STAGE + 1024 + 256;

struct Fp8Scale {
  const float* p;
  int64_t row, blk;       // strides between rows (or groups of 128 rows) and between blocks of K
  int shift;              // 0: one scale per row, 7: per 128 rows
};

struct Fp8GemmParams {
  void* out;
  const void* bias;
  Fp8Scale sa, sb;
  int M, N, K;
  int64_t ldc;
  int out_f32, accumulate, bias_f32;
  int* status;
};

__device__ __forceinline__ void umma_fp8_warp(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  if (elect_one_sync())
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(tmem_d), "l"(da), "l"(db), "r"(idesc), "r"(accumulate)
        : "memory");
}
// e4m3 × e4m3 (format code 0 in both operand fields), fp32 accumulate, both operands K-major
__host__ __device__ constexpr uint32_t make_idesc_e4m3(int M, int N) {
  return (1u << 4) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

__global__ void __launch_bounds__(FB_THREADS, 1)
gemm_fp8_block_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const Fp8GemmParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + FB_STAGES * FB_STAGE);
  uint64_t* full_bar = bars;
  uint64_t* empty_bar = bars + FB_STAGES;
  uint64_t* tmem_full = bars + 2 * FB_STAGES;          // [2]
  uint64_t* tmem_empty = bars + 2 * FB_STAGES + 2;     // [2], four warps
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(bars + 2 * FB_STAGES + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_ptr + 1);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int num_m = (p.M + FB_BM - 1) / FB_BM;
  const int m0 = static_cast<int>(blockIdx.x) % num_m * FB_BM, n0 = static_cast<int>(blockIdx.x) / num_m * FB_BN;
  const int num_kb = (p.K + FB_BK - 1) / FB_BK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < FB_STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(&tmem_full[a], 1); mbar_init(&tmem_empty[a], 4); }
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmap_a);
    tma_prefetch_desc(&tmap_b);
  }
  if (warp == 1) { tmem_alloc(tmem_ptr, 256); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_ptr, 0);

  if (warp == 0) {
    if (lane == 0) {
      for (int kb = 0; kb < num_kb; ++kb) {
        const int st = kb % FB_STAGES; const uint32_t ph = (kb / FB_STAGES) & 1;
        if (!mbar_wait(&empty_bar[st], ph ^ 1, abort_flag, p.status, STATUS_TIMEOUT_EMPTY)) break;
        uint8_t* sa = smem + st * FB_STAGE;
        mbar_arrive_expect_tx(&full_bar[st], FB_STAGE);
        tma_load_2d(sa, &tmap_a, &full_bar[st], kb * FB_BK, m0);
        tma_load_2d(sa + FB_A, &tmap_b, &full_bar[st], kb * FB_BK, n0);
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = make_idesc_e4m3(FB_BM, FB_BN);
    for (int kb = 0; kb < num_kb; ++kb) {
      const int st = kb % FB_STAGES; const uint32_t ph = (kb / FB_STAGES) & 1;
      const int acc = kb & 1; const uint32_t aph = (kb >> 1) & 1;
      if (!mbar_wait_warp(&tmem_empty[acc], aph ^ 1, abort_flag, p.status, STATUS_TIMEOUT_TMEM_EMPTY)) break;
      if (!mbar_wait_warp(&full_bar[st], ph, abort_flag, p.status, STATUS_TIMEOUT_FULL)) break;
      tc_fence_after();
      const uint32_t sa = smem_u32(smem + st * FB_STAGE);
      const uint64_t da = make_smem_desc(sa, 16, 1024), db = make_smem_desc(sa + FB_A, 16, 1024);
#pragma unroll
      for (uint32_t k = 0; k < FB_BK / 32; ++k)
        umma_fp8_warp(tmem_base + acc * FB_BN, da + static_cast<uint64_t>(2 * k), db + static_cast<uint64_t>(2 * k), idesc, k != 0 ? 1u : 0u);
      umma_commit_warp(&empty_bar[st]);
      umma_commit_warp(&tmem_full[acc]);
    }
  } else {
    const int q = warp & 3;
    const int row = m0 + q * 32 + lane;
    const bool live = row < p.M;
    const float* sa = p.sa.p + static_cast<int64_t>(live ? row >> p.sa.shift : 0) * p.sa.row;
    float sum[FB_BN];
#pragma unroll
    for (int i = 0; i < FB_BN; ++i) sum[i] = 0.f;
    bool ok = true;
    for (int kb = 0; kb < num_kb; ++kb) {
      const int acc = kb & 1; const uint32_t aph = (kb >> 1) & 1;
      const float fa = live ? sa[kb * p.sa.blk] : 0.f;
      const float* sb = p.sb.p + kb * p.sb.blk;
      ok = mbar_wait(&tmem_full[acc], aph, abort_flag, p.status, STATUS_TIMEOUT_TMEM_FULL);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < FB_BN / 32; ++c) {
        uint32_t r[32];
        tmem_ld_32x32(tmem_base + acc * FB_BN + c * 32 + (static_cast<uint32_t>(q * 32) << 16), r);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const int col = n0 + c * 32 + i;
          const float fb = col < p.N ? sb[static_cast<int64_t>(col >> p.sb.shift) * p.sb.row] : 0.f;
          sum[c * 32 + i] += __uint_as_float(r[i]) * (fa * fb);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tmem_empty[acc]);
    }
    if (ok && live) {
#pragma unroll
      for (int i = 0; i < FB_BN; ++i) {
        const int col = n0 + i;
        if (col < p.N) {
          float v = sum[i];
          if (p.bias) v += p.bias_f32 ? static_cast<const float*>(p.bias)[col] : __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[col]);
          const int64_t at = static_cast<int64_t>(row) * p.ldc + col;
          if (p.out_f32) {
            float* o = static_cast<float*>(p.out) + at;
            *o = p.accumulate ? *o + v : v;
          } else {
            static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16(v);
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 256);
  }
}

int make_tmap_2d_u8(CUtensorMap* map, const void* ptr, uint64_t inner, uint64_t outer, uint64_t row_stride_bytes,
                    uint32_t box_inner, uint32_t box_outer);

}  // namespace b200

// A [M, K], B [N, K]: e4m3, rows lda / ldb bytes apart (multiples of 16, as the addresses).  sa, sb: scales with strides between rows
// (or groups of 128 rows: *_tile) and between blocks of 128 along K.  out [M, N] fp32 (accumulate: added to) or bf16; bias [N] or null.
extern "C" int b200_gemm_fp8_block(const void* A, int64_t lda, const float* sa, int64_t sa_row, int64_t sa_blk, int sa_tile, const void* B,
                                   int64_t ldb, const float* sb, int64_t sb_row, int64_t sb_blk, int sb_tile, const void* bias, int bias_dtype,
                                   void* out, int64_t ldc, int M, int N, int K, int out_f32, int accumulate, int pair, int num_sms, int* status,
                                   cudaStream_t stream) {
  using namespace b200;
  if (M < 0 || N < 0 || K < 1 || lda % 16 || ldb % 16 || (accumulate && !out_f32)) return -6;
  if (M == 0 || N == 0) return 0;
  if (pair) {
    const auto rows = [](const float* s, int64_t row, int64_t blk) { return row == 1 && blk % 4 == 0 && reinterpret_cast<uintptr_t>(s) % 16 == 0; };
    if (sa_tile || !rows(sa, sa_row, sa_blk) || (!sb_tile && !rows(sb, sb_row, sb_blk))) return -6;
    const int64_t m = (M + 255) / 256, pairs = num_sms / 2;
    // tiles of half the width take 0.55 of the time (a little more than half): narrower where that saves enough of the last wave
    const int64_t wide = (m * ((N + 255) / 256) + pairs - 1) / pairs * 100, narrow = (m * ((N + 127) / 128) + pairs - 1) / pairs * 55;
    return b200_gemm2_fp8_block(A, lda, sa, sa_blk, B, ldb, sb, sb_row, sb_blk, sb_tile, bias, bias_dtype == 0 ? 1 : 0, out, ldc, M, N, K, out_f32,
                                accumulate, narrow < wide ? 128 : 256, num_sms, status, stream);
  }
  CUtensorMap ta, tb;
  int rc = make_tmap_2d_u8(&ta, A, K, M, lda, FB_BK, FB_BM);
  if (rc) return rc;
  rc = make_tmap_2d_u8(&tb, B, K, N, ldb, FB_BK, FB_BN);
  if (rc) return rc;
  const Fp8GemmParams p{out, bias, {sa, sa_row, sa_blk, sa_tile ? 7 : 0}, {sb, sb_row, sb_blk, sb_tile ? 7 : 0}, M, N, K, ldc,
                        out_f32, accumulate, bias_dtype == 0 ? 1 : 0, status};
  if (cudaFuncSetAttribute(gemm_fp8_block_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, FB_SMEM) != cudaSuccess) return -2;
  const int64_t tiles = static_cast<int64_t>((M + FB_BM - 1) / FB_BM) * ((N + FB_BN - 1) / FB_BN);
  if (tiles > 0x7fffffff) return -6;
  gemm_fp8_block_kernel<<<static_cast<unsigned>(tiles), FB_THREADS, FB_SMEM, stream>>>(ta, tb, p);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}
