// Product of e4m3 operands with one fp32 scale per block of 128 along K:
//
//   out[m, n] (+)= Σ_b  sa[m, b] · sb[n, b] · Σ_{k in block b} a[m, k] · b[n, k]   (+ bias[n])
//
// A scale belongs to one row (activations, gradients) or to 128 rows (weights); both operands are K-major.  The tensor cores take no
// fp32 scales, so the products of one block of K are accumulated in tensor memory (exact to fp32 rounding over 128 terms), read
// back, scaled and added to fp32 sums in registers.
//
// This file: the form for few rows of A (single tokens, a batch in decoding, small results of a long K).  It is bound by reading B once (one token:
// 11264 × 2048 weights, 23 MB, 3.5 µs at the copy rate) and, at this size, by the latency of one CTA's chain (7.2 µs).  So 128 rows of B are the M side of the MMA and BT rows of A (16, 32 or 64) its N side, which
// makes neighbouring lanes neighbouring columns of the output, and the blocks of K are split over a cluster of up to eight CTAs.  The
// first loads are issued before tensor memory is allocated.  The CTAs' sums meet in shared memory, in the place of the stages; every CTA
// adds its share of the rows over the ranks in rank order (distributed shared memory), so a result does not depend on scheduling.
//
// Warp 0 TMA, warp 1 MMA, then four warps of sums for every 32 rows of A (thread = row of B, up to 32 sums); all of them add.
#include "api.h"
#include "sm100.cuh"

namespace b200 {

constexpr int FS_BN = 128, FS_BK = 128, FS_CHUNK = 32;

template <int BT>
struct FS {
  static constexpr int B_BYTES = FS_BN * FS_BK, A_BYTES = BT * FS_BK, STAGE = B_BYTES + A_BYTES;
  static constexpr int STAGES = BT == 16 ? 6 : BT == 32 ? 5 : 4;        // two CTAs fit an SM
  static constexpr int ACC = BT <= 32 ? 8 : 4;                     // accumulators: products run ahead of the sums
  static constexpr int TMEM = ACC * BT;
  static constexpr int W = BT < 32 ? BT : 32, GROUPS = BT / W;     // sums of a thread; teams of four warps
  static constexpr int SUMMERS = 128 * GROUPS, THREADS = 64 + SUMMERS;
  static constexpr int SMEM = STAGES * STAGE + FS_CHUNK * BT * 4 + 1024 + 256;
  static_assert(BT * FS_BN * 4 <= STAGES * STAGE, "the sums take the place of the stages");
};

struct Fp8Scale {
  const float* p;
  int64_t row, blk;       // strides between rows (or groups of 128 rows) and between blocks of K
  int shift;              // 0: one scale per row, 7: per 128 rows
};

struct FsParams {
  void* out;
  const void* bias;
  Fp8Scale sa, sb;
  int M, N, K;
  int64_t ldc;
  int out_f32, accumulate, bias_f32, vec;
  int* status;
};

__device__ __forceinline__ void fs_mma(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(tmem_d), "l"(da), "l"(db), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ float4 fs_ld_cluster(uint32_t smem_addr, int rank) {
  uint32_t a;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
  return v;
}

template <int BT, int S>
__global__ void __launch_bounds__(FS<BT>::THREADS, 2)
gemm_fp8_block_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const FsParams p) {
  using T = FS<BT>;
  constexpr int W = T::W;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* part = reinterpret_cast<float*>(smem);        // [BT][128] sums of this CTA, once the stages are read
  float* table = reinterpret_cast<float*>(smem + T::STAGES * T::STAGE);      // [FS_CHUNK][BT] scales of A
  uint64_t* bars = reinterpret_cast<uint64_t*>(table + FS_CHUNK * BT);
  uint64_t* full_bar = bars;
  uint64_t* empty_bar = bars + T::STAGES;
  uint64_t* tmem_full = bars + 2 * T::STAGES;          // [ACC]
  uint64_t* tmem_empty = tmem_full + T::ACC;           // [ACC], the warps of sums
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(tmem_empty + T::ACC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_ptr + 1);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = S > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int num_n = (p.N + FS_BN - 1) / FS_BN;
  const int tile = static_cast<int>(blockIdx.x) / S, n0 = tile % num_n * FS_BN, m0 = tile / num_n * BT;
  const int num_kb = (p.K + FS_BK - 1) / FS_BK, per = (num_kb + S - 1) / S;
  const int kb0 = min(rank * per, num_kb), nkb = min(kb0 + per, num_kb) - kb0;      // the last ranks may have no share

  auto load = [&](int i, int st) {
    uint8_t* sb = smem + st * T::STAGE;
    mbar_arrive_expect_tx(&full_bar[st], T::STAGE);
    tma_load_2d(sb, &tmap_b, &full_bar[st], (kb0 + i) * FS_BK, n0);
    tma_load_2d(sb + T::B_BYTES, &tmap_a, &full_bar[st], (kb0 + i) * FS_BK, m0);
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < T::STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    for (int a = 0; a < T::ACC; ++a) { mbar_init(&tmem_full[a], 1); mbar_init(&tmem_empty[a], 4 * T::GROUPS); }
    *abort_flag = 0;
    mbar_fence_init();
    fence_proxy_async_smem();
    for (int i = 0; i < T::STAGES && i < nkb; ++i) load(i, i);      // the ring is empty: no wait, and under the set-up
  }
  if (warp == 1) { tmem_alloc(tmem_ptr, T::TMEM); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_ptr, 0);
  uint32_t issued = 0;                                 // blocks that this warp has loaded (warp 0) or multiplied (warp 1)

  if (warp == 0) {
    issued = min(T::STAGES, nkb);
    for (int i = T::STAGES; i < nkb; ++i) {
      const int st = i % T::STAGES; const uint32_t ph = (i / T::STAGES) & 1;
      if (!mbar_wait_warp(&empty_bar[st], ph ^ 1, abort_flag, p.status, STATUS_TIMEOUT_EMPTY)) break;
      if (elect_one_sync()) load(i, st);
      ++issued;
    }
  } else if (warp == 1) {
    // e4m3 × e4m3, fp32 accumulate, both operands K-major
    constexpr uint32_t idesc = (1u << 4) | (static_cast<uint32_t>(BT >> 3) << 17) | (static_cast<uint32_t>(FS_BN >> 4) << 24);
    for (int i = 0; i < nkb; ++i) {
      const int st = i % T::STAGES; const uint32_t ph = (i / T::STAGES) & 1;
      const int acc = i % T::ACC; const uint32_t aph = (i / T::ACC) & 1;
      if (!mbar_wait_warp(&full_bar[st], ph, abort_flag, p.status, STATUS_TIMEOUT_FULL)) break;
      if (!mbar_wait_warp(&tmem_empty[acc], aph ^ 1, abort_flag, p.status, STATUS_TIMEOUT_TMEM_EMPTY)) break;
      tc_fence_after();
      const uint32_t sb = smem_u32(smem + st * T::STAGE);
      const uint64_t db = make_smem_desc(sb, 16, 1024), da = make_smem_desc(sb + T::B_BYTES, 16, 1024);
      if (elect_one_sync()) {
#pragma unroll
        for (uint32_t k = 0; k < FS_BK / 32; ++k)
          fs_mma(tmem_base + acc * BT, db + static_cast<uint64_t>(2 * k), da + static_cast<uint64_t>(2 * k), idesc, k != 0 ? 1u : 0u);
        umma_commit(&tmem_full[acc]);
        umma_commit(&empty_bar[st]);
      }
      ++issued;
    }
  } else {
    const int q = warp & 3, t = threadIdx.x - 64, c0 = (warp - 2) / 4 * W;      // lane quarter, first row of A
    const int n = n0 + q * 32 + lane;
    const float* sb = p.sb.p + static_cast<int64_t>(min(n, p.N - 1) >> p.sb.shift) * p.sb.row + kb0 * p.sb.blk;
    float sum[W], scale[8];
#pragma unroll
    for (int i = 0; i < W; ++i) sum[i] = 0.f;
    // A warp whose wait has run out goes on to the barriers of the table, which the others may still reach: every warp arrives at every one
    // of them, and the others' waits end within their limit too.
    bool ok = true;
    for (int i = 0; i < nkb; ++i) {
      const int acc = i % T::ACC; const uint32_t aph = (i / T::ACC) & 1;
      if ((i & 7) == 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) scale[j] = sb[min(i + j, nkb - 1) * p.sb.blk];
      }
      if (i % FS_CHUNK == 0) {                         // scales of A of the next blocks: the same for all rows of B
        if (i) asm volatile("bar.sync 1, %0;" ::"n"(T::SUMMERS) : "memory");
        const int blocks = min(FS_CHUNK, nkb - i);
        for (int j = t; j < blocks * BT; j += T::SUMMERS) {
          const int m = m0 + j % BT;
          table[j] = m < p.M ? p.sa.p[static_cast<int64_t>(m >> p.sa.shift) * p.sa.row + (kb0 + i + j / BT) * p.sa.blk] * kFp8Down : 0.f;
        }
        asm volatile("bar.sync 1, %0;" ::"n"(T::SUMMERS) : "memory");
      }
      const float s01 = (i & 1) ? scale[1] : scale[0], s23 = (i & 1) ? scale[3] : scale[2];
      const float s45 = (i & 1) ? scale[5] : scale[4], s67 = (i & 1) ? scale[7] : scale[6];
      const float f = (i & 4) ? ((i & 2) ? s67 : s45) : ((i & 2) ? s23 : s01);
      const float4* sa = reinterpret_cast<const float4*>(table + i % FS_CHUNK * BT + c0);
      ok = ok && mbar_wait_warp(&tmem_full[acc], aph, abort_flag, p.status, STATUS_TIMEOUT_TMEM_FULL);
      if (!ok) continue;
      tc_fence_after();
      uint32_t r[W];
      const uint32_t taddr = tmem_base + acc * BT + c0 + (static_cast<uint32_t>(q * 32) << 16);
      if constexpr (W == 32) tmem_ld_32x32(taddr, r);
      else tmem_ld_32x16(taddr, r);
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tmem_empty[acc]);
#pragma unroll
      for (int j = 0; j < W; j += 4) {
        const float4 a = sa[j / 4];
        sum[j] = fmaf(__uint_as_float(r[j]) * a.x, f, sum[j]);
        sum[j + 1] = fmaf(__uint_as_float(r[j + 1]) * a.y, f, sum[j + 1]);
        sum[j + 2] = fmaf(__uint_as_float(r[j + 2]) * a.z, f, sum[j + 2]);
        sum[j + 3] = fmaf(__uint_as_float(r[j + 3]) * a.w, f, sum[j + 3]);
      }
    }
    // the last products were waited for, so the loads before them have landed and the stages may be written
    if (ok) {
#pragma unroll
      for (int i = 0; i < W; ++i) part[(c0 + i) * FS_BN + q * 32 + lane] = sum[i] * kFp8Up;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp < 2 && *abort_flag) drain_ring(warp == 0 ? full_bar : empty_bar, T::STAGES, issued);
  __syncwarp();
  if (S > 1) cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, T::TMEM);
  }
  // rows of the output: every CTA of the cluster adds its share over the ranks
  const int rows = min(p.M - m0, BT), first = rank * BT / S, last = min((rank + 1) * BT / S, rows);
  const int col = n0 + lane * 4;
  const uint32_t part_addr = smem_u32(part);
  for (int m = first + warp; m < last; m += T::THREADS / 32) {
    float4 v[S];
#pragma unroll
    for (int r = 0; r < S; ++r) {
      if (S > 1) v[r] = fs_ld_cluster(part_addr + (m * FS_BN + lane * 4) * 4, r);
      else v[r] = *reinterpret_cast<const float4*>(part + m * FS_BN + lane * 4);
    }
#pragma unroll
    for (int r = 1; r < S; ++r) { v[0].x += v[r].x; v[0].y += v[r].y; v[0].z += v[r].z; v[0].w += v[r].w; }
    float o[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
    if (p.bias) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col + e < p.N) o[e] += p.bias_f32 ? static_cast<const float*>(p.bias)[col + e] : __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[col + e]);
    }
    const int64_t at = static_cast<int64_t>(m0 + m) * p.ldc + col;
    if (p.out_f32) {
      float* d = static_cast<float*>(p.out) + at;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col + e < p.N) d[e] = p.accumulate ? d[e] + o[e] : o[e];
    } else {
      __nv_bfloat16* d = static_cast<__nv_bfloat16*>(p.out) + at;
      if (p.vec && col + 4 <= p.N) {
        *reinterpret_cast<uint2*>(d) = make_uint2(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < p.N) d[e] = __float2bfloat16(o[e]);
      }
    }
  }
  if (S > 1) cluster_sync_all();                       // nobody leaves while its sums are read
}

int make_tmap_2d_u8(CUtensorMap* map, const void* ptr, uint64_t inner, uint64_t outer, uint64_t row_stride_bytes,
                    uint32_t box_inner, uint32_t box_outer);

// K is split as far as the CTAs fit the machine at once and have a block each.
static int fs_split(int64_t tiles, int K, int num_sms) {
  const int num_kb = (K + FS_BK - 1) / FS_BK;
  int s = 1;
  while (s < 8 && tiles * 2 * s <= 2 * static_cast<int64_t>(num_sms) && 2 * s <= num_kb) s *= 2;
  return s;
}
double f2_microseconds(int M, int N, int K, int sb_tile, int num_sms);

template <int BT, int S>
static int launch_fs(const CUtensorMap& ta, const CUtensorMap& tb, const FsParams& p, unsigned tiles, cudaStream_t st) {
  auto kern = gemm_fp8_block_kernel<BT, S>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, FS<BT>::SMEM) != cudaSuccess) return -2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(tiles * S);
  cfg.blockDim = dim3(FS<BT>::THREADS);
  cfg.dynamicSmemBytes = FS<BT>::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = S; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = S > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, ta, tb, p) == cudaSuccess ? 0 : -3;
}
template <int BT>
static int launch_fs(const void* A, int64_t lda, const void* B, int64_t ldb, const FsParams& p, int num_sms, cudaStream_t st) {
  CUtensorMap ta, tb;
  int rc = make_tmap_2d_u8(&ta, A, p.K, p.M, lda, FS_BK, BT);
  if (!rc) rc = make_tmap_2d_u8(&tb, B, p.K, p.N, ldb, FS_BK, FS_BN);
  if (rc) return rc;
  const int64_t tiles = static_cast<int64_t>((p.M + BT - 1) / BT) * ((p.N + FS_BN - 1) / FS_BN);
  if (tiles > 0xfffffff) return -6;
  const int s = fs_split(tiles, p.K, num_sms);
  const unsigned t = static_cast<unsigned>(tiles);
  return s == 8 ? launch_fs<BT, 8>(ta, tb, p, t, st) : s == 4 ? launch_fs<BT, 4>(ta, tb, p, t, st)
       : s == 2 ? launch_fs<BT, 2>(ta, tb, p, t, st) : launch_fs<BT, 1>(ta, tb, p, t, st);
}

}  // namespace b200

// Whether a product with one scale per row of A runs on SM pairs.  Up to 64 rows never do.  From there this file's kernel has a fixed time (one more
// microsecond where two CTAs share an SM) and reads 24 KB per tile of 64 x 128 and block of K at 8 TB/s; it wins while its tiles are few: µs of
// it and of the pairs, weight tiles / scales per row, 2048 x 5632 weights 128 rows 11.8 and 18.2 / 11.8 and 28.2, 256 14.3 and 18.7 / 14.4 and 27.3,
// 384 21.5 and 19.1 / 21.6 and 28.3; 11264 x 2048 128 rows 15.9 and 13.2 / 15.9 and 16.5, 512 38 and 22 / 39 and 29.  Over 90 random sizes (65 to 2500 rows)
// what it picks takes 1.010 of the better one's time, the pairs alone 1.25.
extern "C" int b200_gemm_fp8_block_pairs(int M, int N, int K, int sb_tile, int num_sms) {
  using namespace b200;
  if (M <= 64) return 0;
  const int64_t tiles = static_cast<int64_t>((M + 63) / 64) * ((N + FS_BN - 1) / FS_BN);
  const double few = 6.0 + (tiles * fs_split(tiles, K, num_sms) > num_sms ? 1.0 : 0.0) + 0.0031 * static_cast<double>(tiles) * ((K + FS_BK - 1) / FS_BK);
  return few < f2_microseconds(M, N, K, sb_tile, num_sms) ? 0 : 1;
}

// A [M, K], B [N, K]: e4m3, rows lda / ldb bytes apart (multiples of 16, as the addresses).  sa, sb: scales with strides between rows
// (or groups of 128 rows: *_tile) and between blocks of 128 along K.  out [M, N] fp32 (accumulate: added to) or bf16; bias [N] or null.
// pair: on SM pairs, with the workspace that b200_gemm2_fp8_block_workspace names.
extern "C" int b200_gemm_fp8_block(const void* A, int64_t lda, const float* sa, int64_t sa_row, int64_t sa_blk, int sa_tile, const void* B,
                                   int64_t ldb, const float* sb, int64_t sb_row, int64_t sb_blk, int sb_tile, const void* bias, int bias_dtype,
                                   void* out, int64_t ldc, int M, int N, int K, int out_f32, int accumulate, int pair, void* ws, int num_sms,
                                   int* status, cudaStream_t stream) {
  using namespace b200;
  if (M < 0 || N < 0 || K < 1 || lda % 16 || ldb % 16 || (accumulate && !out_f32)) return -6;
  if (M == 0 || N == 0) return 0;
  static thread_local bool ctx_bound = false;          // tensor maps are encoded by the driver, which wants a context on this thread
  if (!ctx_bound) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess) return -5;
    ctx_bound = true;
  }
  if (pair) {
    const auto rows = [](const float* s, int64_t row, int64_t blk) { return row == 1 && blk % 4 == 0 && reinterpret_cast<uintptr_t>(s) % 16 == 0; };
    if (sa_tile || sa_row != 1 || (!sb_tile && !rows(sb, sb_row, sb_blk))) return -6;
    return b200_gemm2_fp8_block(A, lda, sa, sa_blk, B, ldb, sb, sb_row, sb_blk, sb_tile, bias, bias_dtype == 0 ? 1 : 0, out, ldc, M, N, K, out_f32,
                                accumulate, ws, num_sms, status, stream);
  }
  const FsParams p{out, bias, {sa, sa_row, sa_blk, sa_tile ? 7 : 0}, {sb, sb_row, sb_blk, sb_tile ? 7 : 0}, M, N, K, ldc, out_f32, accumulate,
                   bias_dtype == 0 ? 1 : 0, ldc % 4 == 0 && reinterpret_cast<uintptr_t>(out) % 8 == 0 ? 1 : 0, status};
  if (M <= 16) return launch_fs<16>(A, lda, B, ldb, p, num_sms, stream);
  if (M <= 32) return launch_fs<32>(A, lda, B, ldb, p, num_sms, stream);
  return launch_fs<64>(A, lda, B, ldb, p, num_sms, stream);
}
