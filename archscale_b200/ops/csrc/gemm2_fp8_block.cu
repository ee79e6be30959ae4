// The product of gemm_fp8_block.cu on SM pairs (tcgen05.mma.cta_group::2): out[m, n] (+)= Σ_b sa[m, b] · sb[n, b] · (a block · b block) (+ bias[n]),
// one scale of A per row, of B per row or (BTILE) per 128 rows.
//
// Two CTAs share a 256 × NT tile; each stages its 128 rows of A and half of the rows of B.  A block of 128 along K is one accumulation
// of four MMAs into one of two accumulators in tensor memory (2 × NT columns), while eight warps read the other one and add it, scaled, to
// fp32 sums in registers: thread = row, NT / 2 columns.  Scales travel in a ring of their own, deeper than that of the operands, since
// they are needed up to two blocks after the operands' stage is free.
//
// 320 threads: warp 0 TMA, warp 1 MMA (leader CTA), warps 2..9 sums (two warps per lane quarter, one per half of the columns).
#include "api.h"
#include "sm100.cuh"

namespace b200 {

constexpr int F2_BK = 128, F2_THREADS = 320, F2_GROUP_M = 8, F2_SLOTS = 8;

template <int NT, bool BTILE>
struct F2 {
  static constexpr int A_BYTES = 128 * F2_BK, B_BYTES = NT / 2 * F2_BK, STAGE = A_BYTES + B_BYTES;
  static constexpr int SLOT = 512 + (BTILE ? 0 : NT * 4);                       // scales of A, then of B
  static constexpr int STAGES = NT == 256 ? 6 : 8;
  static constexpr int SMEM = STAGES * STAGE + F2_SLOTS * SLOT + 1024 + 512;
};

struct F2Params {
  void* out;
  const void* bias;
  const float* sb;                 // BTILE: scales of 128 rows of B
  int64_t sb_row, sb_blk, ldc;
  int M, N, K;
  int out_f32, accumulate, bias_f32;
  int* status;
};

__device__ __forceinline__ void f2_mma(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  if (elect_one_sync())
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(tmem_d), "l"(da), "l"(db), "r"(idesc), "r"(accumulate)
        : "memory");
}

template <int NT, bool BTILE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(F2_THREADS, 1)
gemm2_fp8_block_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                       const __grid_constant__ CUtensorMap tmap_sa, const __grid_constant__ CUtensorMap tmap_sb, const F2Params p) {
  using T = F2<NT, BTILE>;
  constexpr int W = NT / 2;                            // columns per thread
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* slots = smem + T::STAGES * T::STAGE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(slots + F2_SLOTS * T::SLOT);
  uint64_t* full_bar = bars;                           // [STAGES] used in the leader CTA
  uint64_t* empty_bar = full_bar + T::STAGES;          // [STAGES] each CTA's producer waits on its own
  uint64_t* sfull_bar = empty_bar + T::STAGES;         // [SLOTS]  scales, per CTA
  uint64_t* sempty_bar = sfull_bar + F2_SLOTS;         // [SLOTS]  eight warps
  uint64_t* tmem_full = sempty_bar + F2_SLOTS;         // [2]      each CTA's sums wait on their own
  uint64_t* tmem_empty = tmem_full + 2;                // [2]      used in the leader CTA, 16 warps
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(tmem_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_ptr + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int pair = static_cast<int>(blockIdx.x) >> 1, n_pair = static_cast<int>(gridDim.x) >> 1;
  const int num_m = (p.M + 255) / 256, num_n = (p.N + NT - 1) / NT;
  const int num_tiles = num_m * num_n;
  const int num_kb = (p.K + F2_BK - 1) / F2_BK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < T::STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    for (int s = 0; s < F2_SLOTS; ++s) { mbar_init(&sfull_bar[s], 1); mbar_init(&sempty_bar[s], 8); }
    for (int a = 0; a < 2; ++a) { mbar_init(&tmem_full[a], 1); mbar_init(&tmem_empty[a], 16); }
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmap_a); tma_prefetch_desc(&tmap_b); tma_prefetch_desc(&tmap_sa);
    if (!BTILE) tma_prefetch_desc(&tmap_sb);
  }
  if (warp == 1) { tmem_alloc_2sm(tmem_ptr, 2 * NT); tmem_relinquish_2sm(); }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();          // the peer's barriers are initialised before anything signals them
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_ptr, 0);

  auto tile_coords = [&](int t, int& m0, int& n0) {
    const int per_group = F2_GROUP_M * num_n;
    const int g = t / per_group, first_m = g * F2_GROUP_M;
    const int gsz = min(num_m - first_m, F2_GROUP_M);
    const int r = t - g * per_group;
    m0 = (first_m + (r % gsz)) * 256;
    n0 = (r / gsz) * NT;
  };

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0, slot = 0; uint32_t phase = 0, sphase = 0;
      for (int t = pair; t < num_tiles; t += n_pair) {
        int m0, n0; tile_coords(t, m0, n0);
        const int ma = m0 + rank * 128, nb = n0 + rank * (NT / 2);
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag, p.status, STATUS_TIMEOUT_EMPTY)) goto done;
          uint8_t* sa = smem + stage * T::STAGE;
          if (rank == 0) mbar_arrive_expect_tx(&full_bar[stage], 2 * T::STAGE);       // both CTAs' loads
          tma_load_2d_2sm(sa, &tmap_a, &full_bar[stage], kb * F2_BK, ma);
          tma_load_2d_2sm(sa + T::A_BYTES, &tmap_b, &full_bar[stage], kb * F2_BK, nb);
          if (!mbar_wait(&sempty_bar[slot], sphase ^ 1, abort_flag, p.status, STATUS_TIMEOUT_EMPTY)) goto done;
          mbar_arrive_expect_tx(&sfull_bar[slot], T::SLOT);
          tma_load_2d(slots + slot * T::SLOT, &tmap_sa, &sfull_bar[slot], ma, kb);
          if (!BTILE) tma_load_2d(slots + slot * T::SLOT + 512, &tmap_sb, &sfull_bar[slot], n0, kb);
          if (++stage == T::STAGES) { stage = 0; phase ^= 1; }
          if (++slot == F2_SLOTS) { slot = 0; sphase ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {                                   // the whole warp, converged: one lane is elected per instruction
      // e4m3 × e4m3, fp32 accumulate, both operands K-major
      constexpr uint32_t idesc = (1u << 4) | (static_cast<uint32_t>(NT >> 3) << 17) | (static_cast<uint32_t>(256 >> 4) << 24);
      int stage = 0; uint32_t phase = 0, it = 0;
      for (int t = pair; t < num_tiles; t += n_pair) {
        for (int kb = 0; kb < num_kb; ++kb, ++it) {
          const int acc = it & 1; const uint32_t acc_phase = (it >> 1) & 1;
          if (!mbar_wait_warp(&full_bar[stage], phase, abort_flag, p.status, STATUS_TIMEOUT_FULL)) goto done;
          if (!mbar_wait_warp(&tmem_empty[acc], acc_phase ^ 1, abort_flag, p.status, STATUS_TIMEOUT_TMEM_EMPTY)) goto done;
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * T::STAGE);
          const uint64_t da = make_smem_desc(sa, 16, 1024), db = make_smem_desc(sa + T::A_BYTES, 16, 1024);
#pragma unroll
          for (uint32_t k = 0; k < F2_BK / 32; ++k)
            f2_mma(tmem_base + acc * NT, da + static_cast<uint64_t>(k * 2), db + static_cast<uint64_t>(k * 2), idesc, k != 0 ? 1u : 0u);
          if (elect_one_sync()) { umma_commit_2sm(&empty_bar[stage], 3); umma_commit_2sm(&tmem_full[acc], 3); }
          if (++stage == T::STAGES) { stage = 0; phase ^= 1; }
        }
      }
    }
  } else {
    const int q = warp & 3, half = (warp - 2) >> 2;    // lane quarter, half of the columns
    const int esz = p.out_f32 ? 4 : 2;
    const bool wide = p.ldc * esz % 32 == 0 && reinterpret_cast<uintptr_t>(p.out) % 32 == 0;      // whole sectors per lane
    int slot = 0; uint32_t sphase = 0, it = 0;
    for (int t = pair; t < num_tiles; t += n_pair) {
      int m0, n0; tile_coords(t, m0, n0);
      const int row = m0 + rank * 128 + q * 32 + lane, c0 = n0 + half * W;
      const float* sb = BTILE ? p.sb + static_cast<int64_t>(min(c0, p.N - 1) >> 7) * p.sb_row : nullptr;
      float fb = BTILE ? sb[0] : 0.f;
      float2 sum[W / 2];
#pragma unroll
      for (int i = 0; i < W / 2; ++i) sum[i] = make_float2(0.f, 0.f);
      for (int kb = 0; kb < num_kb; ++kb, ++it) {
        const int acc = it & 1; const uint32_t acc_phase = (it >> 1) & 1;
        const uint32_t taddr = tmem_base + acc * NT + half * W + (static_cast<uint32_t>(q * 32) << 16);
        if (!mbar_wait_warp(&sfull_bar[slot], sphase, abort_flag, p.status, STATUS_TIMEOUT_FULL)) goto done;
        const float* ss = reinterpret_cast<const float*>(slots + slot * T::SLOT);
        float fa = ss[q * 32 + lane];
        const float2* sv = reinterpret_cast<const float2*>(ss + 128 + half * W);
        if (BTILE) {
          fa *= fb;
          if (kb + 1 < num_kb) fb = sb[(kb + 1) * p.sb_blk];
        }
        const float2 fa2 = make_float2(fa, fa);
        if (!mbar_wait_warp(&tmem_full[acc], acc_phase, abort_flag, p.status, STATUS_TIMEOUT_TMEM_FULL)) goto done;
        tc_fence_after();
        uint32_t r[2][16];
        tmem_ld_32x16(taddr, r[0]);
        tmem_ld_wait();
#pragma unroll
        for (int c = 0; c < W / 16; ++c) {
          if (c + 1 < W / 16) tmem_ld_32x16(taddr + (c + 1) * 16, r[(c + 1) & 1]);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float2 v = make_float2(__uint_as_float(r[c & 1][2 * i]), __uint_as_float(r[c & 1][2 * i + 1]));
            if (!BTILE) v = mul_f32x2(v, sv[c * 8 + i]);
            sum[c * 8 + i] = fma_f32x2(v, fa2, sum[c * 8 + i]);
          }
          if (c + 1 < W / 16) tmem_ld_wait();
          if (c + 2 == W / 16) {                       // the last columns are in registers: the accumulator is free
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_leader(&tmem_empty[acc]);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sempty_bar[slot]);
        if (++slot == F2_SLOTS) { slot = 0; sphase ^= 1; }
      }
      if (row < p.M) {
#pragma unroll
        for (int c = 0; c < W / 16; ++c) {
          const int col = c0 + c * 16;
          float v[16];
#pragma unroll
          for (int i = 0; i < 8; ++i) { v[2 * i] = sum[c * 8 + i].x; v[2 * i + 1] = sum[c * 8 + i].y; }
          if (p.bias) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (col + i < p.N)
                v[i] += p.bias_f32 ? static_cast<const float*>(p.bias)[col + i] : __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[col + i]);
          }
          const int64_t at = static_cast<int64_t>(row) * p.ldc + col;
          if (p.out_f32) {
            float* o = static_cast<float*>(p.out) + at;
            if (wide && col + 16 <= p.N) {
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                uint32_t w[8];
                if (p.accumulate) load_32b(o + 8 * j, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] = __float_as_uint(p.accumulate ? __uint_as_float(w[e]) + v[8 * j + e] : v[8 * j + e]);
                store_32b(o + 8 * j, w);
              }
            } else {
#pragma unroll
              for (int i = 0; i < 16; ++i)
                if (col + i < p.N) o[i] = p.accumulate ? o[i] + v[i] : v[i];
            }
          } else {
            __nv_bfloat16* o = static_cast<__nv_bfloat16*>(p.out) + at;
            if (wide && col + 16 <= p.N) {
              uint32_t w[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) w[e] = pack_bf16x2(v[2 * e], v[2 * e + 1]);
              store_32b(o, w);
            } else {
#pragma unroll
              for (int i = 0; i < 16; ++i)
                if (col + i < p.N) o[i] = __float2bfloat16(v[i]);
            }
          }
        }
      }
    }
  }

done:
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc_2sm(tmem_base, 2 * NT);
  }
}

int make_tmap_2d_u8(CUtensorMap* map, const void* ptr, uint64_t inner, uint64_t outer, uint64_t row_stride_bytes,
                    uint32_t box_inner, uint32_t box_outer);

// Scales [blocks][ld] of `rows` rows, boxes of `box` rows of one block (rows past the end read as zeros).
static int make_tmap_scales(CUtensorMap* map, const float* ptr, uint64_t rows, uint64_t blocks, uint64_t ld, uint32_t box) {
  typedef CUresult (*Encode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                             const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static Encode fn = nullptr;
  if (!fn) {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult res;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &res) != cudaSuccess || res != cudaDriverEntryPointSuccess) return -1;
    fn = reinterpret_cast<Encode>(f);
  }
  const cuuint64_t dim[2] = {rows, blocks}, stride[1] = {ld * 4};
  const cuuint32_t boxes[2] = {box, 1}, step[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, const_cast<float*>(ptr), dim, stride, boxes, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : static_cast<int>(r);
}

template <int NT, bool BTILE>
static int launch_f2(const void* A, int64_t lda, const float* sa, int64_t sa_blk, const void* B, int64_t ldb, const float* sb, const F2Params& p,
                     int num_sms, cudaStream_t st) {
  using T = F2<NT, BTILE>;
  CUtensorMap ta, tb, tsa, tsb;
  const uint64_t blocks = (p.K + F2_BK - 1) / F2_BK;
  int rc = make_tmap_2d_u8(&ta, A, p.K, p.M, lda, F2_BK, 128);
  if (!rc) rc = make_tmap_2d_u8(&tb, B, p.K, p.N, ldb, F2_BK, NT / 2);
  if (!rc) rc = make_tmap_scales(&tsa, sa, p.M, blocks, sa_blk, 128);
  tsb = tsa;
  if (!rc && !BTILE) rc = make_tmap_scales(&tsb, sb, p.N, blocks, p.sb_blk, NT);
  if (rc) return rc;
  auto kern = gemm2_fp8_block_kernel<NT, BTILE>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, T::SMEM) != cudaSuccess) return -2;
  const int64_t tiles = static_cast<int64_t>((p.M + 255) / 256) * ((p.N + NT - 1) / NT);
  if (tiles > 0x3fffffff) return -6;
  const int pairs = num_sms / 2;
  kern<<<2 * (tiles < pairs ? static_cast<int>(tiles) : pairs), F2_THREADS, T::SMEM, st>>>(ta, tb, tsa, tsb, p);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

}  // namespace b200

// Contract of b200_gemm_fp8_block, which checks the arguments and calls this: scales of A are per row, stored [block][sa_blk], those
// of B too unless sb_tile; addresses of such scales and their strides are multiples of 16 bytes.
extern "C" int b200_gemm2_fp8_block(const void* A, int64_t lda, const float* sa, int64_t sa_blk, const void* B, int64_t ldb, const float* sb,
                                    int64_t sb_row, int64_t sb_blk, int sb_tile, const void* bias, int bias_f32, void* out, int64_t ldc, int M,
                                    int N, int K, int out_f32, int accumulate, int nt, int num_sms, int* status, cudaStream_t stream) {
  using namespace b200;
  const F2Params p{out, bias, sb, sb_row, sb_blk, ldc, M, N, K, out_f32, accumulate, bias_f32, status};
  if (nt == 256)
    return sb_tile ? launch_f2<256, true>(A, lda, sa, sa_blk, B, ldb, sb, p, num_sms, stream)
                   : launch_f2<256, false>(A, lda, sa, sa_blk, B, ldb, sb, p, num_sms, stream);
  return sb_tile ? launch_f2<128, true>(A, lda, sa, sa_blk, B, ldb, sb, p, num_sms, stream)
                 : launch_f2<128, false>(A, lda, sa, sa_blk, B, ldb, sb, p, num_sms, stream);
}
