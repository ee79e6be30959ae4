// The product of gemm_fp8_block.cu on SM pairs (tcgen05.mma.cta_group::2): out[m, n] (+)= Σ_b sa[m, b] · sb[n, b] · (a block · b block) (+ bias[n]),
// one scale of A per row, of B per row or (BTILE) per 128 rows.
//
// Two CTAs share a 256 × NT tile; each stages its 128 rows of A and half of the rows of B.  A block of 128 along K is one accumulation
// of four MMAs into one of two accumulators in tensor memory (2 × NT columns), while eight warps read the other one and add it, scaled, to
// fp32 sums in registers: thread = row, NT / 2 columns.
//
// What bounds it is that read-out: per block a warp has to see the products done, bring 128 columns to registers and spend 128
// multiply-adds on them (two warps share a scheduler: 256 cycles of the 512 that the products take), and everything that stands beside these
// in its one chain of instructions adds to the block's time.  Hence: the row's scales of eight blocks are loaded together (the wait for them is
// paid once in eight; fetched block by block through a TMA ring, as the operands are, they cost 150 cycles a block), scales of 128 rows of B
// are folded into them there.  Scales per row of B make two operations of every multiply-add and go through shared memory (copied
// asynchronously, each warp its own rows and columns); there a warp reads its accumulator in the shape that gives a thread 4 rows × 32 columns
// instead of one row × 128: with a row per thread, 32 broadcast reads of 16 bytes per block and warp kept the shared memory's port busy for
// twice the time of the products.  (Of the forms that keep a large scale against a small one in range, this one, 11264 × 2048 × 32768 971 µs against 970
// without, was the fastest; the product of the two scales first: 1009.)
// Loads, products and their commits are issued by one elected lane of a converged warp: four loads a block from a branch of one lane
// took longer than the block's products.  Two half-width streams with an MMA warp each read operands twice and were slower.
//
// Tiles that do not fill a last wave of pairs are split along K over the pairs that would be idle.  Each part's sums go to a workspace, and the
// warp that finds itself the last of a region's parts (a counter per region) adds all of them, in the order of K, and stores: nobody waits, and
// the result does not depend on who came last.
//
// 384 threads: warp 0 TMA, warp 1 MMA (leader CTA), warps 4..11 sums (two warps per lane quarter, one per half of the columns).  A sums
// thread holds 128 sums and 64 values on their way from tensor memory: the first warpgroup gives it registers (56 + 224 + 224 = 3 · 168).
// Tiles leave by TMA from shared memory, a piece of 32 rows × 128 bytes per warp at a time, under the next tile's first blocks; an output
// that TMA cannot write (rows not a multiple of 16 bytes) is stored from the same pieces, a row at a time.
#include "api.h"
#include "sm100.cuh"

namespace b200 {

constexpr int F2_BK = 128, F2_THREADS = 384, F2_GROUP_M = 8;
constexpr int F2_PIECE = 32 * 128, F2_RING = 4;        // bytes of a piece of the tile; blocks of B's scales on their way

template <int NT, bool BTILE>
struct F2 {
  static constexpr int A_BYTES = 128 * F2_BK, B_BYTES = NT / 2 * F2_BK, STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = NT == 256 ? 5 : 7;
  static constexpr int SLOT = NT / 2 * 4 + 128;                    // scales of a block: a warp's columns, then its rows
  static constexpr int SV = BTILE ? 0 : F2_RING * SLOT;
  static constexpr int SMEM = STAGES * STAGE + 8 * (F2_PIECE + SV) + 1024 + 256;
};

struct F2Params {
  void* out;
  const void* bias;
  const float *sa, *sb;
  int64_t ldc, sa_blk, sb_row, sb_blk;
  int M, N, K;
  int out_f32, accumulate, bias_f32, tma_out;
  int whole, splits, per;          // tiles computed whole; parts of each of the others and their blocks of K
  float* ws;                       // [part][CTA of the pair][warp][column][32 rows] sums of the parts
  int* arrived;                    // [split tile][CTA][warp] parts that have arrived
  int* status;
};

__device__ __forceinline__ void f2_mma(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(tmem_d), "l"(da), "l"(db), "r"(idesc), "r"(accumulate)
      : "memory");
}

// tcgen05.wait::ld that the registers of the load pass through, so that nothing which uses them can be placed before it.
__device__ __forceinline__ void f2_ld_wait(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                 "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]),
                 "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]),
                 "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

__device__ __forceinline__ void f2_cp_async16(uint32_t dst, const float* src, int bytes) {      // what is past `bytes` is zero
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void f2_cp_async4(uint32_t dst, const float* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// 16 lanes × 64 fp32 columns → 32 registers: thread t has columns 8 i + 2 (t % 4) + {0, 1} of rows t / 4 (registers 4 i, 4 i + 1) and
// t / 4 + 8 (4 i + 2, 4 i + 3).
__device__ __forceinline__ void f2_ld_16x64(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void f2_tma_add_2d(const CUtensorMap* map, const void* smem_src, int x, int y) {
  asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3}], [%1];"
               ::"l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(smem_src)), "r"(x), "r"(y) : "memory");
}
// Pieces to an output that TMA cannot write.  Two warps per scheduler have nothing to hide instructions behind, so these are few per row: eight
// rows on their way at a time, pointers that advance, all that depends on the alignment outside the loop (a plain loop over rows took 25 instructions
// for 32 columns, and 2048 × 11263 × 256 49 µs instead of 33; 11264 columns, by TMA, 21).
// 32 × 32 fp32 values, lane = column.
__device__ __forceinline__ void f2_store_piece32(const uint8_t* piece, const F2Params& p, int row0, int col0, int lane) {
  const int rows = col0 + lane < p.N ? p.M - row0 : 0;
  float* o = static_cast<float*>(p.out) + static_cast<int64_t>(row0) * p.ldc + col0 + lane;
#pragma unroll 1
  for (int r0 = 0; r0 < 32; r0 += 8) {
    float v[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) v[r] = *reinterpret_cast<const float*>(piece + (r0 + r) * 128 + (((lane >> 2) ^ r) << 4) + ((lane & 3) << 2));
    if (p.accumulate) {
      float old[8];
      const float* in = o;
#pragma unroll
      for (int r = 0; r < 8; ++r, in += p.ldc) old[r] = r0 + r < rows ? *in : 0.f;
#pragma unroll
      for (int r = 0; r < 8; ++r) v[r] += old[r];
    }
#pragma unroll
    for (int r = 0; r < 8; ++r, o += p.ldc) if (r0 + r < rows) *o = v[r];
  }
}
// 32 × 64 bf16 values, two per lane: the rows K, K + STEP, ..  They start on 4 bytes, or (ODD) 2 bytes after such an address, and then get their pairs
// one column later, and the first value and the last by themselves.
template <int STEP, int K, bool ODD>
__device__ __forceinline__ void f2_store_rows(const uint8_t* piece, __nv_bfloat16* o, int64_t ldc, int rows, int cols, int lane) {
  const int c = 2 * lane + (ODD ? 1 : 0);
  const int pair = c + 1 < cols ? rows : 0, last = c < cols && !pair ? rows : 0, first = ODD && lane == 0 && cols > 0 ? rows : 0;
  o += K * ldc;
#pragma unroll 1
  for (int r0 = K; r0 < 32; r0 += 8 * STEP) {
    uint32_t v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v[i] = *reinterpret_cast<const uint32_t*>(piece + (r0 + i * STEP) * 128 + (((lane >> 2) ^ ((K + i * STEP) & 7)) << 4) + ((lane & 3) << 2));
#pragma unroll
    for (int i = 0; i < 8; ++i, o += STEP * ldc) {
      const int r = r0 + i * STEP;
      const uint32_t w = ODD ? __funnelshift_r(v[i], __shfl_down_sync(0xffffffffu, v[i], 1), 16) : v[i];
      if (r < pair) *reinterpret_cast<uint32_t*>(o + c) = w;
      if (r < last) o[c] = __ushort_as_bfloat16(static_cast<unsigned short>(w));
      if (r < first) o[0] = __ushort_as_bfloat16(static_cast<unsigned short>(v[i]));
    }
  }
}
__device__ __forceinline__ void f2_store_piece16(const uint8_t* piece, const F2Params& p, int row0, int col0, int lane) {
  const int rows = p.M - row0, cols = p.N - col0 < 64 ? p.N - col0 : 64;
  __nv_bfloat16* o = static_cast<__nv_bfloat16*>(p.out) + static_cast<int64_t>(row0) * p.ldc + col0;
  const bool odd = (reinterpret_cast<uintptr_t>(o) & 2) != 0;
  if (p.ldc & 1) {
    if (odd) { f2_store_rows<2, 0, true>(piece, o, p.ldc, rows, cols, lane); f2_store_rows<2, 1, false>(piece, o, p.ldc, rows, cols, lane); }
    else { f2_store_rows<2, 0, false>(piece, o, p.ldc, rows, cols, lane); f2_store_rows<2, 1, true>(piece, o, p.ldc, rows, cols, lane); }
  } else if (odd) {
    f2_store_rows<1, 0, true>(piece, o, p.ldc, rows, cols, lane);
  } else {
    f2_store_rows<1, 0, false>(piece, o, p.ldc, rows, cols, lane);
  }
}

template <int NT, bool BTILE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(F2_THREADS, 1)
gemm2_fp8_block_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                       const __grid_constant__ CUtensorMap tmap_out, const F2Params p) {
  using T = F2<NT, BTILE>;
  constexpr int W = NT / 2;                            // columns per thread
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* pieces = smem + T::STAGES * T::STAGE;
  uint8_t* svs = pieces + 8 * F2_PIECE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(svs + 8 * T::SV);
  uint64_t* full_bar = bars;                           // [STAGES] used in the leader CTA
  uint64_t* empty_bar = full_bar + T::STAGES;          // [STAGES] each CTA's producer waits on its own
  uint64_t* tmem_full = empty_bar + T::STAGES;         // [2]      each CTA's sums wait on their own
  uint64_t* tmem_empty = tmem_full + 2;                // [2]      used in the leader CTA, 16 warps
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(tmem_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_ptr + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int pair = static_cast<int>(blockIdx.x) >> 1, n_pair = static_cast<int>(gridDim.x) >> 1;
  const int num_m = (p.M + 255) / 256, num_n = (p.N + NT - 1) / NT;
  const int all_kb = (p.K + F2_BK - 1) / F2_BK;
  const int num_units = p.whole + (num_m * num_n - p.whole) * p.splits;

  if (threadIdx.x == 0) {
    for (int s = 0; s < T::STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(&tmem_full[a], 1); mbar_init(&tmem_empty[a], 16); }
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmap_a); tma_prefetch_desc(&tmap_b);
    if (p.tma_out) tma_prefetch_desc(&tmap_out);
  }
  if (warp == 1) { tmem_alloc_2sm(tmem_ptr, 2 * NT); tmem_relinquish_2sm(); }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();          // the peer's barriers are initialised before anything signals them
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_ptr, 0);

  // work of a pair: a tile, or (past the whole ones) one of the parts of a tile along K
  auto unit = [&](int u, int& m0, int& n0, int& kb0, int& kb1) {
    int t = u;
    kb0 = 0; kb1 = all_kb;
    if (u >= p.whole) {
      const int v = u - p.whole, part = v % p.splits;
      t = p.whole + v / p.splits;
      kb0 = part * p.per; kb1 = min(kb0 + p.per, all_kb);
    }
    const int per_group = F2_GROUP_M * num_n;
    const int g = t / per_group, first_m = g * F2_GROUP_M;
    const int gsz = min(num_m - first_m, F2_GROUP_M);
    const int r = t - g * per_group;
    m0 = (first_m + (r % gsz)) * 256;
    n0 = (r / gsz) * NT;
  };

  uint32_t issued = 0;                                 // blocks that this warp has loaded (warp 0) or multiplied (warp 1)
  if (warp == 0) {                                     // converged: a load from inside a branch of one lane takes longer to issue
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    int stage = 0; uint32_t phase = 0;
    for (int u = pair; u < num_units; u += n_pair) {
      int m0, n0, kb0, kb1; unit(u, m0, n0, kb0, kb1);
      const int ma = m0 + rank * 128, nb = n0 + rank * (NT / 2);
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait_warp(&empty_bar[stage], phase ^ 1, abort_flag, p.status, STATUS_TIMEOUT_EMPTY)) goto done;
        uint8_t* sa = smem + stage * T::STAGE;
        if (elect_one_sync()) {
          if (rank == 0) mbar_arrive_expect_tx(&full_bar[stage], 2 * T::STAGE);       // both CTAs' loads
          tma_load_2d_2sm(sa, &tmap_a, &full_bar[stage], kb * F2_BK, ma);
          tma_load_2d_2sm(sa + T::A_BYTES, &tmap_b, &full_bar[stage], kb * F2_BK, nb);
        }
        ++issued;
        if (++stage == T::STAGES) { stage = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (rank == 0) {                                   // the whole warp, converged; one lane is elected per block
      // e4m3 × e4m3, fp32 accumulate, both operands K-major
      constexpr uint32_t idesc = (1u << 4) | (static_cast<uint32_t>(NT >> 3) << 17) | (static_cast<uint32_t>(256 >> 4) << 24);
      int stage = 0; uint32_t phase = 0, it = 0;
      for (int u = pair; u < num_units; u += n_pair) {
        int m0, n0, kb0, kb1; unit(u, m0, n0, kb0, kb1);
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int acc = it & 1; const uint32_t acc_phase = (it >> 1) & 1;
          if (!mbar_wait_warp(&full_bar[stage], phase, abort_flag, p.status, STATUS_TIMEOUT_FULL)) goto done;
          if (!mbar_wait_warp(&tmem_empty[acc], acc_phase ^ 1, abort_flag, p.status, STATUS_TIMEOUT_TMEM_EMPTY)) goto done;
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * T::STAGE);
          const uint64_t da = make_smem_desc(sa, 16, 1024), db = make_smem_desc(sa + T::A_BYTES, 16, 1024);
          if (elect_one_sync()) {
#pragma unroll
            for (uint32_t k = 0; k < F2_BK / 32; ++k)
              f2_mma(tmem_base + acc * NT, da + static_cast<uint64_t>(k * 2), db + static_cast<uint64_t>(k * 2), idesc, k != 0 ? 1u : 0u);
            umma_commit_2sm(&tmem_full[acc], 3);
            umma_commit_2sm(&empty_bar[stage], 3);
          }
          ++issued;
          if (++stage == T::STAGES) { stage = 0; phase ^= 1; }
        }
      }
    }
  } else if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");      // every warp of the group has to give its registers back
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    const int q = warp & 3, half = (warp - 4) >> 2;    // lane quarter, half of the columns
    uint8_t* piece = pieces + (warp - 4) * F2_PIECE;
    uint8_t* sv = svs + (warp - 4) * T::SV;
    uint32_t it = 0;
    for (int u = pair; u < num_units; u += n_pair) {
      int m0, n0, kb0, kb1; unit(u, m0, n0, kb0, kb1);
      const int row0 = m0 + rank * 128 + q * 32, c0 = n0 + half * W;
      const float* sa = p.sa + min(row0 + lane, p.M - 1);
      const float* sb = BTILE ? p.sb + static_cast<int64_t>(min(c0, p.N - 1) >> 7) * p.sb_row : p.sb + min(c0 + 4 * lane, (p.N - 1) & ~3);
      // scales per row of both: each lane copies four columns and one row of a block
      const int sv_bytes = BTILE || lane >= W / 4 ? 0 : max(min(p.N - c0 - 4 * lane, 4), 0) * 4;
      auto copy_sv = [&](int kb) {
        if (!BTILE) {
          const uint32_t slot = smem_u32(sv + (kb % F2_RING) * T::SLOT);
          const int k = min(kb, kb1 - 1);
          if (lane < W / 4) f2_cp_async16(slot + lane * 16, sb + k * p.sb_blk, kb < kb1 ? sv_bytes : 0);
          f2_cp_async4(slot + W * 4 + lane * 4, sa + k * p.sa_blk, kb < kb1 ? 4 : 0);
          asm volatile("cp.async.commit_group;" ::: "memory");
        }
      };
      float sum[W], scale[8];
#pragma unroll
      for (int i = 0; i < W; ++i) sum[i] = 0.f;
#pragma unroll
      for (int j = 0; j < F2_RING - 1; ++j) copy_sv(kb0 + j);
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const int acc = it & 1; const uint32_t acc_phase = (it >> 1) & 1;
        const uint32_t taddr = tmem_base + acc * NT + half * W + (static_cast<uint32_t>(q * 32) << 16);
        if constexpr (BTILE) {
          const int g = (kb - kb0) & 7;
          if (g == 0) {                                // the row's scales of eight blocks
#pragma unroll
            for (int j = 0; j < 8; ++j) scale[j] = sa[min(kb + j, kb1 - 1) * p.sa_blk];
            const float b = sb[min(kb + (lane & 7), kb1 - 1) * p.sb_blk];
#pragma unroll
            for (int j = 0; j < 8; ++j) scale[j] *= __shfl_sync(0xffffffffu, b, j);
          }
          const float s01 = (g & 1) ? scale[1] : scale[0], s23 = (g & 1) ? scale[3] : scale[2];
          const float s45 = (g & 1) ? scale[5] : scale[4], s67 = (g & 1) ? scale[7] : scale[6];
          const float f = (g & 4) ? ((g & 2) ? s67 : s45) : ((g & 2) ? s23 : s01);
          if (!mbar_wait_warp(&tmem_full[acc], acc_phase, abort_flag, p.status, STATUS_TIMEOUT_TMEM_FULL)) goto done;
          tc_fence_after();
          uint32_t r[2][32];
          tmem_ld_32x32(taddr, r[0]);
#pragma unroll
          for (int c = 0; c < W / 32; ++c) {
            f2_ld_wait(r[c & 1]);
            if (c + 1 < W / 32) {
              tmem_ld_32x32(taddr + (c + 1) * 32, r[(c + 1) & 1]);
            } else {                                   // the last columns are in registers: the accumulator is free
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive_leader(&tmem_empty[acc]);
            }
            const uint32_t (&w)[32] = r[c & 1];
            float* o = sum + c * 32;
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = fmaf(__uint_as_float(w[i]), f, o[i]);
          }
        } else {                                       // piece c: columns 64 (c / 2) .., rows 16 (c % 2) ..
          if (!mbar_wait_warp(&tmem_full[acc], acc_phase, abort_flag, p.status, STATUS_TIMEOUT_TMEM_FULL)) goto done;
          tc_fence_after();
          uint32_t r[2][32];
          f2_ld_16x64(taddr, r[0]);
          copy_sv(kb + F2_RING - 1);                   // into the slot of block kb - 1, which every lane has read
          asm volatile("cp.async.wait_group %0;" ::"n"(F2_RING - 1) : "memory");
          __syncwarp();                                // block kb has arrived
          const float* slot = reinterpret_cast<const float*>(sv + (kb % F2_RING) * T::SLOT);
          float fa[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) fa[j] = slot[W + j * 8 + (lane >> 2)];
          float2 fb[8];
#pragma unroll
          for (int c = 0; c < W / 32; ++c) {
            if ((c & 1) == 0) {
#pragma unroll
              for (int i = 0; i < 8; ++i) fb[i] = mul_f32x2(*reinterpret_cast<const float2*>(slot + (c >> 1) * 64 + i * 8 + (lane & 3) * 2), make_float2(kFp8Down, kFp8Down));
            }
            f2_ld_wait(r[c & 1]);
            if (c + 1 < W / 32) {
              f2_ld_16x64(taddr + ((c + 1) >> 1) * 64 + (static_cast<uint32_t>(((c + 1) & 1) * 16) << 16), r[(c + 1) & 1]);
            } else {
              tc_fence_before();
              __syncwarp();                            // (every lane has read its scales, too)
              if (lane == 0) mbar_arrive_leader(&tmem_empty[acc]);
            }
            const uint32_t (&w)[32] = r[c & 1];
            float* o = sum + c * 32;
            const float2 f0 = make_float2(fa[(c & 1) * 2], fa[(c & 1) * 2]), f1 = make_float2(fa[(c & 1) * 2 + 1], fa[(c & 1) * 2 + 1]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float2 x = fma_f32x2(mul_f32x2(make_float2(__uint_as_float(w[4 * i]), __uint_as_float(w[4 * i + 1])), fb[i]), f0,
                                         make_float2(o[4 * i], o[4 * i + 1]));
              const float2 y = fma_f32x2(mul_f32x2(make_float2(__uint_as_float(w[4 * i + 2]), __uint_as_float(w[4 * i + 3])), fb[i]), f1,
                                         make_float2(o[4 * i + 2], o[4 * i + 3]));
              o[4 * i] = x.x; o[4 * i + 1] = x.y; o[4 * i + 2] = y.x; o[4 * i + 3] = y.y;
            }
          }
        }
      }
      if (!BTILE) {
        asm volatile("cp.async.wait_group 0;" ::: "memory");      // copies past the last block (of zeros)
#pragma unroll
        for (int i = 0; i < W; ++i) sum[i] *= kFp8Up;
      }
      if (u >= p.whole) {                              // one of the parts of a tile
        const int v = u - p.whole, w = rank * 8 + warp - 4;
        float* mine = p.ws + (static_cast<int64_t>(v) * 16 + w) * (W * 32) + lane;
#pragma unroll
        for (int i = 0; i < W; ++i) __stcg(mine + i * 32, sum[i]);
        __threadfence();
        __syncwarp();
        int before = 0;
        if (lane == 0) before = atomicAdd(p.arrived + v / p.splits * 16 + w, 1);
        if (__shfl_sync(0xffffffffu, before, 0) != p.splits - 1) continue;
        __threadfence();
        const float* part = p.ws + (static_cast<int64_t>(v / p.splits * p.splits) * 16 + w) * (W * 32) + lane;
#pragma unroll
        for (int i = 0; i < W; ++i) sum[i] = __ldcg(part + i * 32);
        for (int s = 1; s < p.splits; ++s) {
          part += 16 * W * 32;
#pragma unroll
          for (int i = 0; i < W; ++i) sum[i] += __ldcg(part + i * 32);
        }
      }
      if (p.bias) {
#pragma unroll
        for (int c = 0; c < W / 32; ++c) {
          const int col = min(c0 + c * 32 + lane, p.N - 1);
          const float b = p.bias_f32 ? static_cast<const float*>(p.bias)[col] : __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[col]);
          if (BTILE) {
#pragma unroll
            for (int i = 0; i < 32; ++i) sum[c * 32 + i] += __shfl_sync(0xffffffffu, b, i);
          } else {                                     // columns 32 (c % 2) .. of pieces c / 2 · 2 and the one after
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float v = __shfl_sync(0xffffffffu, b, i * 8 + (lane & 3) * 2 + e);
                float* o = sum + (c >> 1) * 64 + (c & 1) * 16 + i * 4 + e;
                o[0] += v; o[2] += v; o[32] += v; o[34] += v;
              }
            }
          }
        }
      }
      // pieces of 32 rows × 128 bytes: 16-byte parts at part ^ (row % 8), the order of the output's tensor map
      auto part = [&](int j) { return reinterpret_cast<uint4*>(piece + lane * 128 + ((j ^ (lane & 7)) << 4)); };
      auto frag = [&](int g, int j) { return piece + (g * 8 + (lane >> 2)) * 128 + ((j ^ (lane >> 2)) << 4); };      // part j of row 8 g + lane / 4
      if (!p.out_f32) {
#pragma unroll
        for (int c = 0; c < W / 64; ++c) {
          if (lane == 0) tma_store_wait_read<0>();
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (BTILE) {
              const float* v = sum + c * 64 + j * 8;
              *part(j) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
            } else {
#pragma unroll
              for (int g = 0; g < 4; ++g) {            // rows 8 g + lane / 4
                const float* v = sum + c * 64 + (g >> 1) * 32 + j * 4 + (g & 1) * 2;
                *reinterpret_cast<uint32_t*>(frag(g, j) + (lane & 3) * 4) = pack_bf16x2(v[0], v[1]);
              }
            }
          }
          if (p.tma_out) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0 && row0 < p.M && c0 + c * 64 < p.N) { tma_store_2d(&tmap_out, piece, c0 + c * 64, row0); tma_store_commit(); }
          } else {
            __syncwarp();
            f2_store_piece16(piece, p, row0, c0 + c * 64, lane);
            __syncwarp();
          }
        }
      } else {
#pragma unroll
        for (int c = 0; c < W / 32; ++c) {
          if (lane == 0) tma_store_wait_read<0>();
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (BTILE) {
              const float* v = sum + c * 32 + j * 4;
              *part(j) = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
            } else if (j < 4) {
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                const float* v = sum + (c >> 1) * 64 + (g >> 1) * 32 + (c & 1) * 16 + j * 4 + (g & 1) * 2;
                *reinterpret_cast<float2*>(frag(g, 2 * j + ((lane & 3) >> 1)) + (lane & 1) * 8) = make_float2(v[0], v[1]);
              }
            }
          }
          if (p.tma_out) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0 && row0 < p.M && c0 + c * 32 < p.N) {
              if (p.accumulate) f2_tma_add_2d(&tmap_out, piece, c0 + c * 32, row0);
              else tma_store_2d(&tmap_out, piece, c0 + c * 32, row0);
              tma_store_commit();
            }
          } else {
            __syncwarp();
            f2_store_piece32(piece, p, row0, c0 + c * 32, lane);
            __syncwarp();
          }
        }
      }
    }
  }

done:
  if (warp >= 4) {
    tmem_ld_wait();                    // a wait that gave up can leave a load on its way
    if (!BTILE) asm volatile("cp.async.wait_all;" ::: "memory");
    tma_store_wait<0>();
  }
  tc_fence_before();
  __syncthreads();
  // full_bar is the leader's; the other CTA knows that its loads have ended by the products that read them
  if (warp < 2 && *abort_flag) drain_ring(warp == 0 && rank == 0 ? full_bar : empty_bar, T::STAGES, issued);
  __syncwarp();
  cluster_sync_all();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc_2sm(tmem_base, 2 * NT);
  }
}

int make_tmap_2d_u8(CUtensorMap* map, const void* ptr, uint64_t inner, uint64_t outer, uint64_t row_stride_bytes,
                    uint32_t box_inner, uint32_t box_outer);

// The output in boxes of 32 rows × 128 bytes, 16-byte parts swizzled by the row.
static int make_tmap_out(CUtensorMap* map, void* ptr, int f32, uint64_t cols, uint64_t rows, uint64_t ld) {
  typedef CUresult (*Encode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                             const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static Encode fn = nullptr;
  if (!fn) {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult res;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &res) != cudaSuccess || res != cudaDriverEntryPointSuccess) return -1;
    fn = reinterpret_cast<Encode>(f);
  }
  const cuuint64_t dim[2] = {cols, rows}, stride[1] = {ld * (f32 ? 4 : 2)};
  const cuuint32_t box[2] = {f32 ? 32u : 64u, 32}, step[2] = {1, 1};
  const CUresult r = fn(map, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, ptr, dim, stride, box, step,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : static_cast<int>(r);
}

template <int NT, bool BTILE>
static int launch_f2(const void* A, int64_t lda, const void* B, int64_t ldb, const F2Params& p, int num_sms, cudaStream_t st) {
  using T = F2<NT, BTILE>;
  CUtensorMap ta, tb, to;
  int rc = make_tmap_2d_u8(&ta, A, p.K, p.M, lda, F2_BK, 128);
  if (!rc) rc = make_tmap_2d_u8(&tb, B, p.K, p.N, ldb, F2_BK, NT / 2);
  to = tb;
  if (!rc && p.tma_out) rc = make_tmap_out(&to, p.out, p.out_f32, p.N, p.M, p.ldc);
  if (rc) return rc;
  auto kern = gemm2_fp8_block_kernel<NT, BTILE>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, T::SMEM) != cudaSuccess) return -2;
  const int64_t tiles = static_cast<int64_t>((p.M + 255) / 256) * ((p.N + NT - 1) / NT);
  const int64_t units = p.whole + (tiles - p.whole) * p.splits;
  if (units > 0x3fffffff) return -6;
  if (p.splits > 1 && cudaMemsetAsync(p.arrived, 0, (tiles - p.whole) * 16 * sizeof(int), st) != cudaSuccess) return -4;
  const int pairs = num_sms / 2;
  kern<<<2 * (units < pairs ? static_cast<int>(units) : pairs), F2_THREADS, T::SMEM, st>>>(ta, tb, to, p);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

}  // namespace b200

// How a product is laid over the pairs of SMs: the width of its tiles, and the split of those that do not fill a last wave.
namespace b200 {
struct F2Plan { int nt, whole, splits, per; int64_t ws_floats; int counters; double cost; };
static F2Plan f2_plan(int M, int N, int K, int num_sms) {
  const int pairs = num_sms / 2, num_kb = (K + F2_BK - 1) / F2_BK;
  F2Plan best{};
  for (int nt = 256; nt >= 128; nt /= 2) {
    const int64_t tiles = static_cast<int64_t>((M + 255) / 256) * ((N + nt - 1) / nt);
    const int rest = static_cast<int>(tiles % pairs);
    // in blocks of 256 columns: a block of 128 columns takes 0.62 of the time; a tile's set-up and end take 4 blocks, the sums of a split tile
    // (written, counted and read again) 10 and 3 per part: 2048 × 5632 × 16384 294 µs whole, 257 with its last tiles split, 1024 × 1024 × 16384 81 and 53, but
    // 700 × 7680 × 2560 33 and 35, 16384 × 5632 × 2048 190 and 199, 128 × 2048 × 5632 25 and 29
    const double blk = nt == 256 ? 1.0 : 0.62, tile = num_kb * blk + 4;
    int splits = 1, per = num_kb;
    double last = rest ? tile : 0;
    if (rest) {
      int s = pairs / rest;
      s = s < 8 ? s : 8;
      s = s < num_kb / 2 ? s : num_kb / 2;
      if (s > 1) {
        const int pk = (num_kb + s - 1) / s;
        s = (num_kb + pk - 1) / pk;
        const double split = pk * blk + 4 + 10 + 3 * s;
        if (split < last) { last = split; splits = s; per = pk; }
      }
    }
    const double cost = static_cast<double>(tiles / pairs) * tile + last;
    if (nt == 256 || cost < best.cost) {
      const int64_t parts = splits > 1 ? static_cast<int64_t>(rest) * splits : 0;
      best = F2Plan{nt, static_cast<int>(splits > 1 ? tiles - rest : tiles), splits, per, parts * 256 * nt, splits > 1 ? rest * 16 : 0, cost};
    }
  }
  return best;
}
// About how many µs the product takes, to choose between this kernel and the one for few rows (a line through 64 to 512 rows by 256 to 11264
// columns, K 256 to 8192).
double f2_microseconds(int M, int N, int K, int sb_tile, int num_sms) {
  const double cost = f2_plan(M, N, K, num_sms).cost;
  return sb_tile ? 2.6 + 0.52 * cost : 3.0 + 0.8 * cost;
}
}  // namespace b200

// Bytes of workspace that b200_gemm2_fp8_block needs for these sizes (0: none).
extern "C" int64_t b200_gemm2_fp8_block_workspace(int M, int N, int K, int num_sms) {
  const b200::F2Plan plan = b200::f2_plan(M, N, K, num_sms);
  return plan.ws_floats * 4 + plan.counters * 4;
}

// Contract of b200_gemm_fp8_block, which checks the arguments and calls this: scales of A are per row, those of B per row or (sb_tile) per 128
// rows; scales per row are stored [block][*_blk], those of B 16-byte aligned.  ws: the bytes that b200_gemm2_fp8_block_workspace names.
extern "C" int b200_gemm2_fp8_block(const void* A, int64_t lda, const float* sa, int64_t sa_blk, const void* B, int64_t ldb, const float* sb,
                                    int64_t sb_row, int64_t sb_blk, int sb_tile, const void* bias, int bias_f32, void* out, int64_t ldc, int M,
                                    int N, int K, int out_f32, int accumulate, void* ws, int num_sms, int* status, cudaStream_t stream) {
  using namespace b200;
  const int tma_out = ldc * (out_f32 ? 4 : 2) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0 ? 1 : 0;
  const F2Plan plan = f2_plan(M, N, K, num_sms);
  if (plan.splits > 1 && !ws) return -6;
  float* sums = static_cast<float*>(ws);
  const F2Params p{out, bias, sa, sb, ldc, sa_blk, sb_row, sb_blk, M, N, K, out_f32, accumulate, bias_f32, tma_out, plan.whole, plan.splits,
                   plan.per, sums, reinterpret_cast<int*>(sums + plan.ws_floats), status};
  if (plan.nt == 256)
    return sb_tile ? launch_f2<256, true>(A, lda, B, ldb, p, num_sms, stream) : launch_f2<256, false>(A, lda, B, ldb, p, num_sms, stream);
  return sb_tile ? launch_f2<128, true>(A, lda, B, ldb, p, num_sms, stream) : launch_f2<128, false>(A, lda, B, ldb, p, num_sms, stream);
}
