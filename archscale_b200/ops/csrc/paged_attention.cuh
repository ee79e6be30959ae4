// Attention of a few new tokens over a paged key-value cache (layout in paged.cuh), keys and values read once for every tile of at most 16 query rows of a
// key head, or 8 of a pair of them: once for a token or a few drafts.  Whole prompt parts are right, but every tile reads the prefix again (2048 new tokens over
// 8192, H 16, G 4, D 128: 1084 us, where the products alone need 94).
//
// Mathematics.  One pass over the keys with a running maximum and sum (base 2, 32 bits):  x_j = log₂e · scale · q·k_j,  p_j = 2^(x_j − m),
// o = Σ p_j v_j / Σ p_j.  Parts of a sequence are joined by  m = max m_i,  l = Σ l_i 2^(m_i − m),  o = Σ o_i 2^(m_i − m).
// In e4m3 a key's power of two multiplies its score; a value's, 2^e_j, goes into the weight, p'_j = 2^(x_j + e_j − m' + 14), whose maximum m' is kept
// beside m: no value is too small or large beside another, whatever their scales.
//
// Tokens are the rows of the MMAs (m16n8k16), query rows their 8 columns: scores are K · Qᵀ, outputs Vᵀ · Pᵀ.  So a call of a few query rows wastes nothing,
// a warp's sums take D · 8 floats, and keys and values are left operands straight from memory order.  P turns from a result (tokens down) into a right
// operand (tokens along k) by transposing 8 × 8 blocks between registers.  Columns:
//   plain    the H/G heads of the key head times T tokens, 8 · NC to a tile
//   PAIRS    differential attention: 4 rows of branch 1 as [q1 | 0], then the same 4 of branch 2 as [0 | q2], against keys [k1 | k2] and
//            values [v1 | v2]: one read and one product for both branches
// Rounding: q is exact (bf16; for fp16 times a power of two of its row).  In bf16 P enters as two halves, hi and p − hi, so that it is good to 2⁻¹⁷: its plain
// rounding, 2⁻⁹ of each weight, would be as large as that of the result, and the second product costs nothing where the tensor cores wait for memory.
// In e4m3 the products run in fp16, weights (from 2¹⁴ down to 2⁻²⁴) as two halves too: good to 2⁻²² where one half left 2⁻¹¹.
//
// What bounds it: memory in bf16 (16 sequences of 16384, H 16, G 4, D 128: 537 MB in 91 us by the kernel alone with cold caches, 0.90 of the copy rate, in pairs
// 93; as called, with launch and join, 64 ragged sequences up to 8192, 605 MB: 111 us, 0.83; 32 in pairs of heads of 64, G 20, 755 MB: 135 us, 0.85).  At most 16 columns are 32 operations a byte; tcgen05 would take 128 rows of keys too, but wants P through shared memory
// and its sums through tensor memory for every tile, which is the longer chain where a CTA has a handful of tiles.  In e4m3 instructions and their
// latency: 770 for a step of 32 tokens, 220 of them conversions (one sequence of 131072 tokens: 135 MB in 37 us, 0.55), with some 12 us of first loads, last
// steps and the second kernel.  Few and short sequences: latency (1000 tokens 4 us behind the launch).
//
// Each warp is on its own: it loads its tokens with cp.async into its own ring (two stages of 16 or 32 tokens, 8 KB; three CTAs an SM; three stages on two
// CTAs were no faster), and no barrier joins warps before the end of a work item.  Pages are looked up two steps ahead, so that their latency is not in the chain.
//
// Work.  Lengths are known on the device only.  An item is (sequence, tile of rows, key head); its keys are chunks, one step of each warp.  Every CTA adds
// up the chunks of all items from the lengths and takes a contiguous share of them, equal to one chunk, so that one long sequence or many short ones fill
// the device alike.  Items that lie in one CTA are finished there; the parts of the others meet in a second kernel (joined in the order of the keys: results
// do not depend on scheduling), which the first one starts early and which needs no counters, so that nothing has to be zero beforehand.  Few items of
// a few chunks run on clusters of eight CTAs instead, which join their parts in shared memory (pa_prepare).
#pragma once
#include <cuda_fp16.h>
#include <atomic>
#include <type_traits>

#include "paged.cuh"

namespace b200 {

constexpr int PA_ENTRIES = 1024;           // (sequence, tile of rows) of one launch

struct PaArgs {
  PagedView c;
  b200_paged_query a;
  int b0, nb, rt0, nrt;                    // sequences and tiles of rows of this launch
  int rows, per;                           // rows of a key head, and of one token among them
  int heads;                               // key heads, or pairs of them
  int ncta, piece, q_words;                // bytes of a copy where rows are not whole 16-byte pieces; queries start on 4-byte boundaries
  int64_t page_b, group_b, slot_b;         // strides in bytes, of keys as of values
  uint32_t page_16, slot_16;               // the same in units of 16 bytes (not GEN)
  uint32_t ks_page, ks_slot, vs_page, vs_slot;      // strides of the scales (not GEN)
  int same_scales, q_wide;                 // those of keys as of values; queries start on 8-byte boundaries
  int page_shift;                          // log2 of the page size, or -1
  float* parts;                            // [ncta][2] parts of items
  int* prefix;                             // chunks before each entry, from CTA 0
};

// What a shape needs.  ES: bytes of an element; DT: values of a row of keys, of both heads of a pair; NC: groups of 8 columns.
template <int ES, int DT, bool PAIRS, int NC>
struct PaShape {
  static constexpr int ROW = DT * ES;                                          // bytes of a token in a stage
  static constexpr int TS = ES == 2 ? (DT == 64 ? 32 : 16) : (DT == 256 ? 16 : 32);   // tokens of a warp's step
  static constexpr int HEADS = PAIRS ? 2 : 1;
  static constexpr int TILE = TS * ROW;
  static constexpr int SCALES = ES == 1 ? HEADS * TS * 8 : 0;                  // factors of keys, exponents of values
  static constexpr int STAGE = 2 * TILE, EXTRA = SCALES + 16;                  // keys and values; beside them the scales and the mask of tokens
  static constexpr int STAGES = 2;
  static constexpr int WARPS = STAGE > 12288 ? 6 : 4;                          // six where one CTA has the SM to itself
  static constexpr int RING = WARPS * STAGES * (STAGE + EXTRA);
  static constexpr int COLS = 8 * NC;
  static constexpr int QROWS = PAIRS ? 4 * NC : 8 * NC;                        // query rows of a tile
  static constexpr int LD = DT + 4;                                            // floats between rows in shared memory: no bank twice
  static constexpr int SLABS = WARPS * COLS * LD * 4;
  static constexpr int CHUNK = WARPS * TS;
  static constexpr int NG = ES == 1 ? HEADS : 0;                               // groups of values with maxima of their own
  static constexpr int PART = COLS * (DT + 4);                                 // floats of a part: sums, then m, l, m' of each column
  static constexpr int SMEM = RING > SLABS + PART * 4 ? RING : SLABS + PART * 4;
  static_assert(SMEM <= 227 * 1024 - 6144, "shared memory");
};
// column of a tile's query row r, in branch 0 or 1
template <bool PAIRS>
__host__ __device__ constexpr int pa_column(int r, int branch) { return PAIRS ? (r >> 2) * 8 + (r & 3) + 4 * branch : r; }

// CTAs of an SM: as many as its shared memory and the registers of the sums allow
template <int ES, int DT, bool PAIRS, int NC>
constexpr int pa_resident() {
  constexpr int one = PaShape<ES, DT, PAIRS, NC>::SMEM + (PA_ENTRIES + 1) * 4 + 2304;      // its static part and what the system keeps
  constexpr int fit = 228 * 1024 / one, regs = DT * NC >= 512 ? 2 : DT * NC >= 256 ? 3 : 4;
  return fit < regs ? fit : regs;
}

// Shares of `all` chunks: CTA c has those from pa_first(c) to pa_first(c + 1), one more or less than any other; pa_owner is the CTA of a chunk.
__device__ __forceinline__ uint32_t pa_first(uint32_t c, uint32_t all, uint32_t ctas) { return static_cast<uint32_t>(static_cast<uint64_t>(c) * all / ctas); }
__device__ __forceinline__ uint32_t pa_owner(uint32_t chunk, uint32_t all, uint32_t ctas) {
  return static_cast<uint32_t>((static_cast<uint64_t>(chunk + 1) * ctas - 1) / all);
}

__device__ __forceinline__ float pa_ex2(float x) {
  float y;
  asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^(x - y) of maxima, 0 where there was none
__device__ __forceinline__ float pa_step(float x, float y) { return x == -INFINITY ? 0.f : pa_ex2(x - y); }

// Keys that the rows of a tile can see: [lo, hi); first position pos0, tokens t0 … t1 (t1 < t0: no row is there).
struct PaSpan { int lo, hi, t0, t1; int64_t pos0; };
template <int QROWS>
__device__ __forceinline__ PaSpan pa_span(const PaArgs& p, int entry) {
  const int b = p.b0 + entry / p.nrt, rt = p.rt0 + entry % p.nrt;
  const int n = paged_new(p.c, b, p.a.T);
  PaSpan s;
  s.pos0 = static_cast<int64_t>(p.c.lengths[b]) - n;
  s.t0 = rt * QROWS / p.per;
  s.t1 = min((min(rt * QROWS + QROWS, p.rows) - 1) / p.per, n - 1);
  const int64_t room = static_cast<int64_t>(p.c.table_cols) * p.c.page_size;
  const int64_t hi = s.t1 < s.t0 ? 0 : max(int64_t(0), min(s.pos0 + s.t1 + 1, room));
  const int64_t lo = p.a.window >= 0 ? max(int64_t(0), s.pos0 + s.t0 - p.a.window) : 0;
  s.hi = static_cast<int>(min(hi, int64_t(0x7fffff00)));
  s.lo = static_cast<int>(min(lo, static_cast<int64_t>(s.hi)));
  return s;
}

// Epilogue of a row, by a warp: v[i] is the sum of column lane + 32 i (and v2 of branch 2), scaled to maxima m, m' and with l the sum of weights.
template <int ES, int DT, bool PAIRS>
__device__ __forceinline__ void pa_finish(const PaArgs& p, int b, int head, int row, bool there, float (&v)[DT / 32], float (&v2)[DT / 32], const float (&m)[2],
                                          const float (&l)[2], const float (&mv)[2][2], int lane) {
  constexpr int N = DT / 32;
  const int D = p.c.dim, t = row / p.per, hh = row % p.per;
  if constexpr (!PAIRS) {
    const int h = head * p.per + hh;
    float top = m[0], sum = l[0];
    if (p.a.sink != nullptr && there) {
      const float s = paged_param(p.a.sink, p.a.sink_type, h) * 1.4426950408889634f;
      const float mm = fmaxf(top, s);
      sum = (top == -INFINITY ? sum : sum * pa_ex2(top - mm)) + pa_step(s, mm);
      top = mm;
    }
    const float f = sum == 0.f ? 0.f : (ES == 1 ? pa_step(mv[0][0], top + 14.f) : pa_step(m[0], top)) / sum;
    if (p.a.lse != nullptr && lane == 0)
      p.a.lse[(static_cast<int64_t>(b) * p.a.H + h) * p.a.T + t] = !there || sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.a.out) + ((static_cast<int64_t>(b) * p.a.T + t) * p.a.H + h) * D;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (lane + 32 * i < D) out[lane + 32 * i] = __float2bfloat16_rn(there && sum != 0.f ? v[i] * f : 0.f);
  } else {
    const int pair = head * p.per + hh;
    const float lam = paged_param(p.a.lam, p.a.lam_type, 0);
    float total = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int g = i >= N / 2;
      const float f1 = l[0] == 0.f ? 0.f : (ES == 1 ? pa_step(mv[0][g], m[0] + 14.f) : 1.f) / l[0];
      const float f2 = l[1] == 0.f ? 0.f : (ES == 1 ? pa_step(mv[1][g], m[1] + 14.f) : 1.f) / l[1];
      v[i] = (l[0] == 0.f ? 0.f : v[i] * f1) - lam * (l[1] == 0.f ? 0.f : v2[i] * f2);         // columns past D are zero
      total += v[i] * v[i];
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    const float r = rsqrtf(total / (2 * D) + p.a.eps) * p.a.gain;
    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.a.out) + ((static_cast<int64_t>(b) * p.a.T + t) * p.a.H + 2 * pair) * D;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int half = i >= N / 2, d = lane + 32 * i - half * (DT / 2), at = half * D + d;
      if (d < D) out[at] = __float2bfloat16_rn(there ? v[i] * r * paged_param(p.a.w, p.a.w_type, at) : 0.f);
    }
  }
}

template <int ES>
__device__ __forceinline__ void pa_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (ES == 2)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the transpose of an 8 × 8 block of 16-bit values
__device__ __forceinline__ uint32_t pa_turn(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <bool TRANS>
__device__ __forceinline__ void pa_ldsm(uint32_t (&r)[4], uint32_t addr) {
  if constexpr (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// four e4m3 values as fp16: the lower two, the upper two
__device__ __forceinline__ void pa_halves(uint32_t four, uint32_t& lo, uint32_t& hi) {
  asm("{ .reg .b16 x, y; mov.b32 {x, y}, %2; cvt.rn.f16x2.e4m3x2 %0, x; cvt.rn.f16x2.e4m3x2 %1, y; }" : "=r"(lo), "=r"(hi) : "r"(four));
}
// x, y in 16 bits, and what that leaves
template <int ES>
__device__ __forceinline__ uint32_t pa_pack(float x, float y) {
  if constexpr (ES == 2) { const __nv_bfloat162 h = __floats2bfloat162_rn(x, y); return *reinterpret_cast<const uint32_t*>(&h); }
  else { const __half2 h = __floats2half2_rn(x, y); return *reinterpret_cast<const uint32_t*>(&h); }
}
template <int ES>
__device__ __forceinline__ uint32_t pa_rest(float x, float y, uint32_t hi) {
  if constexpr (ES == 2) return pa_pack<2>(x - __uint_as_float(hi << 16), y - __uint_as_float(hi & 0xffff0000u));
  else { const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi)); return pa_pack<1>(x - h.x, y - h.y); }
}
template <int BYTES>
__device__ __forceinline__ void pa_copy(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
template <int BYTES>
__device__ __forceinline__ void pa_copy(uint32_t dst, const void* src, bool live) {
  const int n = live ? BYTES : 0;
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(n) : "memory");
}
// byte of 16-byte piece `chunk` of token t in a tile: pieces of 8 tokens that a matrix load takes together lie in 8 different bank groups
template <int ROW>
__device__ __forceinline__ constexpr uint32_t pa_swizzle(int t) { return (ROW >= 128 ? t & 7 : t >> 1 & 3) << 4; }
template <int ROW>
__device__ __forceinline__ uint32_t pa_at(int t, int chunk) { return t * ROW + ((chunk << 4) ^ pa_swizzle<ROW>(t)); }

// the CTAs of a cluster, all threads
__device__ __forceinline__ void pa_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// a float at the place of `p` in the shared memory of the cluster's CTA `rank`
__device__ __forceinline__ float pa_remote(const float* p, int rank) {
  float x;
  asm volatile("{ .reg .b32 a; mapa.shared::cluster.u32 a, %1, %2; ld.shared::cluster.f32 %0, [a]; }" : "=f"(x) : "r"(smem_u32(p)), "r"(rank) : "memory");
  return x;
}

// GEN: rows that are not whole 16-byte pieces, or shorter than DT.  CLUSTER: an item is eight CTAs, which share its keys evenly and join their parts
// through each other's shared memory, each the rows of its rank
template <int ES, int DT, bool PAIRS, int NC, bool GEN, bool CLUSTER>
__global__ void __launch_bounds__(PaShape<ES, DT, PAIRS, NC>::WARPS * 32, pa_resident<ES, DT, PAIRS, NC>()) paged_attention_kernel(const PaArgs p) {
  using S = PaShape<ES, DT, PAIRS, NC>;
  constexpr bool E8 = ES == 1;
  constexpr int TS = S::TS, MT = TS / 16, KS = DT / 16, HEADS = S::HEADS, NG = S::NG, NGX = NG > 0 ? NG : 1;
  extern __shared__ __align__(512) uint8_t smem[];
  __shared__ int s_prefix[PA_ENTRIES + 1];
  __shared__ int s_scan[S::WARPS];
  __shared__ float s_stat[S::WARPS][4][16];                                     // m, l, m' of both groups
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, cq = lane & 3;
  if constexpr (!CLUSTER) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- chunks before every entry
  const int entries = p.nb * p.nrt;
  if constexpr (!CLUSTER) {
    const int each = (entries + S::WARPS * 32 - 1) / (S::WARPS * 32), from = threadIdx.x * each;
    int sum = 0;
    for (int i = from; i < min(from + each, entries); ++i) {
      const PaSpan s = pa_span<S::QROWS>(p, i);
      const int n = max(1, (s.hi - s.lo + S::CHUNK - 1) / S::CHUNK);            // an item without keys is visited for its zeros
      s_prefix[i] = n;
      sum += n;
    }
    int scan = sum;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) { const int y = __shfl_up_sync(0xffffffffu, scan, o); if (lane >= o) scan += y; }
    if (lane == 31) s_scan[warp] = scan;
    __syncthreads();
    int base = scan - sum;
    for (int w = 0; w < warp; ++w) base += s_scan[w];
    for (int i = from; i < min(from + each, entries); ++i) { const int n = s_prefix[i]; s_prefix[i] = base; base += n; }
    if (threadIdx.x == 0) { int all = 0; for (int w = 0; w < S::WARPS; ++w) all += s_scan[w]; s_prefix[entries] = all; }
  }
  if (GEN)                                                                      // columns past D stay zero
    for (int i = threadIdx.x; i < S::RING / 16; i += S::WARPS * 32) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  if (!CLUSTER && blockIdx.x == 0 && p.prefix != nullptr)
    for (int i = threadIdx.x; i <= entries; i += S::WARPS * 32) p.prefix[i] = s_prefix[i];

  uint32_t begin = 0, end = 1;
  if constexpr (!CLUSTER) {
    const uint32_t all = static_cast<uint32_t>(s_prefix[entries]) * p.heads, ctas = min(all, static_cast<uint32_t>(p.ncta));
    if (blockIdx.x >= ctas) return;
    begin = pa_first(blockIdx.x, all, ctas); end = pa_first(blockIdx.x + 1, all, ctas);
  }
  uint8_t* const ring = smem + warp * S::STAGES * S::STAGE;                     // stages start at multiples of 512 bytes, so that addresses in a row are XORs
  uint8_t* const extra = smem + S::WARPS * S::STAGES * S::STAGE + warp * S::STAGES * S::EXTRA;
  const uint32_t ring_u = smem_u32(ring);
  // this lane's row and piece in the matrix loads: keys by rows of tokens, values transposed
  const uint32_t own_k = pa_at<S::ROW>(lane & 15, lane >> 4), own_v = E8 ? own_k : pa_at<S::ROW>((lane & 7) + (lane >> 4) * 8, lane >> 3 & 1);
  constexpr float LOG2E = 1.4426950408889634f;
  constexpr uint32_t FULL = TS == 32 ? 0xffffffffu : (1u << (TS & 31)) - 1u;

#pragma unroll 1
  for (uint32_t at = begin; at < end;) {
    // ---- the item
    int e = 0;
    uint32_t chunks = 0, head = 0, c0 = 0, c1 = 0;
    if constexpr (CLUSTER) {
      e = blockIdx.x / 8 / p.heads; head = blockIdx.x / 8 % p.heads;
    } else {
      for (int hi = entries; hi - e > 1;) { const int mid = (e + hi) >> 1; if (static_cast<uint32_t>(s_prefix[mid]) * p.heads <= at) e = mid; else hi = mid; }
      chunks = s_prefix[e + 1] - s_prefix[e];
      const uint32_t off = at - static_cast<uint32_t>(s_prefix[e]) * p.heads;
      head = off / chunks; c0 = off - head * chunks; c1 = min(chunks, c0 + end - at);
    }
    const int b = p.b0 + e / p.nrt, row0 = (p.rt0 + e % p.nrt) * S::QROWS;
    const PaSpan sp = pa_span<S::QROWS>(p, e);
    if constexpr (CLUSTER) {
      chunks = (sp.hi - sp.lo + S::CHUNK - 1) / S::CHUNK;
      c0 = blockIdx.x % 8 * chunks / 8; c1 = (blockIdx.x % 8 + 1) * chunks / 8;
    }
    const int j_base = sp.lo + c0 * S::CHUNK + warp * TS;                       // first token of this warp's step 0
    const int steps = static_cast<int>(c1 - c0);

    // ---- queries: column gq of each group is loaded by this thread
    auto column = [&](int n, int& row, int& branch) {                           // column n of 8 · NC
      row = row0 + (PAIRS ? (n >> 3) * 4 + (n & 3) : n);
      branch = PAIRS ? n >> 2 & 1 : 0;
    };
    uint32_t qb[NC][KS][2];
    float factor[NC][2];                                                        // of the columns 2 cq, 2 cq + 1 whose scores this thread gets
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      int row, branch;
      column(c * 8 + gq, row, branch);
      const int t = p.a.T == 1 ? 0 : row / p.per, in_group = head * p.per + row - t * p.per, h = PAIRS ? 2 * in_group + branch : in_group;
      const bool there = row < p.rows && t <= sp.t1;
      const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(p.a.q) + b * p.a.q_batch + t * p.a.q_token + h * p.a.q_head;
      auto two = [&](int ks, int w) -> uint32_t {                               // values d, d + 1 (d even; so is D)
        int d = E8 ? 16 * ks + 4 * cq + 2 * w : 16 * ks + 2 * cq + 8 * w;
        if (PAIRS) d -= branch * (DT / 2);
        if (!there || d < 0 || d >= p.c.dim || (PAIRS && d >= DT / 2)) return 0u;
        if (p.q_words) return *reinterpret_cast<const uint32_t*>(src + d);
        return static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(src + d)) | static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(src + d + 1)) << 16;
      };
      if (!GEN && p.q_wide) {                                                   // whole rows: no checks, and 8 bytes at a time where values are neighbours
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          uint2 u = make_uint2(0u, 0u);
          if (there && (!PAIRS || (ks >= KS / 2) == (branch == 1))) {
            const __nv_bfloat16* const at_ks = src + 16 * ks - (PAIRS ? branch * (DT / 2) : 0);
            if constexpr (E8) u = *reinterpret_cast<const uint2*>(at_ks + 4 * cq);
            else u = make_uint2(*reinterpret_cast<const uint32_t*>(at_ks + 2 * cq), *reinterpret_cast<const uint32_t*>(at_ks + 2 * cq + 8));
          }
          qb[c][ks][0] = u.x; qb[c][ks][1] = u.y;
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int w = 0; w < 2; ++w) qb[c][ks][w] = two(ks, w);
      }
    }

    // ---- loads: lane i < TS knows token i of a step
    const uint8_t* const kb = static_cast<const uint8_t*>(p.c.k) + static_cast<int64_t>(head) * HEADS * p.group_b;
    const uint8_t* const vb = static_cast<const uint8_t*>(p.c.v) + static_cast<int64_t>(head) * HEADS * p.group_b;
    const int piece0 = lane % (S::ROW / 16);
    const int64_t lane_b = HEADS == 2 && piece0 >= S::ROW / 32 ? p.group_b + (piece0 - S::ROW / 32) * 16 : piece0 * 16;
    const uint8_t* const k_lane = kb + lane_b;
    const uint8_t* const v_lane = vb + lane_b;
    const int* const table = p.c.table + b * p.c.table_row;
    const uint8_t* const ks = E8 ? p.c.ks + static_cast<int>(head) * HEADS * p.c.ks_group : nullptr;
    const uint8_t* const vs = E8 ? p.c.vs + static_cast<int>(head) * HEADS * p.c.vs_group : nullptr;
    auto page_of = [&](int j) { return p.page_shift >= 0 ? j >> p.page_shift : j / p.c.page_size; };
    // this lane's token of a step, and how many steps have one: hi is within the table, and a step of the item begins before hi
    const int j_lane = j_base + lane, mine_of = lane < TS && j_lane < sp.hi ? min(steps, (sp.hi - j_lane + S::CHUNK - 1) / S::CHUNK) : 0;
    auto look = [&](int step) { return step < mine_of ? table[page_of(j_lane + step * S::CHUNK)] : -1; };      // its page, or -1
    int page_a = look(0), page_b = look(1);
    uint32_t pend_k[HEADS] = {}, pend_v[HEADS] = {};
    auto issue = [&](int step) {
      bool scaled = false;
      int64_t scale_at = 0, scale_at_v = 0;
      if (step < steps) {
        const int j = j_lane + step * S::CHUNK;
        int page = page_a;
        if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(p.c.pages)) {  // no token, or not a page of this cache
          if (step < mine_of && p.c.status) atomicCAS(p.c.status, 0, STATUS_INDEX_RANGE);
          page = -1;
        }
        page_a = page_b;
        page_b = look(step + 2);
        const int slot = page >= 0 ? j - page_of(j) * p.c.page_size : 0;
        if (E8 && page >= 0) {
          scaled = true;
          if constexpr (GEN) { scale_at = page * p.c.ks_page + slot * p.c.ks_slot; scale_at_v = page * p.c.vs_page + slot * p.c.vs_slot; }
          else { scale_at = page * p.ks_page + slot * p.ks_slot; scale_at_v = p.same_scales ? scale_at : page * p.vs_page + slot * p.vs_slot; }
        }
        const uint32_t live = __ballot_sync(0xffffffffu, page >= 0);
        const uint32_t st = ring_u + (step % S::STAGES) * S::STAGE;
        if (lane == 0) *reinterpret_cast<uint32_t*>(extra + (step % S::STAGES) * S::EXTRA + S::SCALES) = live;
        if (live != 0) {
          if constexpr (!GEN) {
            constexpr int PPR = S::ROW / 16;                                    // a lane has one piece of every (32 / PPR)-th token
            const uint32_t mine = page >= 0 ? page * p.page_16 + slot * p.slot_16 : 0u;
            constexpr int TPI = 32 / PPR;
            const uint32_t own = pa_at<S::ROW>(lane / PPR, lane % PPR);
            if (live == FULL) {
#pragma unroll
              for (int i = 0; i < TS / TPI; ++i) {
                const int64_t o = static_cast<int64_t>(__shfl_sync(0xffffffffu, mine, i * TPI + lane / PPR)) * 16;
                const uint32_t to = st + (own ^ pa_swizzle<S::ROW>(i * TPI)) + i * TPI * S::ROW;
                pa_copy<16>(to, k_lane + o);
                pa_copy<16>(to + S::TILE, v_lane + o);
              }
            } else {
#pragma unroll
              for (int i = 0; i < TS / TPI; ++i) {
                const int t = i * TPI + lane / PPR;
                const int64_t o = static_cast<int64_t>(__shfl_sync(0xffffffffu, mine, t)) * 16;
                const uint32_t to = st + (own ^ pa_swizzle<S::ROW>(i * TPI)) + i * TPI * S::ROW;
                pa_copy<16>(to, k_lane + o, live >> t & 1u);
                pa_copy<16>(to + S::TILE, v_lane + o, live >> t & 1u);
              }
            }
          } else {
            const int ppr = p.c.dim * ES / p.piece;
            const int64_t mine = page >= 0 ? page * p.page_b + slot * p.slot_b : -1;
            for (int t = 0; t < TS; ++t) {
              const int64_t o = __shfl_sync(0xffffffffu, mine, t);
#pragma unroll
              for (int h = 0; h < HEADS; ++h)
                for (int pc = lane; pc < ppr; pc += 32) {
                  const int byte = pc * p.piece, in = h * (DT / 2) * ES + byte;
                  const int64_t from = o < 0 ? 0 : o + h * p.group_b + byte;
                  const uint32_t to = st + pa_at<S::ROW>(t, in >> 4) + (in & 15);
                  if (p.piece == 16) { pa_copy<16>(to, kb + from, o >= 0); pa_copy<16>(to + S::TILE, vb + from, o >= 0); }
                  else if (p.piece == 8) { pa_copy<8>(to, kb + from, o >= 0); pa_copy<8>(to + S::TILE, vb + from, o >= 0); }
                  else { pa_copy<4>(to, kb + from, o >= 0); pa_copy<4>(to + S::TILE, vb + from, o >= 0); }
                }
            }
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      if constexpr (E8) {
        if (step > 0 && lane < TS) {                                            // scales asked for one step ago
          float* const to = reinterpret_cast<float*>(extra + ((step - 1) % S::STAGES) * S::EXTRA);
#pragma unroll
          for (int h = 0; h < HEADS; ++h) {
            // 2^(byte − 127), and byte − 127 by the fraction of 2^23 + byte; 255 is NaN in both
            to[h * TS + lane] = __uint_as_float(max(pend_k[h] << 23 | (pend_k[h] + 1) >> 8, 0x400000u));
            to[(HEADS + h) * TS + lane] = pend_v[h] == 255u ? __int_as_float(0x7fffffff) : __uint_as_float(0x4b000000u | pend_v[h]) - 8388735.f;
          }
        }
#pragma unroll
        for (int h = 0; h < HEADS; ++h) {
          pend_k[h] = pend_v[h] = 127u;                                         // tokens that are not there: finite, whatever lies there
          if (scaled) { pend_k[h] = ks[scale_at + h * p.c.ks_group]; pend_v[h] = vs[scale_at_v + h * p.c.vs_group]; }
        }
      }
    };

#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float up = 1.f, f = p.a.scale * LOG2E;
      if constexpr (E8) {
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int w = 0; w < 2; ++w) top = max(top, max(qb[c][k][w] << 16 & 0x7fffffffu, qb[c][k][w] & 0x7fff0000u));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        if (top != 0 && top < 0x7f800000u) {                                    // the largest becomes 2^13 … 2^14
          const int by = min(13 - (static_cast<int>(top >> 23) - 127), 126);
          up = __uint_as_float(static_cast<uint32_t>(127 + by) << 23);
          f *= __uint_as_float(static_cast<uint32_t>(127 - by) << 23);
        }
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const uint32_t u = qb[c][k][w];
            qb[c][k][w] = pa_pack<1>(__uint_as_float(u << 16) * up, __uint_as_float(u & 0xffff0000u) * up);
          }
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) factor[c][k] = __shfl_sync(0xffffffffu, f, 4 * (2 * cq + k));
    }
    int kmin[NC][2], kmax[NC][2];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        int row, branch;
        column(c * 8 + 2 * cq + k, row, branch);
        const int t = p.a.T == 1 ? 0 : row / p.per;
        const int64_t pos = sp.pos0 + t;
        kmax[c][k] = row < p.rows && t <= sp.t1 ? static_cast<int>(max(int64_t(-1), min(pos, int64_t(0x7fffffff)))) : -1;
        kmin[c][k] = p.a.window >= 0 ? static_cast<int>(max(int64_t(0), pos - p.a.window)) : 0;
      }
    // a step from all_lo to all_hi is seen by every row that is there
    const int64_t all_hi = sp.pos0 + sp.t0, all_lo = p.a.window >= 0 ? sp.pos0 + sp.t1 - p.a.window : 0;
    const int kh = PAIRS ? cq >> 1 : 0;                                         // key head of this thread's columns

    float acc[NC][KS][4], m[NC][2], l[NC][2], mv[NC][2][2];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[c][i][k] = 0.f;
#pragma unroll
      for (int k = 0; k < 2; ++k) { m[c][k] = mv[c][k][0] = mv[c][k][1] = -INFINITY; l[c][k] = 0.f; }
    }

#pragma unroll 1
    for (int step = -S::STAGES; step < steps; ++step) {                         // loads run STAGES steps ahead; one loop, so that they are in the code once
      if (step >= 0) {
      asm volatile("cp.async.wait_group %0;" ::"n"(S::STAGES - 1) : "memory");
      __syncwarp();
      const int stage = step % S::STAGES;
      const uint8_t* const st = ring + stage * S::STAGE;
      const uint32_t kt_u = ring_u + stage * S::STAGE + own_k, vt_u = ring_u + stage * S::STAGE + S::TILE + own_v;
      const uint8_t* const ex = extra + stage * S::EXTRA;
      const uint32_t live = *reinterpret_cast<const uint32_t*>(ex + S::SCALES);
      const int j0 = j_base + step * S::CHUNK;
      if (live != 0) {
        // ---- scores: x[c][mt][k] of token mt · 16 + gq (k < 2) or + 8, column 2 cq + (k & 1)
        float x[NC][MT][4];
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int k = 0; k < 4; ++k) x[c][mt][k] = 0.f;
#pragma unroll
        for (int ks = 0; ks < (E8 ? KS / 2 : KS); ++ks)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            uint32_t r[4];
            pa_ldsm<false>(r, (kt_u ^ (ks << 5)) + mt * 16 * S::ROW);
            if constexpr (E8) {                                                 // 16 bytes are a whole step of the product; q is laid out alike
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                uint32_t a0, a1, a2, a3;
                pa_halves(r[2 * h], a0, a2);
                pa_halves(r[2 * h + 1], a1, a3);
#pragma unroll
                for (int c = 0; c < NC; ++c) pa_mma<ES>(x[c][mt], a0, a1, a2, a3, qb[c][2 * ks + h][0], qb[c][2 * ks + h][1]);
              }
            } else {
#pragma unroll
              for (int c = 0; c < NC; ++c) pa_mma<ES>(x[c][mt], r[0], r[1], r[2], r[3], qb[c][ks][0], qb[c][ks][1]);
            }
          }
        const bool masked = live != FULL || j0 + TS - 1 > all_hi || j0 < all_lo;
        const float* const scales = reinterpret_cast<const float*>(ex);
        float ev[NGX][MT][2];                                                   // exponents of the values' scales
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int t = mt * 16 + 8 * h + gq;
            float f = 1.f;
            if constexpr (E8) {
              f = scales[kh * TS + t];
#pragma unroll
              for (int g = 0; g < NG; ++g) ev[g][mt][h] = scales[(HEADS + g) * TS + t];
            }
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
              for (int k = 0; k < 2; ++k) x[c][mt][2 * h + k] *= E8 ? factor[c][k] * f : factor[c][k];
          }
        if (masked) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int t = mt * 16 + 8 * h + gq;
              const bool is = live >> t & 1u;
#pragma unroll
              for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int k = 0; k < 2; ++k)
                  if (!(is && j0 + t <= kmax[c][k] && j0 + t >= kmin[c][k])) x[c][mt][2 * h + k] = -INFINITY;
            }
        }
        // ---- running maxima: lanes compare their own values, and only where one is larger do they meet and the sums follow
        bool grew = false;
        float top[NC][2], tv[NC][2][NGX];
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            top[c][k] = m[c][k];
#pragma unroll
            for (int g = 0; g < NG; ++g) tv[c][k][g] = mv[c][k][g];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                top[c][k] = fmaxf(top[c][k], x[c][mt][2 * h + k]);
#pragma unroll
                for (int g = 0; g < NG; ++g) tv[c][k][g] = fmaxf(tv[c][k][g], x[c][mt][2 * h + k] + ev[g][mt][h]);
              }
            grew = grew || top[c][k] > m[c][k];
#pragma unroll
            for (int g = 0; g < NG; ++g) grew = grew || tv[c][k][g] > mv[c][k][g];
          }
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            float f[2][2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
#pragma unroll
              for (int o = 4; o < 32; o *= 2) {
                top[c][k] = fmaxf(top[c][k], __shfl_xor_sync(0xffffffffu, top[c][k], o));
#pragma unroll
                for (int g = 0; g < NG; ++g) tv[c][k][g] = fmaxf(tv[c][k][g], __shfl_xor_sync(0xffffffffu, tv[c][k][g], o));
              }
              f[k][0] = f[k][1] = pa_step(m[c][k], top[c][k]);
              l[c][k] *= f[k][0];
              m[c][k] = top[c][k];
#pragma unroll
              for (int g = 0; g < NG; ++g) { f[k][g] = pa_step(mv[c][k][g], tv[c][k][g]); mv[c][k][g] = tv[c][k][g]; }
              if (NG == 1) f[k][1] = f[k][0];
            }
#pragma unroll
            for (int i = 0; i < KS; ++i)
#pragma unroll
              for (int k = 0; k < 4; ++k) acc[c][i][k] *= f[k & 1][i >= KS / 2];
          }
        }
        bool unscaled = false;                                                  // a token that some rows may not see has no scale: −∞ + NaN is not −∞
        if (E8 && masked) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int g = 0; g < NG; ++g) unscaled = unscaled || ev[g][mt][h] != ev[g][mt][h];
          unscaled = __any_sync(0xffffffffu, unscaled);
        }
        // ---- weights, turned into right operands: 16 tokens at a time
        uint32_t hi[NC][NGX][MT][2], lo[NC][NGX][MT][2];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          float base[2], bv[2][NGX];                                            // where nothing is seen yet every x is −∞: its weight is 0
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            base[k] = m[c][k] == -INFINITY ? 0.f : m[c][k];
#pragma unroll
            for (int g = 0; g < NG; ++g) bv[k][g] = mv[c][k][g] == -INFINITY ? 14.f : 14.f - mv[c][k][g];
          }
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float y0 = x[c][mt][2 * h], y1 = x[c][mt][2 * h + 1], w0 = pa_ex2(y0 - base[0]), w1 = pa_ex2(y1 - base[1]);
              l[c][0] += w0; l[c][1] += w1;
              if constexpr (E8) {
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                  const float e = ev[g][mt][h];
                  float w2 = pa_ex2(y0 + e + bv[0][g]), w3 = pa_ex2(y1 + e + bv[1][g]);
                  if (unscaled) { w2 = y0 == -INFINITY ? 0.f : w2; w3 = y1 == -INFINITY ? 0.f : w3; }
                  const uint32_t u = pa_pack<1>(w2, w3);
                  hi[c][g][mt][h] = pa_turn(u);
                  lo[c][g][mt][h] = pa_turn(pa_rest<1>(w2, w3, u));
                }
              } else {
                const uint32_t u = pa_pack<2>(w0, w1);
                hi[c][0][mt][h] = pa_turn(u);
                lo[c][0][mt][h] = pa_turn(pa_rest<2>(w0, w1, u));
              }
            }
        }
        // ---- outputs.  A weight of zero times an infinity or NaN is NaN: where rows see different tokens and one of these is not finite, the tokens of
        // each new token's rows go into a product of their own, of which those rows alone are taken.
        bool odd = false;
        if (masked && sp.t1 > sp.t0) {
          const uint32_t* const words = reinterpret_cast<const uint32_t*>(st + S::TILE);
          for (int i = lane; i < S::TILE / 4; i += 32) {
            const uint32_t u = words[i];
            if (E8) odd = odd || (u & 0x7fu) == 0x7fu || (u >> 8 & 0x7fu) == 0x7fu || (u >> 16 & 0x7fu) == 0x7fu || (u >> 24 & 0x7fu) == 0x7fu;
            else odd = odd || (u & 0x7f80u) == 0x7f80u || (u & 0x7f800000u) == 0x7f800000u;
          }
          odd = __any_sync(0xffffffffu, odd);
        }
        auto out_mul = [&](float (&d)[4], int c, int i, int mt, const uint32_t (&a)[4]) {
          const int g = NG == 2 && i >= KS / 2 ? 1 : 0;
          pa_mma<ES>(d, a[0], a[1], a[2], a[3], hi[c][g][mt][0], hi[c][g][mt][1]);
          pa_mma<ES>(d, a[0], a[1], a[2], a[3], lo[c][g][mt][0], lo[c][g][mt][1]);
        };
        // left operands of the 16 or 32 columns of a matrix load: rows gq, gq + 8 are columns gq, gq + 8 (bf16) or 2 gq, 2 gq + 1 of 16 (e4m3)
        constexpr int NB = E8 ? 2 : 1;
        auto values = [&](int mt, int i, uint32_t (&a)[NB][4]) {
          uint32_t r[4];
          if constexpr (E8) {
            pa_ldsm<true>(r, (vt_u ^ (i << 5)) + mt * 16 * S::ROW);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              pa_halves(__byte_perm(r[2 * h], 0, 0x3120), a[h][0], a[h][1]);
              pa_halves(__byte_perm(r[2 * h + 1], 0, 0x3120), a[h][2], a[h][3]);
            }
          } else {
            pa_ldsm<true>(r, (vt_u ^ (i << 5)) + mt * 16 * S::ROW);
            a[0][0] = r[0]; a[0][1] = r[1]; a[0][2] = r[2]; a[0][3] = r[3];
          }
        };
        if (!odd) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < KS / NB; ++i) {
              uint32_t a[NB][4];
              values(mt, i, a);
#pragma unroll
              for (int h = 0; h < NB; ++h)
#pragma unroll
                for (int c = 0; c < NC; ++c) out_mul(acc[c][i * NB + h], c, i * NB + h, mt, a[h]);
            }
        } else {
          for (int t = sp.t0; t <= sp.t1; ++t) {
            const int64_t pos = sp.pos0 + t, back = p.a.window >= 0 ? pos - p.a.window : 0;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              uint32_t keep[2];
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int64_t j = j0 + mt * 16 + 8 * h + 2 * cq;
                keep[h] = (j >= back && j <= pos ? 0xffffu : 0u) | (j + 1 >= back && j + 1 <= pos ? 0xffff0000u : 0u);
              }
#pragma unroll
              for (int i = 0; i < KS / NB; ++i) {
                uint32_t a[NB][4];
                values(mt, i, a);
#pragma unroll
                for (int h = 0; h < NB; ++h) {
                  a[h][0] &= keep[0]; a[h][1] &= keep[0]; a[h][2] &= keep[1]; a[h][3] &= keep[1];
#pragma unroll
                  for (int c = 0; c < NC; ++c) {
                    float d[4] = {0.f, 0.f, 0.f, 0.f};
                    out_mul(d, c, i * NB + h, mt, a[h]);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                      int row, branch;
                      column(c * 8 + 2 * cq + (k & 1), row, branch);
                      if (row / p.per == t) acc[c][i * NB + h][k] += d[k];
                    }
                  }
                }
              }
            }
          }
        }
      }
      __syncwarp();
      }
      issue(step + S::STAGES);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    // ---- the warps' parts, through the memory of the ring
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int o = 4; o < 32; o *= 2) l[c][k] += __shfl_xor_sync(0xffffffffu, l[c][k], o);
    __syncthreads();
    float* const slab = reinterpret_cast<float*>(smem) + warp * S::COLS * S::LD;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int n = c * 8 + 2 * cq + k;
        if (gq == 0) { s_stat[warp][0][n] = m[c][k]; s_stat[warp][1][n] = l[c][k]; s_stat[warp][2][n] = mv[c][k][0]; s_stat[warp][3][n] = mv[c][k][1]; }
        float* const to = slab + n * S::LD;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          if constexpr (E8) *reinterpret_cast<float2*>(to + i * 16 + 2 * gq) = make_float2(acc[c][i][k], acc[c][i][k + 2]);
          else { to[i * 16 + gq] = acc[c][i][k]; to[i * 16 + gq + 8] = acc[c][i][k + 2]; }
        }
      }
    __syncthreads();
    const bool whole = !CLUSTER && c0 == 0 && c1 == chunks;
    float* const part = CLUSTER ? reinterpret_cast<float*>(smem + S::SLABS) : whole ? nullptr : p.parts + (static_cast<int64_t>(blockIdx.x) * 2 + (c0 == 0)) * S::PART;
    for (int r = warp; r < S::QROWS; r += S::WARPS) {
      float v[2][DT / 32], mm[2], ll[2], mmv[2][2];
#pragma unroll
      for (int br = 0; br < HEADS; ++br) {
        const int k = pa_column<PAIRS>(r, br);
        mm[br] = mmv[br][0] = mmv[br][1] = -INFINITY; ll[br] = 0.f;
#pragma unroll
        for (int w = 0; w < S::WARPS; ++w) {
          mm[br] = fmaxf(mm[br], s_stat[w][0][k]);
          mmv[br][0] = fmaxf(mmv[br][0], s_stat[w][2][k]);
          mmv[br][1] = fmaxf(mmv[br][1], s_stat[w][3][k]);
        }
#pragma unroll
        for (int i = 0; i < DT / 32; ++i) v[br][i] = 0.f;
#pragma unroll
        for (int w = 0; w < S::WARPS; ++w) {
          const float f = pa_step(s_stat[w][0][k], mm[br]);
          ll[br] += s_stat[w][1][k] * f;
          const float f0 = E8 ? pa_step(s_stat[w][2][k], mmv[br][0]) : f, f1 = NG == 2 ? pa_step(s_stat[w][3][k], mmv[br][1]) : f0;
#pragma unroll
          for (int i = 0; i < DT / 32; ++i)
            v[br][i] += reinterpret_cast<const float*>(smem)[(w * S::COLS + k) * S::LD + lane + 32 * i] * (i < DT / 64 ? f0 : f1);
        }
        if (!whole) {
#pragma unroll
          for (int i = 0; i < DT / 32; ++i) part[k * DT + lane + 32 * i] = v[br][i];
          if (lane < 4) part[S::COLS * DT + k * 4 + lane] = lane == 0 ? mm[br] : lane == 1 ? ll[br] : lane == 2 ? mmv[br][0] : mmv[br][1];
        }
      }
      if (whole && row0 + r < p.rows)
        pa_finish<ES, DT, PAIRS>(p, b, head, row0 + r, (row0 + r) / p.per <= sp.t1, v[0], v[1], mm, ll, mmv, lane);
    }
    if constexpr (CLUSTER) {
      pa_cluster_sync();                                                        // every CTA's part is in its shared memory
      for (int r = blockIdx.x % 8 + 8 * warp; r < S::QROWS && row0 + r < p.rows; r += 8 * S::WARPS) {
        float v[2][DT / 32], mm[2], ll[2], mmv[2][2];
#pragma unroll
        for (int br = 0; br < HEADS; ++br) {
          const int k = pa_column<PAIRS>(r, br);
          float st[8][4], x[8][DT / 32];
#pragma unroll
          for (int c = 0; c < 8; ++c) {
#pragma unroll
            for (int i = 0; i < 4; ++i) st[c][i] = i < 2 || E8 ? pa_remote(part + S::COLS * DT + k * 4 + i, c) : -INFINITY;
#pragma unroll
            for (int i = 0; i < DT / 32; ++i) x[c][i] = pa_remote(part + k * DT + lane + 32 * i, c);
          }
          mm[br] = mmv[br][0] = mmv[br][1] = -INFINITY; ll[br] = 0.f;
#pragma unroll
          for (int c = 0; c < 8; ++c) { mm[br] = fmaxf(mm[br], st[c][0]); mmv[br][0] = fmaxf(mmv[br][0], st[c][2]); mmv[br][1] = fmaxf(mmv[br][1], st[c][3]); }
#pragma unroll
          for (int i = 0; i < DT / 32; ++i) v[br][i] = 0.f;
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const float f = pa_step(st[c][0], mm[br]), f0 = E8 ? pa_step(st[c][2], mmv[br][0]) : f, f1 = NG == 2 ? pa_step(st[c][3], mmv[br][1]) : f0;
            ll[br] += st[c][1] * f;
#pragma unroll
            for (int i = 0; i < DT / 32; ++i) v[br][i] += x[c][i] * (i < DT / 64 ? f0 : f1);
          }
        }
        pa_finish<ES, DT, PAIRS>(p, b, head, row0 + r, (row0 + r) / p.per <= sp.t1, v[0], v[1], mm, ll, mmv, lane);
      }
      pa_cluster_sync();                                                        // nobody leaves while another reads
      return;
    }
    __syncthreads();                                                            // the ring is used again
    if (GEN)                                                                    // and its unused columns are zero again
      for (int i = threadIdx.x; i < S::SLABS / 16; i += S::WARPS * 32) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
    if (GEN) __syncthreads();
    at += c1 - c0;
  }
}

// The parts of items that lie in several CTAs.  WPR warps share a row, each takes every WPR-th part with all of its loads in flight; a CTA has the rows of
// 16 / WPR (at most 8) neighbours of (item, row).  Few items have many parts each and want warps, many items have few parts and want to be over in
// one wave: 16, 4 or 1, whichever fits the device at once (256 items of 2 to 3 parts: 6 us with 1, 20 with 16; 4 items of 103 parts: 15 with 4, 6 with 16).
// Loads in turn are what such a kernel waits for: factors of all parts first and then a thread per column took 12 us instead of 6.
template <int ES, int DT, bool PAIRS, int NC, int WPR>
__global__ void __launch_bounds__(512 / (WPR == 1 ? 2 : 1)) paged_join_kernel(const PaArgs p) {
  using S = PaShape<ES, DT, PAIRS, NC>;
  constexpr int RPB = WPR == 1 ? 8 : 16 / WPR;
  constexpr int N = DT / 32, BR = PAIRS ? 2 : 1, AHEAD = DT == 256 ? 4 : 8;
  constexpr bool E8 = ES == 1;
  __shared__ float s_sum[RPB][WPR][BR][WPR == 1 ? 1 : DT];
  __shared__ float4 s_stat[RPB][WPR][BR];
  const int warp = threadIdx.x / 32 % WPR, slot = threadIdx.x / 32 / WPR, lane = threadIdx.x & 31;
  const int64_t which = static_cast<int64_t>(blockIdx.x) * RPB + slot;
  const int item = static_cast<int>(which / S::QROWS), r = static_cast<int>(which % S::QROWS);
  const int e = item / p.heads, head = item % p.heads;
  if (e >= p.nb * p.nrt) return;
  const int row0 = (p.rt0 + e % p.nrt) * S::QROWS, b = p.b0 + e / p.nrt;
  const PaSpan sp = pa_span<S::QROWS>(p, e);                                    // nothing of the first kernel is needed for it
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (row0 + r >= p.rows) return;
  const int entries = p.nb * p.nrt;
  const uint32_t before = p.prefix[e], chunks = p.prefix[e + 1] - before;
  const uint32_t all = static_cast<uint32_t>(p.prefix[entries]) * p.heads, ctas = min(all, static_cast<uint32_t>(p.ncta));
  const uint32_t from = before * p.heads + head * chunks;
  const int first = pa_owner(from, all, ctas), last = pa_owner(from + chunks - 1, all, ctas);
  if (first == last) return;                                                    // one CTA had it all
  const int n = last - first + 1;
  float m[2], l[2], mv[2][2], v[2][N];
#pragma unroll
  for (int br = 0; br < BR; ++br) {
    const int k = pa_column<PAIRS>(r, br);
    m[br] = mv[br][0] = mv[br][1] = -INFINITY; l[br] = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) v[br][j] = 0.f;
    for (int i0 = warp; i0 < n; i0 += WPR * AHEAD) {
      float4 st[AHEAD];
      float x[AHEAD][N];
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) {
        const int i = i0 + a * WPR;
        const float* src = p.parts + ((static_cast<int64_t>(first) + i) * 2 + (i == 0)) * S::PART;
        st[a] = i < n ? *reinterpret_cast<const float4*>(src + S::COLS * DT + k * 4) : make_float4(-INFINITY, 0.f, -INFINITY, -INFINITY);
#pragma unroll
        for (int j = 0; j < N; ++j) x[a][j] = i < n ? src[k * DT + lane + 32 * j] : 0.f;
      }
      float top = m[br], t0 = mv[br][0], t1 = mv[br][1];
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) { top = fmaxf(top, st[a].x); t0 = fmaxf(t0, st[a].z); t1 = fmaxf(t1, st[a].w); }
      const float f = pa_step(m[br], top), f0 = E8 ? pa_step(mv[br][0], t0) : f, f1 = S::NG == 2 ? pa_step(mv[br][1], t1) : f0;
      l[br] *= f;
#pragma unroll
      for (int j = 0; j < N; ++j) v[br][j] *= j < N / 2 ? f0 : f1;
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) {
        const float g = pa_step(st[a].x, top), g0 = E8 ? pa_step(st[a].z, t0) : g, g1 = S::NG == 2 ? pa_step(st[a].w, t1) : g0;
        l[br] += st[a].y * g;
#pragma unroll
        for (int j = 0; j < N; ++j) v[br][j] += x[a][j] * (j < N / 2 ? g0 : g1);
      }
      m[br] = top; mv[br][0] = t0; mv[br][1] = t1;
    }
  }
  if constexpr (WPR > 1) {
    // the warps of a row (others may have left): common maxima, sums scaled to them, then columns added up by as many threads as there are
    auto together = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(slot + 1), "n"(WPR * 32) : "memory"); };
#pragma unroll
    for (int br = 0; br < BR; ++br) if (lane == 0) s_stat[slot][warp][br] = make_float4(m[br], l[br], mv[br][0], mv[br][1]);
    together();
#pragma unroll
    for (int br = 0; br < BR; ++br) {
      const float4 st = lane < WPR ? s_stat[slot][lane][br] : make_float4(-INFINITY, 0.f, -INFINITY, -INFINITY);
      float top = st.x, t0 = st.z, t1 = st.w;
#pragma unroll
      for (int o = 16; o; o >>= 1) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (E8) { t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, o)); t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, o)); }
      }
      float sum = st.y * pa_step(st.x, top);
#pragma unroll
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      const float f = pa_step(m[br], top), f0 = E8 ? pa_step(mv[br][0], t0) : f, f1 = S::NG == 2 ? pa_step(mv[br][1], t1) : f0;
#pragma unroll
      for (int j = 0; j < N; ++j) s_sum[slot][warp][br][lane + 32 * j] = v[br][j] * (j < N / 2 ? f0 : f1);
      m[br] = top; l[br] = sum; mv[br][0] = t0; mv[br][1] = t1;
    }
    together();
#pragma unroll
    for (int i = warp * 32 + lane; i < BR * DT; i += WPR * 32) {
      float x = 0.f;
#pragma unroll
      for (int w = 0; w < WPR; ++w) x += s_sum[slot][w][i / DT][i % DT];
      s_sum[slot][0][i / DT][i % DT] = x;
    }
    together();
    if (warp != 0) return;
#pragma unroll
    for (int br = 0; br < BR; ++br)
#pragma unroll
      for (int j = 0; j < N; ++j) v[br][j] = s_sum[slot][0][br][lane + 32 * j];
  }
  pa_finish<ES, DT, PAIRS>(p, b, head, row0 + r, (row0 + r) / p.per <= sp.t1, v[0], v[1], m, l, mv, lane);
}

template <int ES, int DT, bool PAIRS, int NC, bool GEN, bool CLUSTER>
static int pa_main(const PaArgs& p, int ctas, cudaStream_t st) {
  using S = PaShape<ES, DT, PAIRS, NC>;
  auto kernel = paged_attention_kernel<ES, DT, PAIRS, NC, GEN, CLUSTER>;
  static std::atomic<uint64_t> ready{0};                                        // devices (of the first 64) on which the kernel has its shared memory
  int device = 0;
  if (const cudaError_t e = cudaGetDevice(&device); e != cudaSuccess) return static_cast<int>(e);
  const uint64_t bit = device < 64 ? uint64_t(1) << device : 0;
  if (!(ready.load(std::memory_order_acquire) & bit)) {
    if (const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM); e != cudaSuccess) return static_cast<int>(e);
    ready.fetch_or(bit, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(S::WARPS * 32);
  cfg.dynamicSmemBytes = S::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 8; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CLUSTER ? 1 : 0;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kernel, p));
}
template <int ES, int DT, bool PAIRS, int NC, bool GEN>
static int pa_launch(const PaArgs& p, bool cluster, int num_sms, cudaStream_t st) {
  using S = PaShape<ES, DT, PAIRS, NC>;
  if (cluster) return pa_main<ES, DT, PAIRS, NC, GEN, true>(p, p.nb * p.nrt * p.heads * 8, st);
  if (const int rc = pa_main<ES, DT, PAIRS, NC, GEN, false>(p, p.ncta, st)) return rc;
  if (p.prefix == nullptr) return 0;                                            // items of one chunk each: nothing to join
  cudaLaunchConfig_t cfg = {};
  const int64_t rows = static_cast<int64_t>(p.nb) * p.nrt * p.heads * S::QROWS, room = static_cast<int64_t>(num_sms) * 32;      // warps of the device, with 64 registers
  const int wpr = rows * 16 <= room ? 16 : rows * 4 <= room ? 4 : 1, rpb = wpr == 1 ? 8 : 16 / wpr;
  cfg.gridDim = dim3(static_cast<unsigned>((rows + rpb - 1) / rpb));
  cfg.blockDim = dim3(wpr * rpb * 32);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  auto join = wpr == 16 ? paged_join_kernel<ES, DT, PAIRS, NC, 16> : wpr == 4 ? paged_join_kernel<ES, DT, PAIRS, NC, 4> : paged_join_kernel<ES, DT, PAIRS, NC, 1>;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, join, p));
}

// A launch of the sequences and tiles that p names; with `need` only the bytes of its workspace and its CTAs are worked out.
int pa_run_bf16(PaArgs& p, int dt, bool pairs, int nc, bool gen, int span, int num_sms, void* ws, int64_t* need, cudaStream_t st);
int pa_run_e4m3(PaArgs& p, int dt, bool pairs, int nc, bool gen, int span, int num_sms, void* ws, int64_t* need, cudaStream_t st);

template <int ES, int DT, bool PAIRS, int NC>
static int pa_prepare(PaArgs& p, bool gen, int span, int num_sms, void* ws, int64_t* need, cudaStream_t st) {
  using S = PaShape<ES, DT, PAIRS, NC>;
  const int max_chunks = span <= S::CHUNK ? 1 : (span + S::CHUNK - 1) / S::CHUNK;
  // As many CTAs as run at once, each with an equal share; twice as many where a share is long beside the fixed costs of a CTA, so that SMs that are
  // nearer to memory take more of them: bf16, 64 sequences up to 8192, 97 -> 98 us with the cache in the L2, 119 -> 113 without; 32 in pairs 139 -> 135;
  // e4m3, whose warps compute half of the time, 47 -> 51.
  const int64_t work = static_cast<int64_t>(p.nb) * p.nrt * p.heads * max_chunks, full = static_cast<int64_t>(num_sms) * pa_resident<ES, DT, PAIRS, NC>();
  const int64_t most = ES == 2 && work >= 48 * full ? 2 * full : full;
  p.ncta = static_cast<int>(work < most ? work : most);
  // Few items of a few chunks: clusters of eight CTAs, one launch and no second kernel.  A CTA then has an eighth of an item instead of its share of all
  // chunks, which may be three (bf16, up to 128 values a row: four and a half) chunks more before it costs what the second kernel does; clusters leave places of an SM unused, hence four fifths.
  // One sequence of 1000 tokens, 4 key heads of 128: 10.3 -> 8.3 us, 8 of 2500: 17.2 -> 12.3, 8 of 5000 in e4m3: 22.6 -> 16.4; on the other side of the
  // rule 13 of 2500: 18.4 -> 22.5, one of 5000 in e4m3: 12.3 -> 14.4.  The chunks are those of the table, since lengths lie on the device: in a table with room for
  // 8192 tokens the sequence of 1000 takes 10.3 us, 8 of 1000 16.4 instead of 8.4, 8 of 2500 16.5 instead of 12.4.
  const int64_t items = static_cast<int64_t>(p.nb) * p.nrt * p.heads;
  const bool cluster = max_chunks > 1 && max_chunks <= 64 && 10 * items <= full && max_chunks * (full - 8 * items) <= (ES == 2 && DT <= 128 ? 36 : 24) * full;
  const int64_t bytes = max_chunks > 1 && !cluster ? static_cast<int64_t>(p.ncta) * 2 * S::PART * 4 + (PA_ENTRIES + 4) * 4 : 0;
  if (need != nullptr) { *need = bytes; return 0; }
  p.parts = static_cast<float*>(ws);
  p.prefix = bytes > 0 ? reinterpret_cast<int*>(p.parts + static_cast<int64_t>(p.ncta) * 2 * S::PART) : nullptr;
  return gen ? pa_launch<ES, DT, PAIRS, NC, true>(p, cluster, num_sms, st) : pa_launch<ES, DT, PAIRS, NC, false>(p, cluster, num_sms, st);
}
template <int ES>
static int pa_run(PaArgs& p, int dt, bool pairs, int nc, bool gen, int span, int num_sms, void* ws, int64_t* need, cudaStream_t st) {
  auto go = [&](auto dtc, auto pairsc) {
    constexpr int DT = decltype(dtc)::value;
    constexpr bool PAIRS = decltype(pairsc)::value;
    return nc == 1 ? pa_prepare<ES, DT, PAIRS, 1>(p, gen, span, num_sms, ws, need, st) : pa_prepare<ES, DT, PAIRS, 2>(p, gen, span, num_sms, ws, need, st);
  };
  using D64 = std::integral_constant<int, 64>;
  using D128 = std::integral_constant<int, 128>;
  using D256 = std::integral_constant<int, 256>;
  if (pairs) return dt == 128 ? go(D128{}, std::true_type{}) : go(D256{}, std::true_type{});
  return dt == 64 ? go(D64{}, std::false_type{}) : dt == 128 ? go(D128{}, std::false_type{}) : go(D256{}, std::false_type{});
}

}  // namespace b200
