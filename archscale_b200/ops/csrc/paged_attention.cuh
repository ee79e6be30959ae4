// Attention of a few new tokens over a paged key-value cache (layout in paged.cuh), keys and values read once for all query rows of a key head.
//
// Mathematics.  One pass over the keys with a running maximum and sum (base 2, 32 bits):  x_j = log₂e · scale · q·k_j,  p_j = 2^(x_j − m),
// o = Σ p_j v_j / Σ p_j.  Parts of a sequence are joined by  m = max m_i,  l = Σ l_i 2^(m_i − m),  o = Σ o_i 2^(m_i − m).
// In e4m3 a key's power of two multiplies its score; a value's, 2^e_j, goes into the weight, p'_j = 2^(x_j + e_j − m' + 14), whose maximum m' is kept
// beside m: no value is too small or large beside another, whatever their scales.
//
// Rows.  The query rows of a key head (its H/G heads times T tokens) are the 16 rows of an MMA m16n8k16, its columns keys (scores) or values (outputs):
//   ROWS8    up to 8 rows: the weights p enter the second product as two 16-bit halves, hi in rows 0-7 and lo = p − hi in rows 8-15 of one MMA
//   ROWS16   up to 16: two MMAs, for hi and lo
//   PAIRS    differential attention: 8 rows of branch 1 as [q1 | 0], the same 8 of branch 2 as [0 | q2], keys [k1 | k2], values [v1 | v2]: one product
//            each for both branches, and a1 − λ a2 is in one thread
// The halves make p as good as 2⁻¹⁷ (bf16; e4m3 runs in fp16: 2⁻²²), which costs nothing where the tensor cores wait for memory.  q is exact:
// bf16 as it is, for fp16 times a power of two of its row.
//
// What bounds it: memory.  16 rows are 32 operations a byte at most, and tcgen05 would want 128 rows, keys and P written back through shared memory; so the
// keys feed mma.sync from shared memory (4 warps per scheduler would keep up with 1.5 times the bandwidth).  Each warp is on its own: it
// loads its tokens with cp.async into its own ring of three stages (16 to 32 tokens, 8 KB), and no barrier joins warps before the
// end of a work item.  Pages are looked up one step ahead, so that their latency is not in the chain.
//
// Work.  Lengths are known on the device only.  An item is (sequence, tile of rows, key head); its keys are chunks of 4 warps' steps.  Every CTA adds
// up the chunks of all items from the lengths and takes an equal, contiguous share of them, so that one long sequence or many short ones fill the
// device alike.  Items that lie in one CTA are finished there; the parts of the others meet in a second kernel (joined in the order of the keys: results
// do not depend on scheduling), which the first one starts early and which needs no counters, so that nothing has to be zero beforehand.
#pragma once
#include <cuda_fp16.h>

#include "paged.cuh"

namespace b200 {

enum { PA_ROWS8 = 0, PA_ROWS16 = 1, PA_PAIRS = 2 };
constexpr int PA_WARPS = 4;
constexpr int PA_STAGES = 3;
constexpr int PA_ENTRIES = 1024;           // (sequence, tile of rows) of one launch

struct PaArgs {
  PagedView c;
  b200_paged_query a;
  int b0, nb, rt0, nrt;                    // sequences and tiles of rows of this launch
  int rows, per;                           // rows of a key head, and of one token among them
  int heads;                               // key heads, or pairs of them
  int ncta, piece, q_words;                // bytes of a copy where rows are not whole 16-byte pieces; queries start on 4-byte boundaries
  int64_t page_b, group_b, slot_b;         // strides in bytes, of keys as of values
  float* parts;                            // [ncta][2] parts of items
  int* prefix;                             // chunks before each entry, from CTA 0
};

// What a shape needs.
template <int ES, int DT, int MODE>
struct PaShape {
  static constexpr int ROW = DT * ES;                                          // bytes of a token in a stage
  static constexpr int TS = ES == 2 ? (DT == 64 ? 32 : 16) : (DT == 256 ? 16 : 32);   // tokens of a warp's step
  static constexpr int HEADS = MODE == PA_PAIRS ? 2 : 1;
  static constexpr int TILE = TS * ROW;
  static constexpr int SCALES = ES == 1 ? HEADS * TS * 8 : 0;                  // factors of keys, exponents of values
  static constexpr int STAGE = 2 * TILE + SCALES + 16;                         // and the mask of tokens
  static constexpr int RING = PA_WARPS * PA_STAGES * STAGE;
  static constexpr int QROWS = MODE == PA_ROWS16 ? 16 : 8;                     // query rows of a tile
  static constexpr int OROWS = MODE == PA_ROWS8 ? 8 : 16;                      // rows of the output product
  static constexpr int LD = DT + 8;                                            // floats between rows in shared memory: no bank twice
  static constexpr int SLABS = PA_WARPS * OROWS * LD * 4;
  static constexpr int SMEM = RING > SLABS ? RING : SLABS;
  static constexpr int CHUNK = PA_WARPS * TS;
  static constexpr int NG = ES == 1 ? HEADS : 0;                               // groups of columns with maxima of their own
  static constexpr int PART = OROWS * (DT + 4);                                // floats of a part: sums, then m, l, m' of each row
  static_assert(SMEM <= 227 * 1024 - 6144, "shared memory");
};

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
template <int ES, int DT, int MODE>
__device__ __forceinline__ void pa_finish(const PaArgs& p, int b, int head, int row, bool there, float (&v)[DT / 32], float (&v2)[DT / 32], const float (&m)[2],
                                          const float (&l)[2], const float (&mv)[2][2], int lane) {
  constexpr int N = DT / 32;
  const int D = p.c.dim, t = row / p.per, hh = row % p.per;
  if constexpr (MODE != PA_PAIRS) {
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
template <bool TRANS>
__device__ __forceinline__ void pa_ldsm(uint32_t (&r)[4], uint32_t addr) {
  if constexpr (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// two e4m3 values as fp16
__device__ __forceinline__ uint32_t pa_half2(uint32_t two) {
  uint32_t h;
  asm("{ .reg .b16 lo; cvt.u16.u32 lo, %1; cvt.rn.f16x2.e4m3x2 %0, lo; }" : "=r"(h) : "r"(two));
  return h;
}
// x, y as 16-bit hi halves, and what these leave
template <int ES>
__device__ __forceinline__ void pa_split(float x, float y, uint32_t& hi, uint32_t& lo) {
  if constexpr (ES == 2) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    const __nv_bfloat162 r = __floats2bfloat162_rn(x - __uint_as_float(hi << 16), y - __uint_as_float(hi & 0xffff0000u));
    lo = *reinterpret_cast<const uint32_t*>(&r);
  } else {
    const __half2 h = __floats2half2_rn(x, y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    const float2 f = __half22float2(h);
    const __half2 r = __floats2half2_rn(x - f.x, y - f.y);
    lo = *reinterpret_cast<const uint32_t*>(&r);
  }
}
template <int BYTES>
__device__ __forceinline__ void pa_copy(uint32_t dst, const void* src, bool live) {
  const int n = live ? BYTES : 0;
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(n) : "memory");
}
// byte of 16-byte piece `chunk` of token t in a tile: pieces of 8 tokens that a matrix load takes together lie in 8 different bank groups
template <int ROW>
__device__ __forceinline__ uint32_t pa_at(int t, int chunk) {
  return t * ROW + ((ROW >= 128 ? chunk ^ (t & 7) : chunk ^ ((t >> 1) & 3)) << 4);
}

// GEN: rows that are not whole 16-byte pieces, or shorter than DT
template <int ES, int DT, int MODE, bool GEN>
__global__ void __launch_bounds__(PA_WARPS * 32) paged_attention_kernel(const PaArgs p) {
  using S = PaShape<ES, DT, MODE>;
  constexpr bool E8 = ES == 1;
  constexpr int TS = S::TS, NT = TS / 8, KS = DT / 16, NV = DT / 8, NR = MODE == PA_ROWS8 ? 1 : 2, HEADS = S::HEADS, NG = S::NG;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int s_prefix[PA_ENTRIES + 1];
  __shared__ int s_scan[PA_WARPS];
  __shared__ float s_stat[PA_WARPS][4][16];                                     // m, l, m' of both groups
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, cq = lane & 3;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- chunks before every entry
  const int entries = p.nb * p.nrt;
  {
    const int each = (entries + PA_WARPS * 32 - 1) / (PA_WARPS * 32), from = threadIdx.x * each;
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
    if (threadIdx.x == 0) { int all = 0; for (int w = 0; w < PA_WARPS; ++w) all += s_scan[w]; s_prefix[entries] = all; }
  }
  if (GEN)                                                                      // columns past D stay zero
    for (int i = threadIdx.x; i < S::RING / 16; i += PA_WARPS * 32) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  if (blockIdx.x == 0 && p.prefix != nullptr)
    for (int i = threadIdx.x; i <= entries; i += PA_WARPS * 32) p.prefix[i] = s_prefix[i];

  const int64_t all = static_cast<int64_t>(s_prefix[entries]) * p.heads, share = (all + p.ncta - 1) / p.ncta;
  const int64_t end = min(all, (blockIdx.x + 1) * share);
  uint8_t* const ring = smem + warp * PA_STAGES * S::STAGE;
  const uint32_t ring_u = smem_u32(ring);
  constexpr float LOG2E = 1.4426950408889634f;

  for (int64_t at = blockIdx.x * share; at < end;) {
    // ---- the item
    int e = 0;
    for (int hi = entries; hi - e > 1;) { const int mid = (e + hi) >> 1; if (static_cast<int64_t>(s_prefix[mid]) * p.heads <= at) e = mid; else hi = mid; }
    const int chunks = s_prefix[e + 1] - s_prefix[e];
    const int64_t off = at - static_cast<int64_t>(s_prefix[e]) * p.heads;
    const int head = static_cast<int>(off / chunks), c0 = static_cast<int>(off % chunks), c1 = static_cast<int>(min(static_cast<int64_t>(chunks), c0 + end - at));
    const int b = p.b0 + e / p.nrt, row0 = (p.rt0 + e % p.nrt) * S::QROWS;
    const PaSpan sp = pa_span<S::QROWS>(p, e);
    const int j_base = sp.lo + c0 * S::CHUNK + warp * TS;                       // first token of this warp's step 0
    const int steps = c1 - c0;

    // ---- loads: lane i < TS knows token i of a step
    const uint8_t* const kb = static_cast<const uint8_t*>(p.c.k) + static_cast<int64_t>(head) * HEADS * p.group_b;
    const uint8_t* const vb = static_cast<const uint8_t*>(p.c.v) + static_cast<int64_t>(head) * HEADS * p.group_b;
    int next_page = -1;
    uint32_t pend_k[HEADS] = {}, pend_v[HEADS] = {};
    auto look = [&](int step) {                                                 // page of this lane's token, or -1
      const int64_t j = static_cast<int64_t>(j_base) + static_cast<int64_t>(step) * S::CHUNK + lane;
      next_page = step < steps && lane < TS && j < sp.hi ? paged_page(p.c, b, static_cast<int>(j) / p.c.page_size) : -1;
    };
    auto issue = [&](int step) {
      if (E8 && step > 0 && lane < TS) {                                        // scales asked for one step ago
        uint8_t* st = ring + ((step - 1) % PA_STAGES) * S::STAGE + 2 * S::TILE;
#pragma unroll
        for (int h = 0; h < HEADS; ++h) {
          reinterpret_cast<float*>(st)[h * TS + lane] = paged_pow2(pend_k[h]);
          reinterpret_cast<float*>(st)[(HEADS + h) * TS + lane] = pend_v[h] == 255u ? __int_as_float(0x7fffffff) : static_cast<float>(static_cast<int>(pend_v[h]) - 127);
        }
      }
      if (step < steps) {
        const int j = j_base + step * S::CHUNK + lane, page = next_page;
        const int slot = page >= 0 ? j % p.c.page_size : 0;
        const int64_t mine = page >= 0 ? page * p.page_b + slot * p.slot_b : -1;
        const uint32_t live = __ballot_sync(0xffffffffu, page >= 0);
        const uint32_t st = ring_u + (step % PA_STAGES) * S::STAGE;
        if (lane == 0) *reinterpret_cast<uint32_t*>(ring + (step % PA_STAGES) * S::STAGE + 2 * S::TILE + S::SCALES) = live;
        look(step + 1);
        if (live != 0) {
          if (E8 && page >= 0) {
#pragma unroll
            for (int h = 0; h < HEADS; ++h) {
              pend_k[h] = p.c.ks[page * p.c.ks_page + (head * HEADS + h) * p.c.ks_group + slot * p.c.ks_slot];
              pend_v[h] = p.c.vs[page * p.c.vs_page + (head * HEADS + h) * p.c.vs_group + slot * p.c.vs_slot];
            }
          }
          if constexpr (!GEN) {
            constexpr int PPR = S::ROW / 16;
#pragma unroll
            for (int i = 0; i < TS * PPR / 32; ++i) {
              const int idx = i * 32 + lane, t = idx / PPR, pc = idx % PPR;
              const int64_t o = __shfl_sync(0xffffffffu, mine, t);
              const int64_t from = o < 0 ? 0 : o + (HEADS == 2 && pc >= PPR / 2 ? p.group_b + (pc - PPR / 2) * 16 : pc * 16);
              const uint32_t to = st + pa_at<S::ROW>(t, pc);
              pa_copy<16>(to, kb + from, o >= 0);
              pa_copy<16>(to + S::TILE, vb + from, o >= 0);
            }
          } else {
            const int ppr = p.c.dim * ES / p.piece;
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
    };
    look(0);
#pragma unroll
    for (int i = 0; i < PA_STAGES - 1; ++i) issue(i);

    // ---- rows of this thread: gq and, except with 8 rows, gq + 8 of the product
    int row[NR], kmin[NR], kmax[NR];
    float factor[NR];
    uint32_t qa[KS][MODE == PA_ROWS16 ? 4 : 2];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      row[i] = row0 + gq + (MODE == PA_ROWS16 ? 8 * i : 0);
      const int t = row[i] / p.per;
      const bool there = row[i] < p.rows && t <= sp.t1;
      const int64_t pos = sp.pos0 + t;
      kmax[i] = there ? static_cast<int>(max(int64_t(-1), min(pos, int64_t(0x7fffffff)))) : -1;
      kmin[i] = p.a.window >= 0 ? static_cast<int>(max(int64_t(0), pos - p.a.window)) : 0;
      const int h = MODE == PA_PAIRS ? 2 * (head * p.per + row[i] % p.per) + i : head * p.per + row[i] % p.per;
      const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(p.a.q) + b * p.a.q_batch + t * p.a.q_token + h * p.a.q_head;
      auto two = [&](int d) -> uint32_t {                                       // values d, d + 1 (d even; so is D)
        if (!there || d >= p.c.dim) return 0u;
        if (p.q_words) return *reinterpret_cast<const uint32_t*>(src + d);
        return static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(src + d)) | static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(src + d + 1)) << 16;
      };
      constexpr int MINE = MODE == PA_PAIRS ? KS / 2 : KS;                      // steps of the product in which the row is not zero
      factor[i] = p.a.scale * LOG2E;
      float up = 1.f;
      if constexpr (E8) {
        uint32_t top = 0;
#pragma unroll
        for (int ks = 0; ks < MINE; ++ks)
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const uint32_t u = two(16 * ks + 4 * cq + 2 * w);
            top = max(top, max(u << 16 & 0x7fffffffu, u & 0x7fff0000u));
          }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        if (top != 0 && top < 0x7f800000u) {                                    // the largest becomes 2^13 … 2^14
          const int k = min(13 - (static_cast<int>(top >> 23) - 127), 126);
          up = __uint_as_float(static_cast<uint32_t>(127 + k) << 23);
          factor[i] *= __uint_as_float(static_cast<uint32_t>(127 - k) << 23);
        }
      }
#pragma unroll
      for (int ks = 0; ks < MINE; ++ks)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          uint32_t u = two(E8 ? 16 * ks + 4 * cq + 2 * w : 16 * ks + 2 * cq + 8 * w);
          if constexpr (E8) {
            const __half2 hv = __floats2half2_rn(__uint_as_float(u << 16) * up, __uint_as_float(u & 0xffff0000u) * up);
            u = *reinterpret_cast<const uint32_t*>(&hv);
          }
          if constexpr (MODE == PA_ROWS16) qa[ks][2 * w + i] = u;
          else if constexpr (MODE == PA_PAIRS) qa[i * (KS / 2) + ks][w] = u;
          else qa[ks][w] = u;
        }
    }
    // a step from all_lo to all_hi is seen by every row that is there
    const int64_t all_hi = sp.pos0 + sp.t0, all_lo = p.a.window >= 0 ? sp.pos0 + sp.t1 - p.a.window : 0;

    float acc[NV][4], m[NR], l[NR], mv[NR][2];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[i][k] = 0.f;
#pragma unroll
    for (int i = 0; i < NR; ++i) { m[i] = mv[i][0] = mv[i][1] = -INFINITY; l[i] = 0.f; }

    for (int step = 0; step < steps; ++step) {
      asm volatile("cp.async.wait_group %0;" ::"n"(PA_STAGES - 2) : "memory");
      __syncwarp();
      const int stage = step % PA_STAGES;
      const uint8_t* const st = ring + stage * S::STAGE;
      const uint32_t kt_u = ring_u + stage * S::STAGE, vt_u = kt_u + S::TILE;
      const uint32_t live = *reinterpret_cast<const uint32_t*>(st + 2 * S::TILE + S::SCALES);
      const int j0 = j_base + step * S::CHUNK;
      if (live != 0) {
        // ---- scores
        float x[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int k = 0; k < 4; ++k) x[n][k] = 0.f;
#pragma unroll
        for (int ks = 0; ks < (E8 ? KS / 2 : KS); ++ks)
#pragma unroll
          for (int np = 0; np < NT / 2; ++np) {
            uint32_t r[4];
            pa_ldsm<false>(r, kt_u + pa_at<S::ROW>(np * 16 + ((lane >> 4) & 1) * 8 + (lane & 7), ks * 2 + ((lane >> 3) & 1)));
            auto mul = [&](int n, int k, uint32_t b0, uint32_t b1) {
              if constexpr (MODE == PA_ROWS16) pa_mma<ES>(x[n], qa[k][0], qa[k][1], qa[k][2], qa[k][3], b0, b1);
              else if constexpr (MODE == PA_PAIRS) {
                if (k < KS / 2) pa_mma<ES>(x[n], qa[k][0], 0u, qa[k][1], 0u, b0, b1);
                else pa_mma<ES>(x[n], 0u, qa[k][0], 0u, qa[k][1], b0, b1);
              } else pa_mma<ES>(x[n], qa[k][0], 0u, qa[k][1], 0u, b0, b1);
            };
            if constexpr (E8) {                                                 // 16 bytes are a whole step of the product; q is laid out alike
              mul(2 * np, 2 * ks, pa_half2(r[0]), pa_half2(r[0] >> 16));
              mul(2 * np, 2 * ks + 1, pa_half2(r[1]), pa_half2(r[1] >> 16));
              mul(2 * np + 1, 2 * ks, pa_half2(r[2]), pa_half2(r[2] >> 16));
              mul(2 * np + 1, 2 * ks + 1, pa_half2(r[3]), pa_half2(r[3] >> 16));
            } else {
              mul(2 * np, ks, r[0], r[1]);
              mul(2 * np + 1, ks, r[2], r[3]);
            }
          }
        const bool masked = live != (TS == 32 ? 0xffffffffu : (1u << (TS & 31)) - 1u) || j0 + TS - 1 > all_hi || j0 < all_lo;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int k = 0; k < 2 * NR; ++k) {
            const int i = k >> 1, t = n * 8 + 2 * cq + (k & 1);
            x[n][k] *= factor[i];
            if (E8) x[n][k] *= reinterpret_cast<const float*>(st + 2 * S::TILE)[(HEADS == 2 ? i : 0) * TS + t];
            if (masked && !((live >> t & 1u) && j0 + t <= kmax[i] && j0 + t >= kmin[i])) x[n][k] = -INFINITY;
          }
        // ---- running maxima; the sums follow where one grew
        float top[NR], tv[NR][2];
#pragma unroll
        for (int i = 0; i < NR; ++i) {
          top[i] = m[i]; tv[i][0] = mv[i][0]; tv[i][1] = mv[i][1];
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              top[i] = fmaxf(top[i], x[n][2 * i + k]);
#pragma unroll
              for (int g = 0; g < NG; ++g)
                tv[i][g] = fmaxf(tv[i][g], x[n][2 * i + k] + reinterpret_cast<const float*>(st + 2 * S::TILE)[(HEADS + g) * TS + n * 8 + 2 * cq + k]);
            }
#pragma unroll
          for (int o = 1; o < 4; o *= 2) {
            top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
#pragma unroll
            for (int g = 0; g < NG; ++g) tv[i][g] = fmaxf(tv[i][g], __shfl_xor_sync(0xffffffffu, tv[i][g], o));
          }
        }
        bool grew = false;
#pragma unroll
        for (int i = 0; i < NR; ++i) grew = grew || top[i] > m[i] || (NG > 0 && tv[i][0] > mv[i][0]) || (NG > 1 && tv[i][1] > mv[i][1]);
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
          for (int i = 0; i < NR; ++i) {
            const float f = pa_step(m[i], top[i]);
            l[i] *= f;
            const float f0 = E8 ? pa_step(mv[i][0], tv[i][0]) : f, f1 = NG == 2 ? pa_step(mv[i][1], tv[i][1]) : f0;
#pragma unroll
            for (int n = 0; n < NV; ++n) {
              const float fn = n < NV / 2 ? f0 : f1;
              if constexpr (MODE == PA_ROWS8) { acc[n][0] *= fn; acc[n][1] *= fn; acc[n][2] *= fn; acc[n][3] *= fn; }
              else { acc[n][2 * i] *= fn; acc[n][2 * i + 1] *= fn; }
            }
            m[i] = top[i]; mv[i][0] = tv[i][0]; mv[i][1] = tv[i][1];
          }
        }
        // ---- weights: 16 tokens at a time are the left operand of the second product
        uint32_t hi[HEADS][NT][NR], lo[HEADS][NT][NR];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < NR; ++i) {
            float w[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) { const float y = x[n][2 * i + k]; w[k] = pa_step(y, m[i]); l[i] += w[k]; }
            if constexpr (E8) {
#pragma unroll
              for (int g = 0; g < NG; ++g) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                  const float y = x[n][2 * i + k];
                  w[k] = y == -INFINITY ? 0.f : pa_ex2(y + reinterpret_cast<const float*>(st + 2 * S::TILE)[(HEADS + g) * TS + n * 8 + 2 * cq + k] - mv[i][g] + 14.f);
                }
                pa_split<ES>(w[0], w[1], hi[g][n][i], lo[g][n][i]);
              }
            } else {
              pa_split<ES>(w[0], w[1], hi[0][n][i], lo[0][n][i]);
              if (HEADS == 2) { hi[HEADS - 1][n][i] = hi[0][n][i]; lo[HEADS - 1][n][i] = lo[0][n][i]; }
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
        auto out_mul = [&](float (&d)[4], int n, int kt, uint32_t b0, uint32_t b1) {
          const int g = HEADS == 2 && n >= NV / 2 ? 1 : 0;
          if constexpr (MODE == PA_ROWS8) {
            pa_mma<ES>(d, hi[g][2 * kt][0], lo[g][2 * kt][0], hi[g][2 * kt + 1][0], lo[g][2 * kt + 1][0], b0, b1);
          } else {
            pa_mma<ES>(d, hi[g][2 * kt][0], hi[g][2 * kt][1], hi[g][2 * kt + 1][0], hi[g][2 * kt + 1][1], b0, b1);
            pa_mma<ES>(d, lo[g][2 * kt][0], lo[g][2 * kt][1], lo[g][2 * kt + 1][0], lo[g][2 * kt + 1][1], b0, b1);
          }
        };
        auto values = [&](int kt, int dp, uint32_t (&r)[4]) {
          pa_ldsm<true>(r, vt_u + pa_at<S::ROW>(kt * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), dp * 2 + (lane >> 4)));
        };
        // operands of the columns of `values`: NB tiles of 8 columns
        constexpr int NB = E8 ? 4 : 2;
        auto tiles = [&](const uint32_t (&r)[4], uint32_t (&b0)[NB], uint32_t (&b1)[NB]) {
          if constexpr (E8) {                                                   // even columns, odd columns of 16
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t u = __byte_perm(r[2 * h], 0, 0x3120), w = __byte_perm(r[2 * h + 1], 0, 0x3120);
              b0[2 * h] = pa_half2(u); b0[2 * h + 1] = pa_half2(u >> 16);
              b1[2 * h] = pa_half2(w); b1[2 * h + 1] = pa_half2(w >> 16);
            }
          } else { b0[0] = r[0]; b1[0] = r[1]; b0[1] = r[2]; b1[1] = r[3]; }
        };
        if (!odd) {
#pragma unroll
          for (int kt = 0; kt < TS / 16; ++kt)
#pragma unroll
            for (int dp = 0; dp < NV / NB; ++dp) {
              uint32_t r[4], b0[NB], b1[NB];
              values(kt, dp, r);
              tiles(r, b0, b1);
#pragma unroll
              for (int i = 0; i < NB; ++i) out_mul(acc[dp * NB + i], dp * NB + i, kt, b0[i], b1[i]);
            }
        } else {
          for (int t = sp.t0; t <= sp.t1; ++t) {
            const int64_t pos = sp.pos0 + t, back = p.a.window >= 0 ? pos - p.a.window : 0;
            const bool take0 = row[0] / p.per == t, take1 = row[NR - 1] / p.per == t;
#pragma unroll
            for (int kt = 0; kt < TS / 16; ++kt) {
              uint32_t keep[2];
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int64_t j = j0 + kt * 16 + 8 * h + 2 * cq;
                keep[h] = (j >= back && j <= pos ? 0xffffu : 0u) | (j + 1 >= back && j + 1 <= pos ? 0xffff0000u : 0u);
              }
#pragma unroll
              for (int dp = 0; dp < NV / NB; ++dp) {
                uint32_t r[4], b0[NB], b1[NB];
                values(kt, dp, r);
                tiles(r, b0, b1);
#pragma unroll
                for (int i = 0; i < NB; ++i) {
                  float d[4] = {0.f, 0.f, 0.f, 0.f};
                  out_mul(d, dp * NB + i, kt, b0[i] & keep[0], b1[i] & keep[1]);
                  if (take0) { acc[dp * NB + i][0] += d[0]; acc[dp * NB + i][1] += d[1]; }
                  if (take1) { acc[dp * NB + i][2] += d[2]; acc[dp * NB + i][3] += d[3]; }
                }
              }
            }
          }
        }
      }
      __syncwarp();
      issue(step + PA_STAGES - 1);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    // ---- the warps' parts, through the memory of the ring
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
      for (int o = 1; o < 4; o *= 2) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
    __syncthreads();
    float* const slab = reinterpret_cast<float*>(smem) + warp * S::OROWS * S::LD;
    if (cq == 0)
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        s_stat[warp][0][gq + 8 * i] = m[i]; s_stat[warp][1][gq + 8 * i] = l[i];
        s_stat[warp][2][gq + 8 * i] = mv[i][0]; s_stat[warp][3][gq + 8 * i] = mv[i][1];
      }
    if constexpr (MODE == PA_ROWS8) {
#pragma unroll
      for (int n = 0; n < NV; ++n) { acc[n][0] += acc[n][2]; acc[n][1] += acc[n][3]; }
    }
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      float* const to = slab + (gq + 8 * i) * S::LD;
      if constexpr (E8) {
#pragma unroll
        for (int n = 0; n < NV; n += 2)
          *reinterpret_cast<float4*>(to + n * 8 + 4 * cq) = make_float4(acc[n][2 * i], acc[n + 1][2 * i], acc[n][2 * i + 1], acc[n + 1][2 * i + 1]);
      } else {
#pragma unroll
        for (int n = 0; n < NV; ++n) *reinterpret_cast<float2*>(to + n * 8 + 2 * cq) = make_float2(acc[n][2 * i], acc[n][2 * i + 1]);
      }
    }
    __syncthreads();
    const bool whole = c0 == 0 && c1 == chunks;
    float* const part = whole ? nullptr : p.parts + (static_cast<int64_t>(blockIdx.x) * 2 + (c0 == 0)) * S::PART;
    for (int r = warp; r < S::QROWS; r += PA_WARPS) {
      float v[2][DT / 32], mm[2], ll[2], mmv[2][2];
#pragma unroll
      for (int br = 0; br < (MODE == PA_PAIRS ? 2 : 1); ++br) {
        const int k = r + 8 * br;
        mm[br] = mmv[br][0] = mmv[br][1] = -INFINITY; ll[br] = 0.f;
#pragma unroll
        for (int w = 0; w < PA_WARPS; ++w) {
          mm[br] = fmaxf(mm[br], s_stat[w][0][k]);
          mmv[br][0] = fmaxf(mmv[br][0], s_stat[w][2][k]);
          mmv[br][1] = fmaxf(mmv[br][1], s_stat[w][3][k]);
        }
#pragma unroll
        for (int i = 0; i < DT / 32; ++i) v[br][i] = 0.f;
#pragma unroll
        for (int w = 0; w < PA_WARPS; ++w) {
          const float f = pa_step(s_stat[w][0][k], mm[br]);
          ll[br] += s_stat[w][1][k] * f;
          const float f0 = E8 ? pa_step(s_stat[w][2][k], mmv[br][0]) : f, f1 = NG == 2 ? pa_step(s_stat[w][3][k], mmv[br][1]) : f0;
#pragma unroll
          for (int i = 0; i < DT / 32; ++i)
            v[br][i] += reinterpret_cast<const float*>(smem)[(w * S::OROWS + k) * S::LD + lane + 32 * i] * (i < DT / 64 ? f0 : f1);
        }
        if (!whole) {
#pragma unroll
          for (int i = 0; i < DT / 32; ++i) part[k * DT + lane + 32 * i] = v[br][i];
          if (lane < 4) part[S::OROWS * DT + k * 4 + lane] = lane == 0 ? mm[br] : lane == 1 ? ll[br] : lane == 2 ? mmv[br][0] : mmv[br][1];
        }
      }
      if (whole && row0 + r < p.rows)
        pa_finish<ES, DT, MODE>(p, b, head, row0 + r, (row0 + r) / p.per <= sp.t1, v[0], v[1], mm, ll, mmv, lane);
    }
    __syncthreads();                                                            // the ring is used again
    if (GEN)                                                                    // and its unused columns are zero again
      for (int i = threadIdx.x; i < S::SLABS / 16; i += PA_WARPS * 32) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
    if (GEN) __syncthreads();
    at += c1 - c0;
  }
}

// The parts of items that lie in several CTAs: one CTA per item and row.
template <int ES, int DT, int MODE>
__global__ void __launch_bounds__(PA_WARPS * 32) paged_join_kernel(const PaArgs p) {
  using S = PaShape<ES, DT, MODE>;
  constexpr int N = DT / 32, BR = MODE == PA_PAIRS ? 2 : 1;
  constexpr bool E8 = ES == 1;
  __shared__ float s_sum[PA_WARPS][BR][DT];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int e = blockIdx.x / p.heads, head = blockIdx.x % p.heads, r = blockIdx.y;
  const int row0 = (p.rt0 + e % p.nrt) * S::QROWS, b = p.b0 + e / p.nrt;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (row0 + r >= p.rows) return;
  const int entries = p.nb * p.nrt;
  const int64_t all = static_cast<int64_t>(p.prefix[entries]) * p.heads, share = (all + p.ncta - 1) / p.ncta;
  const int before = p.prefix[e], chunks = p.prefix[e + 1] - before;
  const int64_t from = static_cast<int64_t>(before) * p.heads + static_cast<int64_t>(head) * chunks;
  const int first = static_cast<int>(from / share), last = static_cast<int>((from + chunks - 1) / share);
  if (first == last) return;                                                    // one CTA had it all
  const int n = last - first + 1;
  auto part = [&](int i) { return p.parts + ((static_cast<int64_t>(first) + i) * 2 + (i == 0)) * S::PART; };
  float m[2], l[2], mv[2][2], v[2][N];
#pragma unroll
  for (int br = 0; br < BR; ++br) {
    const int k = r + 8 * br;
    m[br] = mv[br][0] = mv[br][1] = -INFINITY; l[br] = 0.f;
    for (int i = lane; i < n; i += 32) {
      const float4 s = *reinterpret_cast<const float4*>(part(i) + S::OROWS * DT + k * 4);
      m[br] = fmaxf(m[br], s.x); mv[br][0] = fmaxf(mv[br][0], s.z); mv[br][1] = fmaxf(mv[br][1], s.w);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      m[br] = fmaxf(m[br], __shfl_xor_sync(0xffffffffu, m[br], o));
      mv[br][0] = fmaxf(mv[br][0], __shfl_xor_sync(0xffffffffu, mv[br][0], o));
      mv[br][1] = fmaxf(mv[br][1], __shfl_xor_sync(0xffffffffu, mv[br][1], o));
    }
    for (int i = lane; i < n; i += 32) {
      const float4 s = *reinterpret_cast<const float4*>(part(i) + S::OROWS * DT + k * 4);
      l[br] += s.y * pa_step(s.x, m[br]);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) l[br] += __shfl_xor_sync(0xffffffffu, l[br], o);
    float sum[N];
#pragma unroll
    for (int j = 0; j < N; ++j) sum[j] = 0.f;
#pragma unroll 4
    for (int i = warp; i < n; i += PA_WARPS) {
      const float* src = part(i);
      const float4 s = *reinterpret_cast<const float4*>(src + S::OROWS * DT + k * 4);
      const float f = pa_step(s.x, m[br]), f0 = E8 ? pa_step(s.z, mv[br][0]) : f, f1 = S::NG == 2 ? pa_step(s.w, mv[br][1]) : f0;
#pragma unroll
      for (int j = 0; j < N; ++j) sum[j] += src[k * DT + lane + 32 * j] * (j < N / 2 ? f0 : f1);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) s_sum[warp][br][lane + 32 * j] = sum[j];
  }
  __syncthreads();
  if (warp != 0) return;
#pragma unroll
  for (int br = 0; br < BR; ++br)
#pragma unroll
    for (int j = 0; j < N; ++j) {
      v[br][j] = 0.f;
#pragma unroll
      for (int w = 0; w < PA_WARPS; ++w) v[br][j] += s_sum[w][br][lane + 32 * j];
    }
  const PaSpan sp = pa_span<S::QROWS>(p, e);
  pa_finish<ES, DT, MODE>(p, b, head, row0 + r, (row0 + r) / p.per <= sp.t1, v[0], v[1], m, l, mv, lane);
}

// CTAs that fit an SM beside one another, by shared memory
template <int ES, int DT, int MODE>
constexpr int pa_resident() {
  constexpr int one = PaShape<ES, DT, MODE>::SMEM + (PA_ENTRIES + 1) * 4 + 2048;      // its static part and what the system keeps
  return 228 * 1024 / one < 4 ? 228 * 1024 / one : 4;
}

template <int ES, int DT, int MODE, bool GEN>
static int pa_launch(PaArgs& p, int max_chunks, int num_sms, cudaStream_t st) {
  using S = PaShape<ES, DT, MODE>;
  auto kernel = paged_attention_kernel<ES, DT, MODE, GEN>;
  if (const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM); e != cudaSuccess) return static_cast<int>(e);
  kernel<<<p.ncta, PA_WARPS * 32, S::SMEM, st>>>(p);
  if (const cudaError_t e = cudaGetLastError(); e != cudaSuccess) return static_cast<int>(e);
  if (p.prefix == nullptr) return 0;                                            // items of one chunk each: nothing to join
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.nb * p.nrt * p.heads), S::QROWS);
  cfg.blockDim = dim3(PA_WARPS * 32);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, paged_join_kernel<ES, DT, MODE>, p));
}

// A launch of the sequences and tiles that p names; with `need` only the bytes of its workspace and its CTAs are worked out.
int pa_run_bf16(PaArgs& p, int dt, int mode, bool gen, int span, int num_sms, void* ws, int64_t* need, cudaStream_t st);
int pa_run_e4m3(PaArgs& p, int dt, int mode, bool gen, int span, int num_sms, void* ws, int64_t* need, cudaStream_t st);

template <int ES, int DT, int MODE>
static int pa_prepare(PaArgs& p, bool gen, int span, int num_sms, void* ws, int64_t* need, cudaStream_t st) {
  using S = PaShape<ES, DT, MODE>;
  const int max_chunks = span <= S::CHUNK ? 1 : (span + S::CHUNK - 1) / S::CHUNK;
  const int64_t work = static_cast<int64_t>(p.nb) * p.nrt * p.heads * max_chunks, full = static_cast<int64_t>(num_sms) * pa_resident<ES, DT, MODE>();
  p.ncta = static_cast<int>(work < full ? work : full);
  const int64_t bytes = max_chunks > 1 ? static_cast<int64_t>(p.ncta) * 2 * S::PART * 4 + (PA_ENTRIES + 4) * 4 : 0;
  if (need != nullptr) { *need = bytes; return 0; }
  p.parts = static_cast<float*>(ws);
  p.prefix = max_chunks > 1 ? reinterpret_cast<int*>(p.parts + static_cast<int64_t>(p.ncta) * 2 * S::PART) : nullptr;
  return gen ? pa_launch<ES, DT, MODE, true>(p, max_chunks, num_sms, st) : pa_launch<ES, DT, MODE, false>(p, max_chunks, num_sms, st);
}
template <int ES>
static int pa_run(PaArgs& p, int dt, int mode, bool gen, int span, int num_sms, void* ws, int64_t* need, cudaStream_t st) {
  if (mode == PA_PAIRS) {
    if (dt == 128) return pa_prepare<ES, 128, PA_PAIRS>(p, gen, span, num_sms, ws, need, st);
    return pa_prepare<ES, 256, PA_PAIRS>(p, gen, span, num_sms, ws, need, st);
  }
  if (mode == PA_ROWS8) {
    if (dt == 64) return pa_prepare<ES, 64, PA_ROWS8>(p, gen, span, num_sms, ws, need, st);
    if (dt == 128) return pa_prepare<ES, 128, PA_ROWS8>(p, gen, span, num_sms, ws, need, st);
    return pa_prepare<ES, 256, PA_ROWS8>(p, gen, span, num_sms, ws, need, st);
  }
  if (dt == 64) return pa_prepare<ES, 64, PA_ROWS16>(p, gen, span, num_sms, ws, need, st);
  if (dt == 128) return pa_prepare<ES, 128, PA_ROWS16>(p, gen, span, num_sms, ws, need, st);
  return pa_prepare<ES, 256, PA_ROWS16>(p, gen, span, num_sms, ws, need, st);
}

}  // namespace b200
