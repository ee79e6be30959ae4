// Quantisers of the 8-bit format with one fp32 scale per block of 128 (e4m3 elements), and the residual addition + RMSNorm that
// writes it.
//
// With a = max(max |x| over the block, 1e-30):  scale = a / 448,  u = 448 / a,  q = e4m3(x · u), all in fp32 with one rounding each (this
// file is built without --use_fast_math), e4m3 rounding to nearest even.  |x · u| ≤ 448 up to one rounding, which e4m3 takes back, so nothing
// saturates.  The floor of 1e-30 keeps u finite: an empty block gets zeros.  An infinity or NaN makes its block's scale infinite or
// NaN and its own element NaN, so that a product shows it (magnitudes are compared as integers, where NaN is the largest).
//
// Scales are stored block-major, [block of 128][row] with the rows padded to a multiple of 4: the GEMM fetches one block's scales of
// 128 neighbouring rows as 512 contiguous bytes.  Elements have rows of a multiple of 16 bytes (TMA).
#include <cuda_fp8.h>

#include "api.h"
#include "sm100.cuh"

namespace b200 {

constexpr float kE4m3Max = 448.f, kBlockFloor = 1e-30f;

__device__ __forceinline__ float block_amax(uint32_t bits) {                        // NaN stays NaN
  return __uint_as_float(max(bits, __float_as_uint(kBlockFloor)));
}
__device__ __forceinline__ float max_abs(float a, float b, float c) {               // NaN if one of them is
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) {
  const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const __nv_fp8x2_storage_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
}

// Two values at a time, each rounded as by itself.
__device__ __forceinline__ void scale8(float (&v)[8], float u) {
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const float2 t = mul_f32x2(make_float2(v[e], v[e + 1]), make_float2(u, u));
    v[e] = t.x; v[e + 1] = t.y;
  }
}
__device__ __forceinline__ void mul8(float (&v)[8], const float (&w)[8]) {
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const float2 t = mul_f32x2(make_float2(v[e], v[e + 1]), make_float2(w[e], w[e + 1]));
    v[e] = t.x; v[e + 1] = t.y;
  }
}
__device__ __forceinline__ uint2 pack_e4m3x8(const float (&v)[8]) {
  return make_uint2(pack_e4m3x4(v[0], v[1], v[2], v[3]), pack_e4m3x4(v[4], v[5], v[6], v[7]));
}

// Eight neighbouring values of a row, the first n of them inside it (the others are zero).
template <typename T> struct Raw8;
template <> struct Raw8<float> { float4 a, b; };
template <> struct Raw8<__nv_bfloat16> { uint4 a; };

// VEC: rows are whole 16-byte pieces, so that n is 8 or not positive: one or two predicated loads, which the compiler issues together
// (with a branch per vector for the general case in between, a tile of bf16 took 3.5 times as long).  Otherwise the row starts anywhere, and
// fp32 is loaded one value at a time; of bf16 the aligned 16-byte pieces that hold at least one of the values are loaded and shifted
// (30568 x 7981 in both orientations 266 µs instead of 317; fp32 that way 457 instead of 336).  Such a piece never leaves the 16-byte granule of
// memory that the value lies in.
template <bool VEC>
__device__ __forceinline__ void load_raw(const float* p, int n, Raw8<float>& r) {
  if (VEC) {
    r.a = r.b = make_float4(0.f, 0.f, 0.f, 0.f);
    if (n > 0) { r.a = *reinterpret_cast<const float4*>(p); r.b = *reinterpret_cast<const float4*>(p + 4); }
  } else {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : 0.f;
    r.a = make_float4(v[0], v[1], v[2], v[3]);
    r.b = make_float4(v[4], v[5], v[6], v[7]);
  }
}
template <bool VEC>
__device__ __forceinline__ void load_raw(const __nv_bfloat16* p, int n, Raw8<__nv_bfloat16>& r) {
  r.a = make_uint4(0u, 0u, 0u, 0u);
  if (VEC) {
    if (n > 0) r.a = *reinterpret_cast<const uint4*>(p);
  } else if (n > 0) {
    const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) & 15u;
    const uint4* base = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(p) - off);
    const uint4 c0 = base[0], c1 = static_cast<int>(off) + n * 2 > 16 ? base[1] : make_uint4(0u, 0u, 0u, 0u);
    const uint32_t w[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
    uint32_t t[6], u[5], o[4];                          // by two words, by one, by half of one
#pragma unroll
    for (int i = 0; i < 6; ++i) t[i] = (off & 8) ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < 5; ++i) u[i] = (off & 4) ? t[i + 1] : t[i];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = __funnelshift_r(u[i], u[i + 1], (off & 2) * 8);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = 2 * i + 1 < n ? o[i] : 2 * i < n ? o[i] & 0xffffu : 0u;
    r.a = make_uint4(o[0], o[1], o[2], o[3]);
  }
}
__device__ __forceinline__ void unpack8(const Raw8<float>& r, float (&v)[8]) {
  v[0] = r.a.x; v[1] = r.a.y; v[2] = r.a.z; v[3] = r.a.w; v[4] = r.b.x; v[5] = r.b.y; v[6] = r.b.z; v[7] = r.b.w;
}
__device__ __forceinline__ void unpack8(const Raw8<__nv_bfloat16>& r, float (&v)[8]) {
  const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
template <bool VEC, typename T>
__device__ __forceinline__ void load8(const T* p, int n, float (&v)[8]) {
  Raw8<T> r;
  load_raw<VEC>(p, n, r);
  unpack8(r, v);
}

struct Fp8TileParams {
  const void* x;
  int64_t ldx;
  int rows, cols, cb;           // cb: column blocks
  int vec;
  uint8_t* q; int64_t ldq;      // [rows][ldq]
  float* s; int64_t lds;        // [cb][lds] per row, or [row block][cb] per tile
  uint8_t* qt; int64_t ldqt;    // [cols][ldqt]
  float* st; int64_t ldst;      // [row block][ldst] per column
  const float* rstd;            // NORM: values are (x · rstd[row]) · w[col]
  const void* w; int w_f32;
};

enum : int { FP8_ROWS = 1, FP8_COLS = 2, FP8_TILE = 4 };

// Largest magnitudes of a thread's 8 × 8 values, as the bits of fp32 numbers: per row, per column, over all.  bf16 is compared two at a
// time as 16-bit integers (NaN is the largest there too).
__device__ __forceinline__ void row_max(const Raw8<float> (&r)[8], uint32_t (&m)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float4 a = r[i].a, b = r[i].b;
    m[i] = __float_as_uint(max_abs(max_abs(max_abs(a.x, a.y, a.z), a.w, b.x), b.y, max_abs(b.z, b.w, 0.f)));
  }
}
__device__ __forceinline__ void row_max(const Raw8<__nv_bfloat16> (&r)[8], uint32_t (&m)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t k = 0x7fff7fffu;
    const uint32_t t = __vmaxu2(__vmaxu2(r[i].a.x & k, r[i].a.y & k), __vmaxu2(r[i].a.z & k, r[i].a.w & k));
    m[i] = max(t & 0xffff0000u, t << 16);
  }
}
__device__ __forceinline__ void col_max(const Raw8<float> (&r)[8], uint32_t (&m)[8]) {
  float t[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) t[e] = 0.f;
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float4 a = r[i].a, b = r[i].b, c = r[i + 1].a, d = r[i + 1].b;
    t[0] = max_abs(t[0], a.x, c.x); t[1] = max_abs(t[1], a.y, c.y); t[2] = max_abs(t[2], a.z, c.z); t[3] = max_abs(t[3], a.w, c.w);
    t[4] = max_abs(t[4], b.x, d.x); t[5] = max_abs(t[5], b.y, d.y); t[6] = max_abs(t[6], b.z, d.z); t[7] = max_abs(t[7], b.w, d.w);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) m[e] = __float_as_uint(t[e]);
}
__device__ __forceinline__ void col_max(const Raw8<__nv_bfloat16> (&r)[8], uint32_t (&m)[8]) {
  uint32_t t[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t w[4] = {r[i].a.x, r[i].a.y, r[i].a.z, r[i].a.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) t[j] = __vmaxu2(t[j], w[j] & 0x7fff7fffu);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) { m[2 * j] = t[j] << 16; m[2 * j + 1] = t[j] & 0xffff0000u; }
}

// A 128 × 128 tile of which a thread holds 8 rows × 8 columns.  Magnitudes meet in shared memory, where one thread per row and per column
// makes the two factors (and writes the scale: 512 contiguous bytes per tile).  The transposed elements turn in shared memory: 16-byte
// pieces (rows of one column) at slot (piece ^ column / 8), two passes per access, no more conflicts.
template <typename T, int MODE>
__device__ __forceinline__ void fp8_tile(const Fp8TileParams& p, const Raw8<T> (&raw)[8], uint32_t* s_row, uint32_t (*s_col)[128], uint8_t* s_t,
                                         int rb, int kb) {
  const int t = threadIdx.x, warp = t >> 5, cg = t & 15, rg = t >> 4;      // column group, row group (8 each)
  const int r0 = rb * 128 + rg * 8, c0 = kb * 128 + cg * 8;
  float u_tile = 1.f;
  if (MODE == FP8_TILE) {
    uint32_t m[8];
    col_max(raw, m);
    uint32_t a = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) a = max(a, m[i]);
    a = __reduce_max_sync(0xffffffffu, a);
    if ((t & 31) == 0) s_row[warp] = a;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) a = max(a, s_row[i]);
    const float top = block_amax(a);
    u_tile = __fdiv_rn(kE4m3Max, top);
    if (t == 0) p.s[static_cast<int64_t>(rb) * p.cb + kb] = __fdiv_rn(top, kE4m3Max);
  } else {
    if (MODE & FP8_ROWS) {
      // eight rows over 16 lanes: at every step a lane hands half of its rows to a neighbour and keeps the other half
      uint32_t m[8];
      row_max(raw, m);
#pragma unroll
      for (int h = 4; h > 0; h >>= 1) {
        const bool up = (t & (2 * h)) != 0;
#pragma unroll
        for (int i = 0; i < h; ++i) {
          const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? m[i] : m[i + h], 2 * h);
          m[i] = max(up ? m[i + h] : m[i], got);
        }
      }
      m[0] = max(m[0], __shfl_xor_sync(0xffffffffu, m[0], 1));
      if ((t & 1) == 0) s_row[rg * 8 + (cg >> 1)] = m[0];
    }
    if (MODE & FP8_COLS) {                               // two row groups of a warp meet: a lane keeps four of its columns
      uint32_t m[8];
      col_max(raw, m);
      const bool up = (t & 16) != 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? m[e] : m[e + 4], 16);
        m[e] = max(up ? m[e + 4] : m[e], got);
      }
      *reinterpret_cast<uint4*>(&s_col[warp][cg * 8 + (up ? 4 : 0)]) = make_uint4(m[0], m[1], m[2], m[3]);
    }
    __syncthreads();
    if ((MODE & FP8_ROWS) && t < 128) {
      const float a = block_amax(s_row[t]);
      s_row[t] = __float_as_uint(__fdiv_rn(kE4m3Max, a));
      if (rb * 128 + t < p.rows) p.s[kb * p.lds + rb * 128 + t] = __fdiv_rn(a, kE4m3Max);
    }
    if ((MODE & FP8_COLS) && t >= 128) {
      const int c = t - 128;
      uint32_t m = s_col[0][c];
#pragma unroll
      for (int i = 1; i < 8; ++i) m = max(m, s_col[i][c]);
      const float a = block_amax(m);
      s_col[0][c] = __float_as_uint(__fdiv_rn(kE4m3Max, a));
      if (kb * 128 + c < p.cols) p.st[rb * p.ldst + kb * 128 + c] = __fdiv_rn(a, kE4m3Max);
    }
    __syncthreads();
  }
  if (((MODE & FP8_ROWS) || MODE == FP8_TILE) && c0 < p.cols) {            // 8-byte pieces: rows are padded to a multiple of 16
    uint8_t* q = p.q + static_cast<int64_t>(r0) * p.ldq + c0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float u = MODE == FP8_TILE ? u_tile : __uint_as_float(s_row[rg * 8 + i]);
      float o[8];
      unpack8(raw[i], o);
      scale8(o, u);
      if (r0 + i < p.rows) *reinterpret_cast<uint2*>(q + i * p.ldq) = pack_e4m3x8(o);
    }
  }
  if ((MODE & FP8_COLS) || (MODE == FP8_TILE && p.qt)) {
    float v[8][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) unpack8(raw[i], v[i]);
    float uc[8];
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      const float4 f = MODE == FP8_TILE ? make_float4(u_tile, u_tile, u_tile, u_tile) : *reinterpret_cast<const float4*>(&s_col[0][cg * 8 + e]);
      uc[e] = f.x; uc[e + 1] = f.y; uc[e + 2] = f.z; uc[e + 3] = f.w;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = v[i][e];
      scale8(o, uc[e]);
      *reinterpret_cast<uint2*>(s_t + (cg * 8 + e) * 128 + (((rg >> 1) ^ (cg & 7)) << 4) + ((rg & 1) << 3)) = pack_e4m3x8(o);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = i * 32 + (t >> 3), piece = t & 7;
      const int row = rb * 128 + piece * 16;
      if (kb * 128 + c < p.cols && row < p.rows)
        *reinterpret_cast<uint4*>(p.qt + static_cast<int64_t>(kb * 128 + c) * p.ldqt + row) =
            *reinterpret_cast<const uint4*>(s_t + c * 128 + ((piece ^ ((c >> 3) & 7)) << 4));
    }
  }
}

// One CTA per tile, read once.  Four fit an SM with bf16 (the form for any alignment has to be told: with 70 registers 317 µs instead of 270 at
// 30568 × 7981); fp32 takes the registers that it needs.
template <typename T, int MODE, bool NORM, bool VEC>
__global__ void __launch_bounds__(256, sizeof(T) == 2 && !NORM && !VEC ? 4 : 0) fp8_tile_kernel(const Fp8TileParams p) {
  __shared__ uint32_t s_row[128];
  __shared__ __align__(16) uint32_t s_col[8][128];
  __shared__ __align__(16) uint8_t s_t[(MODE & FP8_COLS) || MODE == FP8_TILE ? 128 * 128 : 16];
  const int cg = threadIdx.x & 15, rg = threadIdx.x >> 4;      // column group, row group (8 each)
  const int rb = blockIdx.x / p.cb, kb = blockIdx.x - rb * p.cb;
  const int r0 = rb * 128 + rg * 8, c0 = kb * 128 + cg * 8;
  const int nc = min(max(p.cols - c0, 0), 8);
  const T* x = static_cast<const T*>(p.x) + static_cast<int64_t>(r0) * p.ldx + c0;
  Raw8<T> raw[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) load_raw<VEC>(x + i * p.ldx, r0 + i < p.rows ? nc : 0, raw[i]);
  if (NORM) {                                            // (x · rstd[row]) · w[col] in fp32, kept in registers
    float w[8];
    if (p.w_f32) load8<false>(static_cast<const float*>(p.w) + c0, nc, w);
    else load8<false>(static_cast<const __nv_bfloat16*>(p.w) + c0, nc, w);
    Raw8<float> v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float rs = r0 + i < p.rows ? p.rstd[r0 + i] : 0.f;
      float t[8];
      unpack8(raw[i], t);
      scale8(t, rs);
      mul8(t, w);
      v[i].a = make_float4(t[0], t[1], t[2], t[3]);
      v[i].b = make_float4(t[4], t[5], t[6], t[7]);
    }
    fp8_tile<float, MODE>(p, v, s_row, s_col, s_t, rb, kb);
  } else {
    fp8_tile<T, MODE>(p, raw, s_row, s_col, s_t, rb, kb);
  }
}

template <typename T, int MODE, bool NORM>
static int launch_tile(const Fp8TileParams& p, cudaStream_t st) {
  const int64_t tiles = static_cast<int64_t>((p.rows + 127) / 128) * p.cb;
  if (tiles > 0x7fffffff) return -6;
  if (p.vec) fp8_tile_kernel<T, MODE, NORM, true><<<static_cast<unsigned>(tiles), 256, 0, st>>>(p);
  else fp8_tile_kernel<T, MODE, NORM, false><<<static_cast<unsigned>(tiles), 256, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

// ------------------------------------------------------------------ residual addition + RMSNorm → e4m3
//   x = res + h_scale · h (fp32, rounded to the stream's type),  n = x · rsqrt(mean x² + eps) · w (fp32),  n quantised in blocks of 128
// n is never rounded to 16 bits: the only rounding between the stream and the tensor cores is the one to e4m3.  1 / rms is common to a block, so
// with y = x · w (exact for bf16) and m = max |y| of the block, a = m / rms and n · 448 / a is y · (448 / m), where 448 / m is held with its rest
// in two numbers: what is rounded to e4m3 is off by half a unit of fp32, and values half way between two of e4m3, which factors of 8 bits
// make one in ten thousand, are found to be so.  Blocks at the floor of a, or with m below it, take (y / rms) · (448 / a).
struct Fp8NormParams {
  const void* res; const __nv_bfloat16* h; const void* w;
  float h_scale, eps;
  int rows, cols, vec, w_f32;
  void* x;                      // new stream (null without h)
  uint8_t* q; int64_t ldq;
  float* s; int64_t lds;
  float* rstd;                  // [rows] or null
};

// Eight values of a row per lane, neighbouring lanes' next to each other, by all lanes of a warp (n ≤ 0: none of this lane's).  Rows that start
// anywhere leave in aligned 16-byte pieces all the same: a lane gives its first values to the lane before it and takes the next one's; what no
// whole piece covers goes value by value.
template <bool VEC>
__device__ __forceinline__ void store_row(float* p, int n, const float (&v)[8]) {
  if (VEC) {
    if (n <= 0) return;
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
    return;
  }
  const int lane = threadIdx.x & 31, s = (-static_cast<int>(reinterpret_cast<uintptr_t>(p) >> 2)) & 3;       // values up to a boundary
  float w[11], t[9];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = v[i];
#pragma unroll
  for (int i = 0; i < 3; ++i) w[8 + i] = __shfl_down_sync(0xffffffffu, v[i], 1);
  const int behind = __shfl_down_sync(0xffffffffu, n, 1);
  const bool one = n >= s + 4, two = n >= 8 && (s == 0 || (lane < 31 && behind >= s));
  const bool before = __shfl_up_sync(0xffffffffu, two ? 1 : 0, 1) && lane > 0;
#pragma unroll
  for (int i = 0; i < 9; ++i) t[i] = (s & 2) ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = (s & 1) ? t[i + 1] : t[i];
  if (one) *reinterpret_cast<float4*>(p + s) = make_float4(w[0], w[1], w[2], w[3]);
  if (two) *reinterpret_cast<float4*>(p + s + 4) = make_float4(w[4], w[5], w[6], w[7]);
#pragma unroll
  for (int e = 0; e < 8; ++e) if (e < n && !(e < s ? before : e < s + 4 ? one : two)) p[e] = v[e];
}
template <bool VEC>
__device__ __forceinline__ void store_row(__nv_bfloat16* p, int n, const float (&v)[8]) {
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
  if (VEC) {
    if (n > 0) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    return;
  }
  const int lane = threadIdx.x & 31, s = (-static_cast<int>(reinterpret_cast<uintptr_t>(p) >> 1)) & 7;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[4 + i] = __shfl_down_sync(0xffffffffu, w[i], 1);
  const int behind = __shfl_down_sync(0xffffffffu, n, 1);
  const bool full = n >= 8 && (s == 0 || (lane < 31 && behind >= s));
  const bool before = __shfl_up_sync(0xffffffffu, full ? 1 : 0, 1) && lane > 0;
  uint32_t t[6], u[5], o[4];
#pragma unroll
  for (int i = 0; i < 6; ++i) t[i] = (s & 4) ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) u[i] = (s & 2) ? t[i + 1] : t[i];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = __funnelshift_r(u[i], u[i + 1], (s & 1) * 16);
  if (full) *reinterpret_cast<uint4*>(p + s) = make_uint4(o[0], o[1], o[2], o[3]);
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < n && !(e < s ? before : full)) p[e] = __ushort_as_bfloat16(static_cast<unsigned short>(w[e >> 1] >> ((e & 1) * 16)));
}
// bf16 in pairs that lie on 4 bytes: fewer instructions, which the norm itself is bound by (30568 × 7981: 515 µs this way, 584 in whole pieces,
// while its gradients take 1392 and 1183; fp32 880 and 642, 1834 and 1148).
__device__ __forceinline__ void store_pairs(__nv_bfloat16* p, int n, const float (&v)[8]) {
  if (n >= 8) {
    const int odd = static_cast<int>(reinterpret_cast<uintptr_t>(p) >> 1) & 1;
    if (odd) {
      p[0] = __float2bfloat16(v[0]);
#pragma unroll
      for (int i = 1; i < 7; i += 2) *reinterpret_cast<uint32_t*>(p + i) = pack_bf16x2(v[i], v[i + 1]);
      p[7] = __float2bfloat16(v[7]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i += 2) *reinterpret_cast<uint32_t*>(p + i) = pack_bf16x2(v[i], v[i + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) if (i < n) p[i] = __float2bfloat16(v[i]);
  }
}
__device__ __forceinline__ float round_to(float v, const float*) { return v; }
__device__ __forceinline__ float round_to(float v, const __nv_bfloat16*) { return __bfloat162float(__float2bfloat16(v)); }

// The sum of `v` over the CTAs of a cluster, which each have the threads' sums of one part of a row: every CTA writes its own to all of them
// (part: a buffer that nobody reads any more) and adds them in the order of the ranks.
template <int CL>
__device__ __forceinline__ float cluster_row_sum(float v, float* warps, float* part, int n_warps) {
  if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x < CL) {
    v = 0.f;
    for (int i = 0; i < n_warps; ++i) v += warps[i];
    uint32_t to;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_u32(part + cluster_ctarank())), "r"(threadIdx.x));
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(v) : "memory");
  }
  __syncwarp();
  cluster_sync_all();
  v = 0.f;
#pragma unroll
  for (int r = 0; r < CL; ++r) v += part[r];
  return v;
}

constexpr int NORM_V = 2;       // vectors of 8 values per thread
// PACK threads per row, or (0) a whole block, or a cluster of CL blocks: the row stays in registers.  16 neighbouring threads hold one block
// of 128.  Instructions cost nearly as much as bytes do (81 % of the issue slots were taken), hence values in pairs, maxima of three, and a
// half warp's four divisions at once: 16384 × 8192 bf16 149 µs (6.3 TB/s) instead of 189, 32768 × 2048 76 (6.2 TB/s) instead of 85.  40 registers
// (1536 threads per SM) are worth the few that are spilled: fp32 at 30568 × 7981 874 µs, 1002 with 44 to 51.
template <typename T, typename TO, int PACK, int CL, bool VEC, bool H>
__global__ void __launch_bounds__(PACK ? 128 : 512, PACK ? 12 : 3) fp8_norm_kernel(const Fp8NormParams p) {
  constexpr int V = NORM_V;
  __shared__ float s_sum[32], s_part[CL];
  const int TPR = PACK ? PACK : blockDim.x, RPC = PACK ? 128 / PACK : 1, WPR = TPR / 32;
  const int t = (PACK ? threadIdx.x % PACK : threadIdx.x) + (CL > 1 ? static_cast<int>(cluster_ctarank()) * TPR * V : 0);
  const int sub = PACK ? threadIdx.x / PACK : 0, row = static_cast<int>(blockIdx.x) / CL * RPC + sub;
  const bool live = row < p.rows;
  const int64_t base = static_cast<int64_t>(row) * p.cols;
  Raw8<T> xr[V];
  Raw8<__nv_bfloat16> hr[H ? V : 1];
#pragma unroll
  for (int i = 0; i < V; ++i) {                          // all of the row's loads first
    const int c = (t + i * TPR) * 8;
    const int n = live ? min(max(p.cols - c, 0), 8) : 0;
    load_raw<VEC>(static_cast<const T*>(p.res) + base + c, n, xr[i]);
    if (H) load_raw<VEC>(p.h + base + c, n, hr[i]);
  }
  if (CL > 1) cluster_sync_all();                        // every block of the cluster has started
  float v[V][8];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = (t + i * TPR) * 8;
    const int n = live ? min(max(p.cols - c, 0), 8) : 0;
    unpack8(xr[i], v[i]);
    if (H) {
      float h[8];
      unpack8(hr[i], h);
      scale8(h, p.h_scale);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = round_to(__fadd_rn(v[i][e], h[e]), static_cast<const TO*>(nullptr));
      if constexpr (!VEC && sizeof(TO) == 2) store_pairs(static_cast<TO*>(p.x) + base + c, n, v[i]);
      else store_row<VEC>(static_cast<TO*>(p.x) + base + c, n, v[i]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += v[i][e] * v[i][e];
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (CL > 1) {
    ss = cluster_row_sum<CL>(ss, s_sum, s_part, WPR);
  } else if (WPR > 1) {
    if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x >> 5] = ss;
    __syncthreads();
    ss = 0.f;
    for (int i = 0; i < WPR; ++i) ss += s_sum[sub * WPR + i];
  }
  const float rs = rsqrtf(ss / static_cast<float>(p.cols) + p.eps);
  if (live && t == 0 && p.rstd) p.rstd[row] = rs;
  float m[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = (t + i * TPR) * 8;
    const int n = live ? min(max(p.cols - c, 0), 8) : 0;
    float w[8];
    if (p.w_f32) load8<VEC>(static_cast<const float*>(p.w) + c, n, w);
    else load8<VEC>(static_cast<const __nv_bfloat16*>(p.w) + c, n, w);
    mul8(v[i], w);
    m[i] = max_abs(max_abs(max_abs(v[i][0], v[i][1], v[i][2]), v[i][3], v[i][4]), v[i][5], max_abs(v[i][6], v[i][7], 0.f));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m[i] = max_abs(m[i], __shfl_xor_sync(0xffffffffu, m[i], o), 0.f);
  }
  // the four divisions of two blocks on four lanes of each half warp: scales on the even ones, on the odd ones u = 448 / m and its rest, or,
  // marked by a rest that is no number, 448 / a
  static_assert(V == 2);
  const bool odd = (t & 1) != 0;
  const float top = (t & 2) ? m[1] : m[0], a = max_abs(__fmul_rn(top, rs), kBlockFloor, 0.f);
  const bool large = a > kBlockFloor && top > kBlockFloor;
  const float f = __fdiv_rn(odd ? kE4m3Max : a, !odd ? kE4m3Max : large ? top : a);
  const float rest = large ? fmaf(-f, top, kE4m3Max) * f * (1.f / kE4m3Max) : __int_as_float(0x7fffffff);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = (t + i * TPR) * 8;
    const float u = __shfl_sync(0xffffffffu, f, 2 * i + 1, 16);
    float u2 = __shfl_sync(0xffffffffu, rest, 2 * i + 1, 16);
    if (live && (t & 15) == 2 * i && c - 16 * i < p.cols) p.s[(c >> 7) * p.lds + row] = f;
    if (live && c < p.cols) {
      if (u2 != u2) { scale8(v[i], rs); u2 = 0.f; }
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float2 y = make_float2(v[i][e], v[i][e + 1]);
        const float2 z = fma_f32x2(y, make_float2(u, u), mul_f32x2(y, make_float2(u2, u2)));
        v[i][e] = z.x; v[i][e + 1] = z.y;
      }
      *reinterpret_cast<uint2*>(p.q + row * p.ldq + c) = pack_e4m3x8(v[i]);
    }
  }
}

// Rows share a block up to 1024 columns; wider ones have as many threads as leave none idle (2560 columns: 160), and past 8192 columns a
// cluster of blocks.  (One block of 1024 threads with four vectors each leaves 64 registers a thread: 32768 rows of 11264 bf16 took 1075 µs
// instead of 590 and their gradients 6775 instead of 1091; 8192 rows of 32768 2144 instead of 820, but the norm itself 383 instead of 473.)
struct NormShape { int pack, cl, threads; };
static NormShape norm_shape(int cols) {
  const int vecs = (cols + 7) / 8;
  if (vecs <= 64) return {32, 1, 128};
  if (vecs <= 128) return {64, 1, 128};
  const int cl = vecs <= 1024 ? 1 : vecs <= 2048 ? 2 : 4;
  return {0, cl, ((vecs + cl - 1) / cl + 32 * NORM_V - 1) / (32 * NORM_V) * 32};
}
template <typename P>
static int launch_rows(void (*kern)(P), const P& p, int blocks, const NormShape& shape, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks * shape.cl);
  cfg.blockDim = dim3(shape.threads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = shape.cl; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = shape.cl > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, p) == cudaSuccess ? 0 : -3;
}

template <typename T, typename TO>
static int launch_norm(const Fp8NormParams& p, cudaStream_t st) {
  const NormShape shape = norm_shape(p.cols);
  const int rpc = shape.pack ? 128 / shape.pack : 1;
  const int64_t blocks = (static_cast<int64_t>(p.rows) + rpc - 1) / rpc;
  if (blocks * shape.cl > 0x7fffffff) return -6;
#define FP8_NORM(PACK, CL)                                                                                                       \
  if (shape.pack == PACK && shape.cl == CL)                                                                                      \
    return launch_rows(p.vec ? (p.h ? fp8_norm_kernel<T, TO, PACK, CL, true, true> : fp8_norm_kernel<T, TO, PACK, CL, true, false>) \
                             : (p.h ? fp8_norm_kernel<T, TO, PACK, CL, false, true> : fp8_norm_kernel<T, TO, PACK, CL, false, false>), \
                       p, static_cast<int>(blocks), shape, st);
  FP8_NORM(32, 1) FP8_NORM(64, 1) FP8_NORM(0, 1) FP8_NORM(0, 2) FP8_NORM(0, 4)
#undef FP8_NORM
  return -6;
}

// ------------------------------------------------------------------ gradients of the norm and the addition
// With x̂ = x · rstd, t = dn · w:   d_res = g_x + rstd · (t − x̂ · mean(t · x̂)),   d_h = h_scale · d_res,   d_w = Σ_rows dn · x̂.
// dn is the fp32 output of the product behind the norm: rounded to bf16 it made the sums over rows 1.5 times as far off.
// Threads hold the columns that they hold in the forward kernel, so that d_w is summed in registers over a block's rows; the blocks' sums meet in
// a second kernel, in a fixed order.  Bound by memory: 12 bytes per element with a bf16 stream (32768 × 2048 136 µs, 5.9 TB/s).
struct Fp8NormBwdParams {
  const float* dn; int64_t ld_dn;       // rows of whole 32-byte pieces, whatever cols is
  const void *x, *gx, *w;
  const float* rstd;
  void* dres; __nv_bfloat16* dh;
  float* dw_part;               // [grid][cols] or null
  float h_scale;
  int rows, cols, vec, w_f32;
};

template <typename T, int PACK, int CL, bool VEC>
__global__ void __maxnreg__(CL > 1 ? 128 : 96) fp8_norm_bwd_kernel(const Fp8NormBwdParams p) {
  constexpr int RPC = PACK ? 128 / (PACK ? PACK : 1) : 1, V = NORM_V;
  __shared__ float s_sum[2][32], s_part[2][CL];
  __shared__ float s_dw[PACK ? 128 * V * 8 : 1];
  const int TPR = PACK ? PACK : blockDim.x, WPR = TPR / 32;
  const int t = (PACK ? threadIdx.x % PACK : threadIdx.x) + (CL > 1 ? static_cast<int>(cluster_ctarank()) * TPR * V : 0);
  const int sub = PACK ? threadIdx.x / PACK : 0, blk = static_cast<int>(blockIdx.x) / CL, blks = static_cast<int>(gridDim.x) / CL;
  float w[V][8], dw[V][8];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = (t + i * TPR) * 8, n = min(max(p.cols - c, 0), 8);
    if (p.w_f32) load8<VEC>(static_cast<const float*>(p.w) + c, n, w[i]);
    else load8<VEC>(static_cast<const __nv_bfloat16*>(p.w) + c, n, w[i]);
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[i][e] = 0.f;
  }
  if (CL > 1) cluster_sync_all();                        // every block of the cluster has started
  int it = 0;
  for (int64_t r0 = static_cast<int64_t>(blk) * RPC; r0 < p.rows; r0 += blks * RPC, ++it) {      // as many turns for all threads of a block or cluster
    const int64_t row = r0 + sub, base = row * p.cols;
    const bool live = row < p.rows;
    Raw8<float> dr[V];
    Raw8<T> xr[V], gr[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (t + i * TPR) * 8;
      const int n = live ? min(max(p.cols - c, 0), 8) : 0;
      load_raw<true>(p.dn + row * p.ld_dn + c, n, dr[i]);
      load_raw<VEC>(static_cast<const T*>(p.x) + base + c, n, xr[i]);
      load_raw<VEC>(static_cast<const T*>(p.gx) + base + c, p.gx ? n : 0, gr[i]);
    }
    const float rs = live ? p.rstd[row] : 0.f;
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (t + i * TPR) * 8;
      float d[8], x[8];
      unpack8(dr[i], d); unpack8(xr[i], x);
      if (!VEC && c + 8 > p.cols) {                      // what lies past the row is anything
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] = c + e < p.cols ? d[e] : 0.f;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float xhat = x[e] * rs;
        dot += d[e] * w[i][e] * xhat;
        dw[i][e] += d[e] * xhat;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    if (CL > 1) {                                        // two buffers: one barrier per row
      dot = cluster_row_sum<CL>(dot, s_sum[it & 1], s_part[it & 1], WPR);
    } else if (WPR > 1) {
      if ((threadIdx.x & 31) == 0) s_sum[it & 1][threadIdx.x >> 5] = dot;
      __syncthreads();
      dot = 0.f;
      for (int i = 0; i < WPR; ++i) dot += s_sum[it & 1][sub * WPR + i];
    }
    const float mean = dot / static_cast<float>(p.cols);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (t + i * TPR) * 8;
      const int n = live ? min(max(p.cols - c, 0), 8) : 0;
      float d[8], x[8], g[8];
      unpack8(dr[i], d); unpack8(xr[i], x); unpack8(gr[i], g);
#pragma unroll
      for (int e = 0; e < 8; ++e) g[e] += rs * (d[e] * w[i][e] - x[e] * rs * mean);
      if (p.dres) store_row<VEC>(static_cast<T*>(p.dres) + base + c, n, g);
      if (p.dh) {
        scale8(g, p.h_scale);
        store_row<VEC>(p.dh + base + c, n, g);
      }
    }
  }
  if (!p.dw_part) return;
  float* out = p.dw_part + static_cast<int64_t>(blk) * p.cols;
  if (PACK) {                                            // the block's rows in order
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) s_dw[(i * 8 + e) * 128 + threadIdx.x] = dw[i][e];
    __syncthreads();
    if (sub == 0) {
#pragma unroll
      for (int i = 0; i < V; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          for (int j = 1; j < RPC; ++j) dw[i][e] += s_dw[(i * 8 + e) * 128 + t + j * PACK];
    }
  }
  if (sub == 0) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (t + i * TPR) * 8;
      store_row<VEC>(out + c, min(max(p.cols - c, 0), 8), dw[i]);
    }
  }
}
__global__ void __launch_bounds__(1024) fp8_norm_dw_kernel(const float* __restrict__ part, float* __restrict__ out, int n, int cols) {
  const float t = column_sum_block(part, n, cols);
  const int c = blockIdx.x * 32 + threadIdx.x;
  if (threadIdx.x < 32 && c < cols) out[c] = t;
}

// Blocks (or clusters) of the backward kernel, and rows of its partial sums: as many blocks as fit the machine at once (96 registers a thread; with
// up to 128, as the compiler chose, only four of the five blocks per SM fit and 32768 × 2048 took 177 µs instead of 142).  How many clusters fit
// depends on the machine's groups of SMs, so there are several times as many, which even out.
static int norm_bwd_grid(int rows, int cols, int num_sms) {
  const NormShape shape = norm_shape(cols);
  const int rpc = shape.pack ? 128 / shape.pack : 1;
  const int64_t need = (static_cast<int64_t>(rows) + rpc - 1) / rpc;
  const int64_t room = shape.cl > 1 ? num_sms : static_cast<int64_t>(num_sms) * max(1, 640 / shape.threads);
  return static_cast<int>(need < room ? need : room);
}

template <typename T>
static int launch_norm_bwd(const Fp8NormBwdParams& p, int grid, cudaStream_t st) {
  const NormShape shape = norm_shape(p.cols);
#define FP8_NORM_BWD(PACK, CL)                                                                                                       \
  if (shape.pack == PACK && shape.cl == CL)                                                                                          \
    return launch_rows(p.vec ? fp8_norm_bwd_kernel<T, PACK, CL, true> : fp8_norm_bwd_kernel<T, PACK, CL, false>, p, grid, shape, st);
  FP8_NORM_BWD(32, 1) FP8_NORM_BWD(64, 1) FP8_NORM_BWD(0, 1) FP8_NORM_BWD(0, 2) FP8_NORM_BWD(0, 4)
#undef FP8_NORM_BWD
  return -6;
}

}  // namespace b200

// x [rows, cols] (dtype 0 fp32, 1 bf16, rows ldx elements apart).  mode: 1 rows (q, s), 2 columns (qt, st), 3 both, 4 tiles of
// 128 × 128 (q, s and, unless null, qt).  With rstd, w: the values are (x · rstd[row]) · w[col] (mode 2).  ldq, ldqt: multiples of 16.
extern "C" int b200_fp8_quantize(const void* x, int dtype, int64_t ldx, int rows, int cols, int mode, void* q, int64_t ldq, float* s,
                                 int64_t lds, void* qt, int64_t ldqt, float* st, int64_t ldst, const float* rstd, const void* w,
                                 int w_dtype, cudaStream_t stream) {
  using namespace b200;
  if (rows < 0 || cols < 0 || (dtype != 0 && dtype != 1) || mode < 1 || mode > 4 || (rstd && mode != 2)) return -6;
  if (rows == 0 || cols == 0) return 0;
  const int esz = dtype == 0 ? 4 : 2;
  Fp8TileParams p{x, ldx, rows, cols, (cols + 127) / 128,
                  cols % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx * esz % 16 == 0 ? 1 : 0,
                  static_cast<uint8_t*>(q), ldq, s, lds, static_cast<uint8_t*>(qt), ldqt, st, ldst, rstd, w, w_dtype == 0 ? 1 : 0};
  if (dtype == 0) {
    if (rstd) return launch_tile<float, FP8_COLS, true>(p, stream);
    if (mode == 1) return launch_tile<float, FP8_ROWS, false>(p, stream);
    if (mode == 2) return launch_tile<float, FP8_COLS, false>(p, stream);
    if (mode == 3) return launch_tile<float, FP8_ROWS | FP8_COLS, false>(p, stream);
    return launch_tile<float, FP8_TILE, false>(p, stream);
  }
  if (rstd) return launch_tile<__nv_bfloat16, FP8_COLS, true>(p, stream);
  if (mode == 1) return launch_tile<__nv_bfloat16, FP8_ROWS, false>(p, stream);
  if (mode == 2) return launch_tile<__nv_bfloat16, FP8_COLS, false>(p, stream);
  if (mode == 3) return launch_tile<__nv_bfloat16, FP8_ROWS | FP8_COLS, false>(p, stream);
  return launch_tile<__nv_bfloat16, FP8_TILE, false>(p, stream);
}

// res, x [rows, cols] dense (dtype 0 fp32, 1 bf16; x null without h), h bf16 or null, w [cols].  cols ≤ 32768.
extern "C" int b200_add_rmsnorm_fp8(const void* res, int res_dtype, const void* h, float h_scale, const void* w, int w_dtype, void* x,
                                    int x_dtype, void* q, int64_t ldq, float* s, int64_t lds, float* rstd, int rows, int cols, float eps,
                                    cudaStream_t stream) {
  using namespace b200;
  if (rows < 0 || cols < 1 || cols > 32768 || (x_dtype == 1 && res_dtype != 1)) return -6;
  if (rows == 0) return 0;
  const auto al = [](const void* ptr) { return reinterpret_cast<uintptr_t>(ptr) % 16 == 0; };
  const int vec = cols % 8 == 0 && al(res) && al(h) && al(x) && al(w) ? 1 : 0;
  Fp8NormParams p{res, static_cast<const __nv_bfloat16*>(h), w, h_scale, eps, rows, cols, vec,
                  w_dtype == 0 ? 1 : 0, x, static_cast<uint8_t*>(q), ldq, s, lds, rstd};
  if (res_dtype == 0) return launch_norm<float, float>(p, stream);
  return x_dtype == 0 ? launch_norm<__nv_bfloat16, float>(p, stream) : launch_norm<__nv_bfloat16, __nv_bfloat16>(p, stream);
}

// x, gx (or null) of x_dtype [rows, cols] dense; dn fp32, 16-byte aligned, its rows ld_dn apart, a multiple of 8 (the last row's padding is
// read too); dres (x_dtype), dh (bf16), dw (fp32 [cols], with dw_part [grid][cols]): null if not wanted.  grid: b200_add_rmsnorm_fp8_bwd_grid.
extern "C" int b200_add_rmsnorm_fp8_bwd_grid(int rows, int cols, int num_sms) { return b200::norm_bwd_grid(rows, cols, num_sms); }
extern "C" int b200_add_rmsnorm_fp8_bwd(const float* dn, int64_t ld_dn, const void* x, int x_dtype, const void* gx, const void* w, int w_dtype, const float* rstd,
                                        void* dres, void* dh, float h_scale, float* dw_part, float* dw, int rows, int cols, int grid,
                                        cudaStream_t stream) {
  using namespace b200;
  if (rows < 0 || cols < 1 || cols > 32768 || ld_dn % 8 || ld_dn < cols || reinterpret_cast<uintptr_t>(dn) % 16) return -6;
  if (rows == 0) return dw && cudaMemsetAsync(dw, 0, cols * sizeof(float), stream) != cudaSuccess ? -4 : 0;
  const auto al = [](const void* ptr) { return reinterpret_cast<uintptr_t>(ptr) % 16 == 0; };
  const int vec = cols % 8 == 0 && al(x) && al(gx) && al(w) && al(dres) && al(dh) ? 1 : 0;
  const Fp8NormBwdParams p{dn, ld_dn, x, gx, w, rstd, dres, static_cast<__nv_bfloat16*>(dh), dw ? dw_part : nullptr, h_scale, rows, cols, vec,
                           w_dtype == 0 ? 1 : 0};
  const int rc = x_dtype == 0 ? launch_norm_bwd<float>(p, grid, stream) : launch_norm_bwd<__nv_bfloat16>(p, grid, stream);
  if (rc || !dw) return rc;
  fp8_norm_dw_kernel<<<(cols + 31) / 32, 1024, 0, stream>>>(dw_part, dw, grid, cols);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}
