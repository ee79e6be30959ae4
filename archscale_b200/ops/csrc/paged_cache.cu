// Writer and reader of the paged key-value cache (layout in paged.cuh).
//
//   write   x = k[b, i, g, :] goes to its slot; in e4m3 with a = max |x|, e the smallest integer ≥ −127 with 448 · 2^e ≥ a:  q = e4m3(x · 2^−e), byte e + 127.
//           448 = 1.75 · 2^8, so e + 127 is the exponent field of a less 8, one more where the mantissa is above 1.75: one addition on the bits.  A
//           power of two costs nothing against a / 448 in a floating-point format (the relative spacing is the same) and makes the value that
//           is read back a bf16 number.  A head with an infinity or NaN gets byte 255 and reads back as NaN.
//   read    x = q · 2^e into dense rows, zeros past the end of a sequence.
//
// Memory-bound.  A head's row is held by D / 8 lanes, 8 values each (one 16-byte load of bf16), keys and values by the same lanes; rows that no 16 bytes
// divide go value by value on a whole warp.  A row waits for its length, its page and then its data, so a thread has two or four rows under way where
// there are enough of them to fill the device all the same, and one where latency counts.  Instructions were the next bound: no division per row,
// maxima of two bf16 values at a time.  G 4, D 128: 8 x 8192 tokens read from e4m3 41 us (4.9 TB/s; 65 with one row a thread), 4 x 4096 tokens written
// into e4m3 10.3 us (4.9 TB/s), both without the launch; one token 8.5 us, all of it the host's.
#include <cuda_fp8.h>
#include <type_traits>

#include "paged.cuh"

namespace b200 {

template <class T> struct Eight;         // 8 values as they are loaded, and as they are stored
template <> struct Eight<__nv_bfloat16> {
  uint4 u;
  __device__ void load(const __nv_bfloat16* p) { u = *reinterpret_cast<const uint4*>(p); }
  __device__ uint32_t top() const {                                             // of two at a time: magnitudes order as their bits do
    const uint32_t m = __vmaxu2(__vmaxu2(u.x & 0x7fff7fffu, u.y & 0x7fff7fffu), __vmaxu2(u.z & 0x7fff7fffu, u.w & 0x7fff7fffu));
    return max(m << 16, m & 0xffff0000u);
  }
  __device__ void get(float (&x)[8]) const {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
  }
  static __device__ void store(__nv_bfloat16* p, const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) { const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]); w[i] = *reinterpret_cast<const uint32_t*>(&h); }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <> struct Eight<float> {
  float4 u, v;
  __device__ void load(const float* p) { u = *reinterpret_cast<const float4*>(p); v = *reinterpret_cast<const float4*>(p + 4); }
  __device__ uint32_t top() const {
    float x[8];
    get(x);
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
    return m;
  }
  __device__ void get(float (&x)[8]) const { x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w; x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w; }
  static __device__ void store(float* p, const float (&x)[8]) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
  }
};
template <> struct Eight<__nv_fp8_e4m3> {
  uint2 u;
  __device__ void load(const __nv_fp8_e4m3* p) { u = *reinterpret_cast<const uint2*>(p); }
  __device__ void get(float (&x)[8]) const {
    const uint32_t w[2] = {u.x, u.y};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w[i >> 1] >> (16 * (i & 1))), __NV_E4M3);
      const float2 f = __half22float2(__half2(h));
      x[2 * i] = f.x; x[2 * i + 1] = f.y;
    }
  }
  static __device__ void store(__nv_fp8_e4m3* p, const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __nv_cvt_float2_to_fp8x2(make_float2(x[2 * i], x[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
  }
};
__device__ __forceinline__ float one_value(const float* p) { return *p; }
__device__ __forceinline__ float one_value(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float one_value(const __nv_fp8_e4m3* p) { return static_cast<float>(*p); }
__device__ __forceinline__ void put_value(float* p, float x) { *p = x; }
__device__ __forceinline__ void put_value(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ void put_value(__nv_fp8_e4m3* p, float x) { p->__x = __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3); }

// A lane's share of a row: 8 neighbouring values (VEC), or every 32nd value, up to 8 of them.
template <bool VEC, class T> struct Share;
template <class T> struct Share<true, T> {
  Eight<T> e;
  __device__ void load(const T* row, int lane, int D) { if (8 * lane < D) e.load(row + 8 * lane); else e = {}; }
  __device__ void get(float (&x)[8]) const { e.get(x); }
  __device__ uint32_t top() const { return e.top(); }
  static __device__ void store(T* row, int lane, int D, const float (&x)[8]) { if (8 * lane < D) Eight<T>::store(row + 8 * lane, x); }
};
template <class T> struct Share<false, T> {
  float v[8];
  __device__ void load(const T* row, int lane, int D) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = lane + 32 * i < D ? one_value(row + lane + 32 * i) : 0.f;
  }
  __device__ void get(float (&x)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = v[i];
  }
  __device__ uint32_t top() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    return m;
  }
  static __device__ void store(T* row, int lane, int D, const float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) if (lane + 32 * i < D) put_value(row + lane + 32 * i, x[i]);
  }
};

// Scale byte of a row from the bits of a lane's largest magnitude (NaN above all), and the power of two that its values are multiplied with (0: they are
// zeros).  LANES neighbouring lanes hold the row.
template <int LANES>
__device__ __forceinline__ uint32_t to_scale(uint32_t top, float& up) {
#pragma unroll
  for (int o = 1; o < LANES; o *= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  const uint32_t code = max(0, static_cast<int>((top + 0x1fffffu) >> 23) - 8);
  up = __uint_as_float((254u - code) << 23);
  return top >= 0x7f800000u ? 255u : code;
}
// token and head of a row, and the steps to this thread's next one
struct Place {
  int t, g, dt, dg, groups;
  __device__ Place(uint32_t row, uint32_t step, int groups_) : groups(groups_) {
    const uint32_t n = groups_;
    t = row / n; g = row % n; dt = step / n; dg = step % n;
  }
  __device__ void next() {
    t += dt; g += dg;
    if (g >= groups) { g -= groups; ++t; }
  }
};
// page of a token's position in its sequence, and slot in the page
__device__ __forceinline__ int page_index(int pos, int size, int shift) { return shift >= 0 ? pos >> shift : pos / size; }

constexpr int PC_THREADS = 256;

// ROWS: rows (token, head) of a thread, a grid's step apart from each other
template <class In, class Cache, int LANES, bool VEC, int ROWS>
__global__ void __launch_bounds__(PC_THREADS) paged_write_kernel(const PagedView c, const In* k, const In* v, int64_t kb, int64_t kt, int64_t kh, int64_t vb,
                                                                 int64_t vt, int64_t vh, int B, int T, int shift, bool alike) {
  constexpr bool E8 = sizeof(Cache) == 1;
  constexpr int STEP = PC_THREADS / LANES;
  const int lane = threadIdx.x % LANES;
  const uint32_t row0 = blockIdx.x * (STEP * ROWS) + threadIdx.x / LANES;
  for (int b = blockIdx.y; b < B; b += gridDim.y) {
    const int n = paged_new(c, b, T);
    const int64_t first = static_cast<int64_t>(c.lengths[b]) - n;
    Share<VEC, In> x[ROWS], y[ROWS];
    int page[ROWS], slot[ROWS], g[ROWS];
    Place at(row0, STEP, c.groups);
#pragma unroll
    for (int i = 0; i < ROWS; ++i, at.next()) {
      page[i] = -1; slot[i] = 0; g[i] = at.g;
      if (at.t < n && first + at.t >= 0) {
        const int pos = static_cast<int>(first + at.t), index = page_index(pos, c.page_size, shift);
        page[i] = paged_page(c, b, index);
        slot[i] = pos - index * c.page_size;
        x[i].load(k + b * kb + at.t * kt + at.g * kh, lane, c.dim);
        y[i].load(v + b * vb + at.t * vt + at.g * vh, lane, c.dim);
      } else x[i] = y[i] = {};
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      float p[8], q[8];
      x[i].get(p); y[i].get(q);
      uint32_t ex = 0, ey = 0;
      if constexpr (E8) {                                                       // all lanes take part in the exchange of maxima
        float px, py;
        ex = to_scale<LANES>(x[i].top(), px); ey = to_scale<LANES>(y[i].top(), py);
#pragma unroll
        for (int j = 0; j < 8; ++j) { p[j] = ex == 255u ? 0.f : p[j] * px; q[j] = ey == 255u ? 0.f : q[j] * py; }
      }
      if (page[i] < 0) continue;                                                // the same for the lanes of a row
      const int64_t to = page[i] * c.k_page + g[i] * c.k_group + slot[i] * c.k_slot;
      Share<VEC, Cache>::store(static_cast<Cache*>(c.k) + to, lane, c.dim, p);
      Share<VEC, Cache>::store(static_cast<Cache*>(c.v) + (alike ? to : page[i] * c.v_page + g[i] * c.v_group + slot[i] * c.v_slot), lane, c.dim, q);
      if (E8 && lane == 0) {
        c.ks[page[i] * c.ks_page + g[i] * c.ks_group + slot[i] * c.ks_slot] = ex;
        c.vs[page[i] * c.vs_page + g[i] * c.vs_group + slot[i] * c.vs_slot] = ey;
      }
    }
  }
}

template <class Cache, class Out, int LANES, bool VEC, int ROWS>
__global__ void __launch_bounds__(PC_THREADS) paged_read_kernel(const PagedView c, Out* k, Out* v, int B, int tokens, int shift, bool alike) {
  constexpr bool E8 = sizeof(Cache) == 1;
  constexpr int STEP = PC_THREADS / LANES;
  const int lane = threadIdx.x % LANES;
  const uint32_t row0 = blockIdx.x * (STEP * ROWS) + threadIdx.x / LANES;
  for (int b = blockIdx.y; b < B; b += gridDim.y) {
    const int length = c.lengths[b];
    Share<VEC, Cache> x[ROWS], y[ROWS];
    int page[ROWS], slot[ROWS], g[ROWS];
    Place at(row0, STEP, c.groups);
#pragma unroll
    for (int i = 0; i < ROWS; ++i, at.next()) {                                 // all pages, then all rows
      const int index = page_index(at.t, c.page_size, shift);
      g[i] = at.g;
      page[i] = at.t < tokens && at.t < length ? paged_page(c, b, index) : -1;
      slot[i] = at.t - index * c.page_size;
    }
    float sx[ROWS], sy[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      sx[i] = sy[i] = 0.f;
      if (page[i] < 0) { x[i] = y[i] = {}; continue; }
      const int64_t from = page[i] * c.k_page + g[i] * c.k_group + slot[i] * c.k_slot;
      x[i].load(static_cast<const Cache*>(c.k) + from, lane, c.dim);
      y[i].load(static_cast<const Cache*>(c.v) + (alike ? from : page[i] * c.v_page + g[i] * c.v_group + slot[i] * c.v_slot), lane, c.dim);
      if constexpr (E8) {
        sx[i] = paged_pow2(c.ks[page[i] * c.ks_page + g[i] * c.ks_group + slot[i] * c.ks_slot]);
        sy[i] = paged_pow2(c.vs[page[i] * c.vs_page + g[i] * c.vs_group + slot[i] * c.vs_slot]);
      }
    }
    const uint32_t rows = static_cast<uint32_t>(tokens) * c.groups;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const uint32_t row = row0 + i * STEP;
      if (row >= rows) continue;
      float p[8], q[8];
      x[i].get(p); y[i].get(q);
      if constexpr (E8) {
#pragma unroll
        for (int j = 0; j < 8; ++j) { p[j] *= sx[i]; q[j] *= sy[i]; }
      }
      const int64_t to = (static_cast<int64_t>(b) * rows + row) * c.dim;
      Share<VEC, Out>::store(k + to, lane, c.dim, p);
      Share<VEC, Out>::store(v + to, lane, c.dim, q);
    }
  }
}

// log2 of the page size, or -1
static int pc_shift(const PagedView& c) {
  for (int i = 0; i < 31; ++i) if (c.page_size == 1 << i) return i;
  return -1;
}
static bool pc_alike(const PagedView& c) { return c.k_page == c.v_page && c.k_group == c.v_group && c.k_slot == c.v_slot; }
static bool whole(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
static int element(int type) { return type == 0 ? 4 : type == 1 ? 2 : 1; }
static int align8(int type) { return type == 2 ? 8 : 16; }             // bytes of the widest access to 8 values
// whether rows of the cache can be moved 8 values at a time
static bool cache_vec(const PagedView& c) {
  const int64_t strides = c.k_page | c.k_group | c.k_slot | c.v_page | c.v_group | c.v_slot;
  return c.dim % 8 == 0 && strides % (align8(c.type) / element(c.type)) == 0 && whole(c.k, align8(c.type)) && whole(c.v, align8(c.type));
}

// Lanes of a row.
template <class F>
static void pc_lanes(int dim, bool vec, F&& go) {
  if (!vec) go(std::integral_constant<int, 32>{}, std::false_type{});
  else if (dim <= 64) go(std::integral_constant<int, 8>{}, std::true_type{});
  else if (dim <= 128) go(std::integral_constant<int, 16>{}, std::true_type{});
  else go(std::integral_constant<int, 32>{}, std::true_type{});
}
// Rows of a thread: four where that still gives every SM its 2048 threads.
template <class F>
static void pc_grid(int64_t rows, int B, int lanes, F&& go) {
  const int step = PC_THREADS / lanes, per = rows * lanes * B >= 8LL * 148 * 2048 ? 4 : rows * lanes * B >= 2LL * 148 * 2048 ? 2 : 1;
  go(per, dim3(static_cast<unsigned>((rows + step * per - 1) / (step * per)), static_cast<unsigned>(B < 65535 ? B : 65535)));
}

template <class In, class Cache>
static int write_as(const PagedView& c, const void* k, const void* v, int64_t kb, int64_t kt, int64_t kh, int64_t vb, int64_t vt, int64_t vh, int B, int T,
                    bool vec, cudaStream_t st) {
  auto go = [&](auto lanes_c, auto vec_c) {
    constexpr int LANES = decltype(lanes_c)::value;
    constexpr bool VEC = decltype(vec_c)::value;
    pc_grid(static_cast<int64_t>(T) * c.groups, B, LANES, [&](int per, dim3 grid) {
      auto kernel = per == 1 ? paged_write_kernel<In, Cache, LANES, VEC, 1> : per == 2 ? paged_write_kernel<In, Cache, LANES, VEC, 2> : paged_write_kernel<In, Cache, LANES, VEC, 4>;
      kernel<<<grid, PC_THREADS, 0, st>>>(c, static_cast<const In*>(k), static_cast<const In*>(v), kb, kt, kh, vb, vt, vh, B, T, pc_shift(c), pc_alike(c));
    });
  };
  pc_lanes(c.dim, vec, go);
  return static_cast<int>(cudaGetLastError());
}

template <class Cache, class Out>
static int read_as(const PagedView& c, void* k, void* v, int B, int tokens, bool vec, cudaStream_t st) {
  auto go = [&](auto lanes_c, auto vec_c) {
    constexpr int LANES = decltype(lanes_c)::value;
    constexpr bool VEC = decltype(vec_c)::value;
    pc_grid(static_cast<int64_t>(tokens) * c.groups, B, LANES, [&](int per, dim3 grid) {
      auto kernel = per == 1 ? paged_read_kernel<Cache, Out, LANES, VEC, 1> : per == 2 ? paged_read_kernel<Cache, Out, LANES, VEC, 2> : paged_read_kernel<Cache, Out, LANES, VEC, 4>;
      kernel<<<grid, PC_THREADS, 0, st>>>(c, static_cast<Out*>(k), static_cast<Out*>(v), B, tokens, pc_shift(c), pc_alike(c));
    });
  };
  pc_lanes(c.dim, vec, go);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace b200

extern "C" int b200_paged_write(const b200_paged_view* c, const void* k, const void* v, int type, int64_t kb, int64_t kt, int64_t kh, int64_t vb, int64_t vt,
                                int64_t vh, int B, int T, cudaStream_t st) {
  using namespace b200;
  if (B <= 0 || T <= 0) return 0;
  if (static_cast<int64_t>(T) * c->groups > 0x7fff0000LL) return STATUS_BAD_ARG;      // rows are counted in 32 bits
  const int64_t unit = 16 / element(type);
  const bool vec = cache_vec(*c) && (kb | kt | kh | vb | vt | vh) % unit == 0 && whole(k, 16) && whole(v, 16);
  auto go = [&](auto in) {
    using In = decltype(in);
    if (c->type == 0) return write_as<In, float>(*c, k, v, kb, kt, kh, vb, vt, vh, B, T, vec, st);
    if (c->type == 1) return write_as<In, __nv_bfloat16>(*c, k, v, kb, kt, kh, vb, vt, vh, B, T, vec, st);
    return write_as<In, __nv_fp8_e4m3>(*c, k, v, kb, kt, kh, vb, vt, vh, B, T, vec, st);
  };
  return type == 0 ? go(float{}) : go(__nv_bfloat16{});
}

extern "C" int b200_paged_read(const b200_paged_view* c, void* k, void* v, int type, int B, int tokens, cudaStream_t st) {
  using namespace b200;
  if (B <= 0 || tokens <= 0) return 0;
  if (static_cast<int64_t>(tokens) * c->groups > 0x7fff0000LL) return STATUS_BAD_ARG;      // rows are counted in 32 bits
  const bool vec = cache_vec(*c) && whole(k, 16) && whole(v, 16);
  auto go = [&](auto out) {
    using Out = decltype(out);
    if (c->type == 0) return read_as<float, Out>(*c, k, v, B, tokens, vec, st);
    if (c->type == 1) return read_as<__nv_bfloat16, Out>(*c, k, v, B, tokens, vec, st);
    return read_as<__nv_fp8_e4m3, Out>(*c, k, v, B, tokens, vec, st);
  };
  return type == 0 ? go(float{}) : go(__nv_bfloat16{});
}
