// Writer and reader of the paged key-value cache (layout in paged.cuh).
//
//   write   x = k[b, i, g, :] goes to its slot; in e4m3 with a = max |x|, e the smallest integer ≥ −127 with 448 · 2^e ≥ a:  q = e4m3(x · 2^−e), byte e + 127.
//           448 = 1.75 · 2^8, so e + 127 is the exponent field of a less 8, one more where the mantissa is above 1.75: one addition on the bits.  A
//           power of two costs nothing against a / 448 in a floating-point format (the relative spacing is the same) and makes the value that
//           is read back a bf16 number.  A head with an infinity or NaN gets byte 255 and reads back as NaN.
//   read    x = q · 2^e into dense rows, zeros past the end of a sequence.
//
// Memory-bound.  A head's row is held by D / 8 lanes, 8 values each (one 16-byte load of bf16), keys and values by the same lanes; rows that no 16 bytes
// divide go value by value on a whole warp.
#include <cuda_fp8.h>

#include "paged.cuh"

namespace b200 {

template <class T> struct Vals;          // 8 values as they are loaded and stored
template <> struct Vals<__nv_bfloat16> {
  static __device__ void load(const __nv_bfloat16* p, float (&x)[8]) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
  }
  static __device__ void store(__nv_bfloat16* p, const float (&x)[8]) {
    uint4 u;
    uint32_t* w = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) { const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]); w[i] = *reinterpret_cast<const uint32_t*>(&h); }
    *reinterpret_cast<uint4*>(p) = u;
  }
};
template <> struct Vals<float> {
  static __device__ void load(const float* p, float (&x)[8]) {
    *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(p);
    *reinterpret_cast<float4*>(x + 4) = *reinterpret_cast<const float4*>(p + 4);
  }
  static __device__ void store(float* p, const float (&x)[8]) {
    *reinterpret_cast<float4*>(p) = *reinterpret_cast<const float4*>(x);
    *reinterpret_cast<float4*>(p + 4) = *reinterpret_cast<const float4*>(x + 4);
  }
};
template <> struct Vals<__nv_fp8_e4m3> {
  static __device__ void load(const __nv_fp8_e4m3* p, float (&x)[8]) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
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
template <bool VEC, class T>
__device__ __forceinline__ void load_share(const T* row, int lane, int D, float (&x)[8]) {
  if constexpr (VEC) {
    if (8 * lane < D) { Vals<T>::load(row + 8 * lane, x); return; }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.f;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = lane + 32 * i < D ? one_value(row + lane + 32 * i) : 0.f;
  }
}
template <bool VEC, class T>
__device__ __forceinline__ void store_share(T* row, int lane, int D, const float (&x)[8]) {
  if constexpr (VEC) {
    if (8 * lane < D) Vals<T>::store(row + 8 * lane, x);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) if (lane + 32 * i < D) put_value(row + lane + 32 * i, x[i]);
  }
}

// Scale byte of a row from its values, which become x · 2^−e.  LANES neighbouring lanes hold the row.
template <int LANES>
__device__ __forceinline__ uint32_t to_scale(float (&x)[8]) {
  uint32_t top = 0;                        // magnitudes order as their bits do, NaN above all
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
  for (int o = 1; o < LANES; o *= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (top >= 0x7f800000u) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.f;
    return 255u;
  }
  const int code = max(0, static_cast<int>((top + 0x1fffffu) >> 23) - 8);
  const float up = __uint_as_float(static_cast<uint32_t>(254 - code) << 23);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] *= up;
  return code;
}

constexpr int PC_THREADS = 256;

template <class In, class Cache, int LANES, bool VEC>
__global__ void __launch_bounds__(PC_THREADS) paged_write_kernel(const PagedView c, const In* k, const In* v, int64_t kb, int64_t kt, int64_t kh, int64_t vb,
                                                                 int64_t vt, int64_t vh, int B, int T) {
  constexpr bool E8 = sizeof(Cache) == 1;
  const int lane = threadIdx.x % LANES;
  const uint32_t row = blockIdx.x * (PC_THREADS / LANES) + threadIdx.x / LANES;                            // (token, head)
  const int t = static_cast<int>(row / static_cast<uint32_t>(c.groups)), g = static_cast<int>(row % static_cast<uint32_t>(c.groups));
  for (int b = blockIdx.y; b < B; b += gridDim.y) {
    const int n = paged_new(c, b, T);
    int page = -1, slot = 0;
    if (t < n) {
      const int64_t pos = static_cast<int64_t>(c.lengths[b]) - n + t;
      if (pos >= 0) { page = paged_page(c, b, static_cast<int>(pos) / c.page_size); slot = static_cast<int>(pos) % c.page_size; }
    }
    const bool live = page >= 0;           // the same for the lanes of a row; all lanes take part in the exchange of maxima
    float x[8] = {}, y[8] = {};
    if (live) {
      load_share<VEC>(k + b * kb + t * kt + g * kh, lane, c.dim, x);
      load_share<VEC>(v + b * vb + t * vt + g * vh, lane, c.dim, y);
    }
    uint32_t ex = 0, ey = 0;
    if constexpr (E8) { ex = to_scale<LANES>(x); ey = to_scale<LANES>(y); }
    if (live) {
      store_share<VEC>(static_cast<Cache*>(c.k) + page * c.k_page + g * c.k_group + slot * c.k_slot, lane, c.dim, x);
      store_share<VEC>(static_cast<Cache*>(c.v) + page * c.v_page + g * c.v_group + slot * c.v_slot, lane, c.dim, y);
      if (E8 && lane == 0) {
        c.ks[page * c.ks_page + g * c.ks_group + slot * c.ks_slot] = ex;
        c.vs[page * c.vs_page + g * c.vs_group + slot * c.vs_slot] = ey;
      }
    }
  }
}

template <class Cache, class Out, int LANES, bool VEC>
__global__ void __launch_bounds__(PC_THREADS) paged_read_kernel(const PagedView c, Out* k, Out* v, int B, int tokens) {
  constexpr bool E8 = sizeof(Cache) == 1;
  const int lane = threadIdx.x % LANES;
  const uint32_t row = blockIdx.x * (PC_THREADS / LANES) + threadIdx.x / LANES;
  const int t = static_cast<int>(row / static_cast<uint32_t>(c.groups)), g = static_cast<int>(row % static_cast<uint32_t>(c.groups));
  if (t >= tokens) return;
  for (int b = blockIdx.y; b < B; b += gridDim.y) {
    const int page = t < c.lengths[b] ? paged_page(c, b, t / c.page_size) : -1, slot = t % c.page_size;
    float x[8] = {}, y[8] = {};
    if (page >= 0) {
      load_share<VEC>(static_cast<const Cache*>(c.k) + page * c.k_page + g * c.k_group + slot * c.k_slot, lane, c.dim, x);
      load_share<VEC>(static_cast<const Cache*>(c.v) + page * c.v_page + g * c.v_group + slot * c.v_slot, lane, c.dim, y);
      if constexpr (E8) {
        const float sx = paged_pow2(c.ks[page * c.ks_page + g * c.ks_group + slot * c.ks_slot]);
        const float sy = paged_pow2(c.vs[page * c.vs_page + g * c.vs_group + slot * c.vs_slot]);
#pragma unroll
        for (int i = 0; i < 8; ++i) { x[i] *= sx; y[i] *= sy; }
      }
    }
    const int64_t at = (static_cast<int64_t>(b) * tokens * c.groups + row) * c.dim;
    store_share<VEC>(k + at, lane, c.dim, x);
    store_share<VEC>(v + at, lane, c.dim, y);
  }
}

static bool whole(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
static int element(int type) { return type == 0 ? 4 : type == 1 ? 2 : 1; }
static int align8(int type) { return type == 2 ? 8 : 16; }             // bytes of the widest access to 8 values
// whether rows of the cache can be moved 8 values at a time
static bool cache_vec(const PagedView& c) {
  const int64_t strides = c.k_page | c.k_group | c.k_slot | c.v_page | c.v_group | c.v_slot;
  return c.dim % 8 == 0 && strides % (align8(c.type) / element(c.type)) == 0 && whole(c.k, align8(c.type)) && whole(c.v, align8(c.type));
}

template <class In, class Cache>
static int write_as(const PagedView& c, const void* k, const void* v, int64_t kb, int64_t kt, int64_t kh, int64_t vb, int64_t vt, int64_t vh, int B, int T,
                    bool vec, cudaStream_t st) {
  const int64_t rows = static_cast<int64_t>(T) * c.groups;
  auto go = [&](auto kernel, int lanes) {
    const int64_t per = PC_THREADS / lanes;
    kernel<<<dim3(static_cast<unsigned>((rows + per - 1) / per), static_cast<unsigned>(B < 65535 ? B : 65535)), PC_THREADS, 0, st>>>(
        c, static_cast<const In*>(k), static_cast<const In*>(v), kb, kt, kh, vb, vt, vh, B, T);
  };
  if (!vec) go(paged_write_kernel<In, Cache, 32, false>, 32);
  else if (c.dim <= 64) go(paged_write_kernel<In, Cache, 8, true>, 8);
  else if (c.dim <= 128) go(paged_write_kernel<In, Cache, 16, true>, 16);
  else go(paged_write_kernel<In, Cache, 32, true>, 32);
  return static_cast<int>(cudaGetLastError());
}

template <class Cache, class Out>
static int read_as(const PagedView& c, void* k, void* v, int B, int tokens, bool vec, cudaStream_t st) {
  const int64_t rows = static_cast<int64_t>(tokens) * c.groups;
  auto go = [&](auto kernel, int lanes) {
    const int64_t per = PC_THREADS / lanes;
    kernel<<<dim3(static_cast<unsigned>((rows + per - 1) / per), static_cast<unsigned>(B < 65535 ? B : 65535)), PC_THREADS, 0, st>>>(
        c, static_cast<Out*>(k), static_cast<Out*>(v), B, tokens);
  };
  if (!vec) go(paged_read_kernel<Cache, Out, 32, false>, 32);
  else if (c.dim <= 64) go(paged_read_kernel<Cache, Out, 8, true>, 8);
  else if (c.dim <= 128) go(paged_read_kernel<Cache, Out, 16, true>, 16);
  else go(paged_read_kernel<Cache, Out, 32, true>, 32);
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
