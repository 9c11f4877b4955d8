// What 8-bit operands with a scale for each block of 128 values have in common (fp8_block.cu, gemm_fp8_block.cu, gemm_fp8_block_few.cu).
//
//   scale = max(amax, 2^-100) / 448,  q = e4m3(x * 448 / amax),  x' = q * scale
//
// 448 is the largest e4m3 value.  Values of 16-bit types often lie exactly halfway between two codes: there the quotient has to be exact for
// the half to go to the even code, so the product with the reciprocal is corrected by its remainder (one step of Newton's method with a fused
// multiply-add).  A block that holds an infinity or NaN has the scale NaN, so that an overflow stays visible.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "f32x2.cuh"

namespace sb {
namespace blk8 {

typedef __nv_bfloat16 bf16;
constexpr int BLOCK = 128;

__device__ __forceinline__ uint32_t magnitude(float f) { return __float_as_uint(f) & 0x7fffffffu; }

// The reciprocal is CUDA's approximate one: the remainder makes good what it lacks.  The quotient is in units of 2^20, in which x * 448 cannot overflow and a magnitude of 2^-100 is still far from the subnormal numbers.
struct Coder {
  float scale, minus_amax, inv;
  // m: bits of the block's largest magnitude.  rounded: CUDA's correctly rounded reciprocal instead
  __device__ __forceinline__ explicit Coder(uint32_t m, bool rounded = false) {
    const float a = fmaxf(__uint_as_float(m), 7.8886090522101181e-31f);  // 2^-100
    scale = m < 0x7f800000u ? __fmul_rn(a, 1.f / 448.f) : __uint_as_float(0x7fffffffu);
    const float amax = a * 9.5367431640625e-07f;
    minus_amax = -amax;
    if (rounded) inv = __frcp_rn(amax);
    else asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(amax));
  }
};
// Two values as two codes: of one block, or of two (columns)
__device__ __forceinline__ uint32_t code2(f2 x, f2 inv, f2 minus_amax) {
  const float top = 448.f * 9.5367431640625e-07f;
  const f2 n = f2_mul(x, f2_pack(top, top)), q = f2_mul(n, inv);
  return __nv_cvt_float2_to_fp8x2(f2_unpack(f2_fma(f2_fma(q, minus_amax, n), inv, q)), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint2 encode(const Coder& c, const f2 (&v)[4]) {
  const f2 inv = f2_pack(c.inv, c.inv), m = f2_pack(c.minus_amax, c.minus_amax);
  return make_uint2(code2(v[0], inv, m) | code2(v[1], inv, m) << 16, code2(v[2], inv, m) | code2(v[3], inv, m) << 16);
}
__device__ __forceinline__ float2 decode2(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(two & 0xffffu), __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// Magnitudes of eight values in columns of their own, their element-wise maximum, the largest of all and one of them (as fp32 bits).  Those of
// 16-bit types order as integers, two in a word.
template <class T> struct Magnitudes {
  uint32_t w[sizeof(T) == 2 ? 4 : 8];
};
template <class T> __device__ __forceinline__ uint32_t widen(uint32_t m16);
template <> __device__ __forceinline__ uint32_t widen<__nv_bfloat16>(uint32_t m) { return m << 16; }
template <> __device__ __forceinline__ uint32_t widen<__half>(uint32_t m) { return __float_as_uint(__half2float(__ushort_as_half((unsigned short)m))); }
template <> __device__ __forceinline__ uint32_t widen<float>(uint32_t m) { return m; }
template <class T> __device__ __forceinline__ uint32_t max_of(uint32_t a, uint32_t b) { return sizeof(T) == 2 ? __vmaxu2(a, b) : max(a, b); }
template <class T> __device__ __forceinline__ uint32_t largest(const Magnitudes<T>& m) {
  constexpr int N = sizeof(T) == 2 ? 4 : 8;
  uint32_t r = m.w[0];
#pragma unroll
  for (int i = 1; i < N; ++i) r = max_of<T>(r, m.w[i]);
  return sizeof(T) == 2 ? widen<T>(max(r & 0xffffu, r >> 16)) : r;
}

// The largest magnitudes of eight values of each of two rows, over the 16 threads that share the rows.  16-bit magnitudes travel two in a word.
template <class T> __device__ __forceinline__ void largest_of_rows(const Magnitudes<T>& a, const Magnitudes<T>& b, uint32_t& ma, uint32_t& mb) {
  if constexpr (sizeof(T) == 2) {
    const uint32_t x = __vmaxu2(__vmaxu2(a.w[0], a.w[1]), __vmaxu2(a.w[2], a.w[3])), y = __vmaxu2(__vmaxu2(b.w[0], b.w[1]), __vmaxu2(b.w[2], b.w[3]));
    uint32_t m = __vmaxu2(__byte_perm(x, y, 0x5410), __byte_perm(x, y, 0x7632));
#pragma unroll
    for (int o = 8; o; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
    ma = widen<T>(m & 0xffffu);
    mb = widen<T>(m >> 16);
  } else {
    ma = largest(a);
    mb = largest(b);
#pragma unroll
    for (int o = 8; o; o >>= 1) {
      ma = max(ma, __shfl_xor_sync(0xffffffffu, ma, o));
      mb = max(mb, __shfl_xor_sync(0xffffffffu, mb, o));
    }
  }
}

__device__ __forceinline__ float up(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float up(__half v) { return __half2float(v); }
__device__ __forceinline__ float up(float v) { return v; }
template <class T> __device__ __forceinline__ T down(float f);
template <> __device__ __forceinline__ bf16 down<bf16>(float f) { return __float2bfloat16_rn(f); }
template <> __device__ __forceinline__ __half down<__half>(float f) { return __float2half_rn(f); }
template <> __device__ __forceinline__ float down<float>(float f) { return f; }

// The calling thread's current device has its context bound; allowed while a stream is captured.
static inline bool bind_context() {
  static thread_local int bound = -1;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  if (dev != bound && cudaSetDevice(dev) != cudaSuccess) return false;
  bound = dev;
  return true;
}
// Lets a kernel have its dynamic shared memory, once on each device (the call takes half a microsecond).
template <class F> static bool allow_shared(std::atomic<unsigned long long>& known, F kern, int bytes) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const unsigned long long bit = 1ull << (dev & 63);
  if (dev < 64 && (known.load(std::memory_order_relaxed) & bit)) return true;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
  if (dev < 64) known.fetch_or(bit);
  return true;
}

// Eight consecutive values as they lie in memory.
template <class T> struct alignas(16) Eight { uint4 v[sizeof(T) / 2]; };
template <class T> __device__ __forceinline__ Eight<T> none() {
  Eight<T> e;
#pragma unroll
  for (int i = 0; i < int(sizeof(T)) / 2; ++i) e.v[i] = make_uint4(0, 0, 0, 0);
  return e;
}
// n: how many of them there are (the others come as zero); VEC: on 16-byte boundaries, all or none of them
template <bool VEC, class T> __device__ __forceinline__ Eight<T> fetch(const T* p, int n) {
  Eight<T> e = none<T>();
  if (VEC) {
    if (n > 0) e = *reinterpret_cast<const Eight<T>*>(p);
  } else {
    T* d = reinterpret_cast<T*>(&e);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) d[j] = p[j];
  }
  return e;
}
template <bool VEC, class T> __device__ __forceinline__ void put(T* p, const Eight<T>& e, int n) {
  if (VEC) {
    if (n > 0) *reinterpret_cast<Eight<T>*>(p) = e;
  } else {
    const T* s = reinterpret_cast<const T*>(&e);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = s[j];
  }
}
__device__ __forceinline__ void unpack(const Eight<bf16>& e, float (&f)[8]) {
  const uint32_t w[4] = {e.v[0].x, e.v[0].y, e.v[0].z, e.v[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
__device__ __forceinline__ void unpack(const Eight<__half>& e, float (&f)[8]) {
  const uint32_t w[4] = {e.v[0].x, e.v[0].y, e.v[0].z, e.v[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    f[2 * i] = t.x; f[2 * i + 1] = t.y;
  }
}
__device__ __forceinline__ void unpack(const Eight<float>& e, float (&f)[8]) {
  const uint32_t w[8] = {e.v[0].x, e.v[0].y, e.v[0].z, e.v[0].w, e.v[1].x, e.v[1].y, e.v[1].z, e.v[1].w};
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(w[i]);
}
__device__ __forceinline__ void pairs(const Eight<bf16>& e, f2 (&v)[4]) {
  v[0] = f2_bf(e.v[0].x); v[1] = f2_bf(e.v[0].y); v[2] = f2_bf(e.v[0].z); v[3] = f2_bf(e.v[0].w);
}
template <class T> __device__ __forceinline__ void pairs(const Eight<T>& e, f2 (&v)[4]) {
  float f[8];
  unpack(e, f);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = f2_pack(f[2 * i], f[2 * i + 1]);
}
template <class T> __device__ __forceinline__ Magnitudes<T> magnitudes(const Eight<T>& e) {
  Magnitudes<T> m;
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&e);
#pragma unroll
  for (int i = 0; i < (sizeof(T) == 2 ? 4 : 8); ++i) m.w[i] = w[i] & (sizeof(T) == 2 ? 0x7fff7fffu : 0x7fffffffu);
  return m;
}
__device__ __forceinline__ Magnitudes<float> magnitudes(const f2 (&v)[4]) {
  Magnitudes<float> m;
#pragma unroll
  for (int i = 0; i < 4; ++i) { const float2 t = f2_unpack(v[i]); m.w[2 * i] = magnitude(t.x); m.w[2 * i + 1] = magnitude(t.y); }
  return m;
}
template <class T> __device__ __forceinline__ Eight<T> pack(const float (&f)[8]) {
  Eight<T> e;
  T* d = reinterpret_cast<T*>(&e);
#pragma unroll
  for (int j = 0; j < 8; ++j) d[j] = down<T>(f[j]);
  return e;
}

}  // namespace blk8
}  // namespace sb
