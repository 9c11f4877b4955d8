// Activations in 8 bits and back: what a checkpointed block keeps of its input until the backward pass.
//
//   scale = amax / 127 over 128 consecutive values of a row (its last block may be shorter),  q = rint(x * (127 / amax)),  x' = q * scale
//
// |x - x'| is at most amax / 254 and a rounding to x's own type.  The largest magnitude is taken over the bit patterns, where NaN lies above
// infinity: a block that holds one of them gets such a scale and comes back as NaN, so that an overflow stays visible.  A block below 1e-30
// comes back as nearly zero.
//
// Bound by memory: 2 + 1 bytes a value for 16-bit types, one pass; a lane has four 16-byte loads on their way.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "entries.h"

namespace sb {
namespace act8 {

typedef __nv_bfloat16 bf16;
constexpr int BLOCK = 128;               // values that share a scale
constexpr float TINY = 1e-30f;

__device__ __forceinline__ float up(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float up(__half v) { return __half2float(v); }
__device__ __forceinline__ float up(float v) { return v; }
__device__ __forceinline__ void down(float f, bf16& v) { v = __float2bfloat16_rn(f); }
__device__ __forceinline__ void down(float f, __half& v) { v = __float2half_rn(f); }
__device__ __forceinline__ void down(float f, float& v) { v = f; }

template <class T, int N> struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Pack { T v[N]; };

__device__ __forceinline__ uint32_t magnitude(float f) { return __float_as_uint(f) & 0x7fffffffu; }
__device__ __forceinline__ float inverse(float amax) { return 127.f / (amax < TINY ? TINY : amax); }     // NaN stays NaN
__device__ __forceinline__ int8_t code(float x, float inv) {
  const float r = rintf(x * inv);
  return (int8_t)(r >= 127.f ? 127 : r <= -127.f ? -127 : r == r ? (int)r : 0);
}

// Eight values a lane, 16 lanes a block, D % 8 == 0 and 16-byte boundaries; U blocks a half-warp, all loaded before the first is used.
template <class T, int U>
__global__ void __launch_bounds__(256)
quantize_vec_kernel(const T* __restrict__ x, int8_t* __restrict__ q, float* __restrict__ scale, long long blocks, int per_row, int D) {
  const long long first = ((long long)blockIdx.x * 16 + (threadIdx.x >> 4)) * U;
  const int l = threadIdx.x & 15;
  Pack<T, 8> in[U];
  long long at[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long b = first + u, row = b / per_row;
    const int c = int(b - row * per_row) * BLOCK + l * 8;
    at[u] = b < blocks && c < D ? row * D + c : -1;
    if (at[u] >= 0) in[u] = *reinterpret_cast<const Pack<T, 8>*>(x + at[u]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float f[8];
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) { f[j] = at[u] >= 0 ? up(in[u].v[j]) : 0.f; m = max(m, magnitude(f[j])); }
#pragma unroll
    for (int o = 8; o; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float amax = __uint_as_float(m), inv = inverse(amax);
    Pack<int8_t, 8> out;
#pragma unroll
    for (int j = 0; j < 8; ++j) out.v[j] = code(f[j], inv);
    if (at[u] >= 0) *reinterpret_cast<Pack<int8_t, 8>*>(q + at[u]) = out;
    if (l == 0 && first + u < blocks) scale[first + u] = amax / 127.f;
  }
}

// Any width and alignment: a warp a block, four values a lane.
template <class T>
__global__ void __launch_bounds__(256)
quantize_any_kernel(const T* __restrict__ x, int8_t* __restrict__ q, float* __restrict__ scale, long long blocks, int per_row, int D) {
  const long long b = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (b >= blocks) return;
  const int l = threadIdx.x & 31;
  const long long row = b / per_row;
  const int c0 = int(b - row * per_row) * BLOCK;
  float f[4];
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int c = c0 + l + 32 * j;
    f[j] = c < D ? up(x[row * D + c]) : 0.f;
    m = max(m, magnitude(f[j]));
  }
  m = __reduce_max_sync(0xffffffffu, m);
  const float amax = __uint_as_float(m), inv = inverse(amax);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int c = c0 + l + 32 * j;
    if (c < D) q[row * D + c] = code(f[j], inv);
  }
  if (l == 0) scale[b] = amax / 127.f;
}

template <class T, int U>
__global__ void __launch_bounds__(256)
dequantize_vec_kernel(const int8_t* __restrict__ q, const float* __restrict__ scale, T* __restrict__ x, long long blocks, int per_row, int D) {
  const long long first = ((long long)blockIdx.x * 16 + (threadIdx.x >> 4)) * U;
  const int l = threadIdx.x & 15;
  Pack<int8_t, 8> in[U];
  float s[U];
  long long at[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long b = first + u, row = b / per_row;
    const int c = int(b - row * per_row) * BLOCK + l * 8;
    at[u] = b < blocks && c < D ? row * D + c : -1;
    if (at[u] >= 0) { in[u] = *reinterpret_cast<const Pack<int8_t, 8>*>(q + at[u]); s[u] = scale[b]; }
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (at[u] >= 0) {
      Pack<T, 8> out;
#pragma unroll
      for (int j = 0; j < 8; ++j) down((float)in[u].v[j] * s[u], out.v[j]);
      *reinterpret_cast<Pack<T, 8>*>(x + at[u]) = out;
    }
}

template <class T>
__global__ void __launch_bounds__(256)
dequantize_any_kernel(const int8_t* __restrict__ q, const float* __restrict__ scale, T* __restrict__ x, long long blocks, int per_row, int D) {
  const long long b = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (b >= blocks) return;
  const long long row = b / per_row;
  const int c0 = int(b - row * per_row) * BLOCK;
  const float s = scale[b];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int c = c0 + (threadIdx.x & 31) + 32 * j;
    if (c < D) down((float)q[row * D + c] * s, x[row * D + c]);
  }
}

constexpr int U = 4;

template <class T>
static int quantize(const void* x, void* q, float* scale, long long rows, int D, bool vec, cudaStream_t st) {
  const int per = (D + BLOCK - 1) / BLOCK;
  const long long blocks = rows * per, grid = vec ? (blocks + 16 * U - 1) / (16 * U) : (blocks + 7) / 8;
  if (grid > 0x7fffffffLL) return -1;
  if (vec) quantize_vec_kernel<T, U><<<(unsigned)grid, 256, 0, st>>>((const T*)x, (int8_t*)q, scale, blocks, per, D);
  else quantize_any_kernel<T><<<(unsigned)grid, 256, 0, st>>>((const T*)x, (int8_t*)q, scale, blocks, per, D);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}
template <class T>
static int dequantize(const void* q, const float* scale, void* x, long long rows, int D, bool vec, cudaStream_t st) {
  const int per = (D + BLOCK - 1) / BLOCK;
  const long long blocks = rows * per, grid = vec ? (blocks + 16 * U - 1) / (16 * U) : (blocks + 7) / 8;
  if (grid > 0x7fffffffLL) return -1;
  if (vec) dequantize_vec_kernel<T, U><<<(unsigned)grid, 256, 0, st>>>((const int8_t*)q, scale, (T*)x, blocks, per, D);
  else dequantize_any_kernel<T><<<(unsigned)grid, 256, 0, st>>>((const int8_t*)q, scale, (T*)x, blocks, per, D);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}
static bool by_vector(const void* x, const void* q, int D) {
  return D % 8 == 0 && ((reinterpret_cast<uintptr_t>(x) & 15) | (reinterpret_cast<uintptr_t>(q) & 7)) == 0;
}

}  // namespace act8
}  // namespace sb

using namespace sb::act8;

// x [rows, D] of type 0 (bf16), 1 (fp16) or 2 (fp32) -> q [rows, D] int8 and scale [rows, ceil(D / 128)] fp32.
extern "C" int sb_act8_quantize(const void* x, void* q, float* scale, long long rows, int D, int type, cudaStream_t st) {
  if (rows < 0 || D < 1 || type < 0 || type > 2) return -1;
  if (rows == 0) return 0;
  const bool vec = by_vector(x, q, D);
  return type == 0 ? quantize<bf16>(x, q, scale, rows, D, vec, st) : type == 1 ? quantize<__half>(x, q, scale, rows, D, vec, st)
                                                                              : quantize<float>(x, q, scale, rows, D, vec, st);
}
extern "C" int sb_act8_dequantize(const void* q, const float* scale, void* x, long long rows, int D, int type, cudaStream_t st) {
  if (rows < 0 || D < 1 || type < 0 || type > 2) return -1;
  if (rows == 0) return 0;
  const bool vec = by_vector(x, q, D);
  return type == 0 ? dequantize<bf16>(q, scale, x, rows, D, vec, st) : type == 1 ? dequantize<__half>(q, scale, x, rows, D, vec, st)
                                                                                : dequantize<float>(q, scale, x, rows, D, vec, st);
}
