// Activations in 8 bits and back: what a checkpointed block keeps of its input until the backward pass.
//
//   scale = amax / 127 over 128 consecutive values of a row (its last block may be shorter),  q = rint(x * (127 / amax)),  x' = q * scale
//
// |x - x'| is at most amax / 254 and a rounding to x's own type.  The largest magnitude is taken over the bit patterns, where NaN lies above
// infinity: a block that holds one of them has a scale of NaN and comes back as NaN, so that an overflow stays visible.  A block below 1e-30
// comes back as nearly zero.
//
// Bound by memory: 2 + 1 bytes a value for 16-bit types, one pass; a lane has two 16-byte loads on their way.  8192 x 4096 bf16: 18.6 us there and
// 20.2 back (a copy of as many bytes takes 15.5); four loads a lane 19.0 and 24.2, eight 20.4 and 24.1.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "entries.h"

namespace sb {
namespace act8 {

typedef __nv_bfloat16 bf16;
constexpr int BLOCK = 128;               // values that share a scale
constexpr int MAX_D = 0x7fffffff - (BLOCK - 1);          // of a row: the number of its blocks is counted in 32 bits
constexpr float TINY = 1e-30f;

__device__ __forceinline__ float up(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float up(__half v) { return __half2float(v); }
__device__ __forceinline__ float up(float v) { return v; }
__device__ __forceinline__ void down(float f, bf16& v) { v = __float2bfloat16_rn(f); }
__device__ __forceinline__ void down(float f, __half& v) { v = __float2half_rn(f); }
__device__ __forceinline__ void down(float f, float& v) { v = f; }

template <class T, int N> struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Pack { T v[N]; };

__device__ __forceinline__ uint32_t magnitude(float f) { return __float_as_uint(f) & 0x7fffffffu; }
// 127 / amax as the statement in PyTorch's operations rounds it, so that both give the same codes: a value at the border between two codes goes
// to the same side.  NaN stays NaN.
__device__ __forceinline__ float inverse(float amax) { return __fmul_rn(__frcp_rn(amax < TINY ? TINY : amax), 127.f); }
// rint(x * inv), whose magnitude is at most 127, in the low byte: a product of up to 2^22 added to 1.5 * 2^23 is rounded to an integer, half
// to even.  (A conversion instruction for each value ran at a quarter of the rate.)  The product is rounded by itself, as the statement's is: 16-bit values
// often lie halfway between two codes, and there its rounding mostly makes good that of inv, where a fused one would fall to a side by chance.
__device__ __forceinline__ uint32_t code(float x, float inv) { return __float_as_uint(__fadd_rn(__fmul_rn(x, inv), 12582912.f)); }
__device__ __forceinline__ uint32_t four(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// The scale of a block whose largest magnitude has the bits m: NaN for infinity and NaN.
__device__ __forceinline__ float step_of(uint32_t m) { return m < 0x7f800000u ? __uint_as_float(m) / 127.f : __uint_as_float(0x7fffffffu); }
// The four codes of a word as floats: 2^23 + (q + 128) by its bits, from which 2^23 + 128 is taken.
__device__ __forceinline__ void uncode(uint32_t w, float (&f)[4]) {
  w ^= 0x80808080u;
#pragma unroll
  for (int j = 0; j < 4; ++j) f[j] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 + j)) - 8388736.f;
}

// The values that a lane loads at once, their largest magnitude (as fp32 bits) and one by one.
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) { return __vmaxu2(a, b); }
template <class T> struct Eight { uint4 v; };
template <> struct Eight<float> { uint4 v, w; };
__device__ __forceinline__ uint32_t top(const uint4& v) {            // both halves of each word: magnitudes of 16-bit types order as integers
  const uint32_t k = 0x7fff7fffu, m = max_u16x2(max_u16x2(v.x & k, v.y & k), max_u16x2(v.z & k, v.w & k));
  return max(m & 0xffffu, m >> 16);
}
__device__ __forceinline__ uint32_t top(const Eight<bf16>& e) { return top(e.v) << 16; }
__device__ __forceinline__ uint32_t top(const Eight<__half>& e) { return __float_as_uint(__half2float(__ushort_as_half((unsigned short)top(e.v)))); }
__device__ __forceinline__ uint32_t top(const Eight<float>& e) {
  const uint32_t k = 0x7fffffffu;
  return max(max(max(e.v.x & k, e.v.y & k), max(e.v.z & k, e.v.w & k)), max(max(e.w.x & k, e.w.y & k), max(e.w.z & k, e.w.w & k)));
}
__device__ __forceinline__ void values(const Eight<bf16>& e, float (&f)[8]) {
  const uint32_t w[4] = {e.v.x, e.v.y, e.v.z, e.v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
__device__ __forceinline__ void values(const Eight<__half>& e, float (&f)[8]) {
  const uint32_t w[4] = {e.v.x, e.v.y, e.v.z, e.v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    f[2 * i] = t.x; f[2 * i + 1] = t.y;
  }
}
__device__ __forceinline__ void values(const Eight<float>& e, float (&f)[8]) {
  const uint32_t w[8] = {e.v.x, e.v.y, e.v.z, e.v.w, e.w.x, e.w.y, e.w.z, e.w.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(w[i]);
}

// First value of 128-block b, and how many of the block there are.  WHOLE: D % 128 == 0, the blocks lie one behind the other.
struct Rows { uint32_t per_row, D; };
template <bool WHOLE>
__device__ __forceinline__ long long place(long long b, const Rows& r, int& n) {
  n = BLOCK;
  if (WHOLE) return b * BLOCK;
  const long long row = b < 0x80000000LL ? (long long)((uint32_t)b / r.per_row) : b / r.per_row;
  const uint32_t c = uint32_t(b - row * r.per_row) * BLOCK;
  n = min((uint32_t)BLOCK, r.D - c);
  return row * r.D + c;
}

// Eight values a lane, 16 lanes a block, D % 8 == 0 and 16-byte boundaries; U blocks a half-warp, all loaded before the first is used.
template <class T, int U, bool WHOLE>
__global__ void __launch_bounds__(256)
quantize_vec_kernel(const T* __restrict__ x, int8_t* __restrict__ q, float* __restrict__ scale, long long blocks, Rows r) {
  const long long first = ((long long)blockIdx.x * 16 + (threadIdx.x >> 4)) * U;
  const int l = threadIdx.x & 15;
  Eight<T> in[U];
  long long at[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    int n;
    at[u] = place<WHOLE>(first + u, r, n) + l * 8;
    if (first + u >= blocks || l * 8 >= n) at[u] = -1;
    in[u] = Eight<T>{};
    if (at[u] >= 0) in[u] = *reinterpret_cast<const Eight<T>*>(x + at[u]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    uint32_t m = top(in[u]);
#pragma unroll
    for (int o = 8; o; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float inv = inverse(__uint_as_float(m));
    float f[8];
    values(in[u], f);
    uint32_t c[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = code(f[j], inv);
    if (at[u] >= 0) *reinterpret_cast<uint2*>(q + at[u]) = make_uint2(four(c[0], c[1], c[2], c[3]), four(c[4], c[5], c[6], c[7]));
    if (l == 0 && at[u] >= 0) scale[first + u] = step_of(m);
  }
}

// Any width and alignment: a warp a block, four values a lane.
template <class T>
__global__ void __launch_bounds__(256)
quantize_any_kernel(const T* __restrict__ x, int8_t* __restrict__ q, float* __restrict__ scale, long long blocks, Rows r) {
  const long long b = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (b >= blocks) return;
  const int l = threadIdx.x & 31;
  int n;
  const long long at = place<false>(b, r, n);
  float f[4];
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    f[j] = l + 32 * j < n ? up(x[at + l + 32 * j]) : 0.f;
    m = max(m, magnitude(f[j]));
  }
  m = __reduce_max_sync(0xffffffffu, m);
  const float inv = inverse(__uint_as_float(m));
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (l + 32 * j < n) q[at + l + 32 * j] = (int8_t)(uint8_t)code(f[j], inv);
  if (l == 0) scale[b] = step_of(m);
}

// 16 values a lane, eight lanes a block, where the blocks are whole and q lies on a 16-byte boundary, else eight values and 16 lanes.
template <class T, int U, bool WHOLE, int N>
__global__ void __launch_bounds__(256)
dequantize_vec_kernel(const int8_t* __restrict__ q, const float* __restrict__ scale, T* __restrict__ x, long long blocks, Rows r) {
  constexpr int LANES = BLOCK / N;
  const long long first = ((long long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES) * U;
  const int l = threadIdx.x % LANES;
  Pack<uint32_t, N / 4> in[U];
  float s[U];
  long long at[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    int n;
    at[u] = place<WHOLE>(first + u, r, n) + l * N;
    if (first + u >= blocks || l * N >= n) at[u] = -1;
    if (at[u] >= 0) { in[u] = *reinterpret_cast<const Pack<uint32_t, N / 4>*>(q + at[u]); s[u] = scale[first + u]; }
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (at[u] >= 0) {
#pragma unroll
      for (int h = 0; h < N / 8; ++h) {
        float f[8];
        uncode(in[u].v[2 * h], reinterpret_cast<float(&)[4]>(f[0]));
        uncode(in[u].v[2 * h + 1], reinterpret_cast<float(&)[4]>(f[4]));
        Pack<T, 8> out;
#pragma unroll
        for (int j = 0; j < 8; ++j) down(f[j] * s[u], out.v[j]);
        *reinterpret_cast<Pack<T, 8>*>(x + at[u] + 8 * h) = out;
      }
    }
}

template <class T>
__global__ void __launch_bounds__(256)
dequantize_any_kernel(const int8_t* __restrict__ q, const float* __restrict__ scale, T* __restrict__ x, long long blocks, Rows r) {
  const long long b = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (b >= blocks) return;
  int n;
  const long long at = place<false>(b, r, n);
  const float s = scale[b];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int c = (threadIdx.x & 31) + 32 * j;
    if (c < n) down((float)q[at + c] * s, x[at + c]);
  }
}

template <class T>
static int quantize(const void* x, void* q, float* scale, long long rows, int D, bool vec, cudaStream_t st) {
  constexpr int U = 2;
  const Rows r{(uint32_t)((D + BLOCK - 1) / BLOCK), (uint32_t)D};
  const long long blocks = rows * r.per_row, per = vec ? 16 * U : 8, grid = (blocks + per - 1) / per;
  if (grid > 0x7fffffffLL) return -1;
  if (!vec) quantize_any_kernel<T><<<(unsigned)grid, 256, 0, st>>>((const T*)x, (int8_t*)q, scale, blocks, r);
  else if (D % BLOCK == 0) quantize_vec_kernel<T, U, true><<<(unsigned)grid, 256, 0, st>>>((const T*)x, (int8_t*)q, scale, blocks, r);
  else quantize_vec_kernel<T, U, false><<<(unsigned)grid, 256, 0, st>>>((const T*)x, (int8_t*)q, scale, blocks, r);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}
template <class T>
static int dequantize(const void* q, const float* scale, void* x, long long rows, int D, bool vec, cudaStream_t st) {
  constexpr int U = 2;
  const Rows r{(uint32_t)((D + BLOCK - 1) / BLOCK), (uint32_t)D};
  const bool wide = vec && D % BLOCK == 0 && (reinterpret_cast<uintptr_t>(q) & 15) == 0;
  const long long blocks = rows * r.per_row, per = wide ? 32 * U : vec ? 16 * U : 8, grid = (blocks + per - 1) / per;
  if (grid > 0x7fffffffLL) return -1;
  if (wide) dequantize_vec_kernel<T, U, true, 16><<<(unsigned)grid, 256, 0, st>>>((const int8_t*)q, scale, (T*)x, blocks, r);
  else if (vec) dequantize_vec_kernel<T, U, false, 8><<<(unsigned)grid, 256, 0, st>>>((const int8_t*)q, scale, (T*)x, blocks, r);
  else dequantize_any_kernel<T><<<(unsigned)grid, 256, 0, st>>>((const int8_t*)q, scale, (T*)x, blocks, r);
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
  if (rows < 0 || D < 1 || D > MAX_D || type < 0 || type > 2) return -1;
  if (rows == 0) return 0;
  const bool vec = by_vector(x, q, D);
  return type == 0 ? quantize<bf16>(x, q, scale, rows, D, vec, st) : type == 1 ? quantize<__half>(x, q, scale, rows, D, vec, st)
                                                                              : quantize<float>(x, q, scale, rows, D, vec, st);
}
extern "C" int sb_act8_dequantize(const void* q, const float* scale, void* x, long long rows, int D, int type, cudaStream_t st) {
  if (rows < 0 || D < 1 || D > MAX_D || type < 0 || type > 2) return -1;
  if (rows == 0) return 0;
  const bool vec = by_vector(x, q, D);
  return type == 0 ? dequantize<bf16>(q, scale, x, rows, D, vec, st) : type == 1 ? dequantize<__half>(q, scale, x, rows, D, vec, st)
                                                                                : dequantize<float>(q, scale, x, rows, D, vec, st);
}
