// Layer norm over the last dimension, forward and backward, of bf16, fp16 or fp32 rows (statistics and sums in fp32).
//
//   y = (x - mean) rstd w + b,   rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   g = dy w,  xh = (x - mean) rstd:   dx = rstd (g - mean(g) - xh mean(g xh)) (+ gres),   dw = sum over rows of dy xh,   db = sum of dy
//
// The variance is that of the differences from the mean, never the difference of two large sums: a warp takes it around its own mean, and
// warps are joined by  M2 = sum_w M2_w + n_w (mean_w - mean)^2.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "device_info.h"
#include "entries.h"
#include "f32x2.cuh"
#include "pdl.cuh"

namespace sb {
namespace ln {

typedef __nv_bfloat16 bf16;

// What 16 bytes of a type hold, and single values of it.
template <class T> struct Of;
template <> struct Of<bf16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint4& v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
  }
  static __device__ __forceinline__ uint32_t two(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ uint4 put(const float (&f)[8]) {
    return make_uint4(two(f[0], f[1]), two(f[2], f[3]), two(f[4], f[5]), two(f[6], f[7]));
  }
  static __device__ __forceinline__ float one(bf16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ bf16 from(float v) { return __float2bfloat16_rn(v); }
};
template <> struct Of<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint4& v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = t.x; f[2 * i + 1] = t.y;
    }
  }
  static __device__ __forceinline__ uint32_t two(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ uint4 put(const float (&f)[8]) {
    return make_uint4(two(f[0], f[1]), two(f[2], f[3]), two(f[4], f[5]), two(f[6], f[7]));
  }
  static __device__ __forceinline__ float one(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half from(float v) { return __float2half_rn(v); }
};
template <> struct Of<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void get(const uint4& v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ uint4 put(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
  static __device__ __forceinline__ float one(float v) { return v; }
  static __device__ __forceinline__ float from(float v) { return v; }
};

// The same as pairs (f32x2.cuh)
template <class T> __device__ __forceinline__ void get2(const uint4& v, f2 (&f)[Of<T>::N / 2]) {
  float t[Of<T>::N];
  Of<T>::get(v, t);
#pragma unroll
  for (int i = 0; i < Of<T>::N / 2; ++i) f[i] = f2_pack(t[2 * i], t[2 * i + 1]);
}
template <class T> __device__ __forceinline__ uint4 put2(const f2 (&f)[Of<T>::N / 2]) {
  float t[Of<T>::N];
#pragma unroll
  for (int i = 0; i < Of<T>::N / 2; ++i) { const float2 p = f2_unpack(f[i]); t[2 * i] = p.x; t[2 * i + 1] = p.y; }
  return Of<T>::put(t);
}

// Vector or value i of a row: VEC is Of<T>::N (16-byte accesses) or 1 (any width, any alignment).
template <class T, int VEC> __device__ __forceinline__ void load(const T* p, size_t i, float (&f)[VEC]) {
  if constexpr (VEC == 1) f[0] = Of<T>::one(p[i]);
  else Of<T>::get(reinterpret_cast<const uint4*>(p)[i], f);
}
template <class T, int VEC> __device__ __forceinline__ void store(T* p, size_t i, const float (&f)[VEC]) {
  if constexpr (VEC == 1) p[i] = Of<T>::from(f[0]);
  else reinterpret_cast<uint4*>(p)[i] = Of<T>::put(f);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Widths that N = 16 / sizeof(T) does not divide (SHIFT): a row is `head` values up to the next 16-byte boundary, nv vectors, and `tail` values.  The
// single ones, 14 at most, are spread over the lanes of the row's first warp.  Rows that are N (or N / 2, ..: `classes`) apart are cut alike.
// bf16, us, single values throughout -> here: forward 8192 x 1027 22.6 -> 12.3, 8192 x 4095 95 -> 37; backward 45 -> 22.5, 1045 -> 62.  (Whole vectors
// with the neighbours' values masked: 69 and 88 at 8192 x 4095, most of it spent on the two ends.)  In the backward the single values' registers fit
// blocks of 384 threads where a row has no more than 12 warps: 8192 x 3001 63 -> 48, 40000 x 203 with residual 35 -> 25 against 512.
template <class T> struct Cut {
  int head, nv, tail;
  __device__ __forceinline__ Cut(int row, int D) {
    constexpr int N = Of<T>::N;
    const int a = row % N * (D % N) % N;
    head = min((N - a) % N, D);
    nv = (D - head) / N;
    tail = D - head - nv * N;
  }
  __device__ __forceinline__ int single(int lane) const {        // the column of a lane's single value, or -1
    constexpr int N = Of<T>::N;
    return lane < head ? lane : lane >= 16 && lane - 16 < tail ? head + nv * N + lane - 16 : -1;
  }
};

__device__ __forceinline__ uint4 halves(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t e) {
  return make_uint4(__funnelshift_r(a, b, 16), __funnelshift_r(b, c, 16), __funnelshift_r(c, d, 16), __funnelshift_r(d, e, 16));
}
// The N weights from column c on (c + N <= D) out of two vectors of w, which lies on a 16-byte boundary.  `c` is the same modulo N in all lanes.
template <class T> __device__ __forceinline__ uint4 weights_at(const T* w, int c, int D) {
  constexpr int N = Of<T>::N;
  const int k = c / N, e = c - k * N;                    // first vector, values into it
  const uint4 lo = __ldg(reinterpret_cast<const uint4*>(w) + k);
  if (e == 0) return lo;
  uint4 hi;
  if ((k + 2) * N <= D) {
    hi = __ldg(reinterpret_cast<const uint4*>(w) + k + 1);
  } else {                                               // the last vector ends beyond the row
    float t[N];
#pragma unroll
    for (int j = 0; j < N; ++j) t[j] = j < e ? Of<T>::one(w[(k + 1) * N + j]) : 0.f;
    hi = Of<T>::put(t);
  }
  const bool half = sizeof(T) == 2 && (e & 1);           // whole words, then half a one
  switch (e * (int)sizeof(T) / 4) {
    case 0: return halves(lo.x, lo.y, lo.z, lo.w, hi.x);
    case 1: return half ? halves(lo.y, lo.z, lo.w, hi.x, hi.y) : make_uint4(lo.y, lo.z, lo.w, hi.x);
    case 2: return half ? halves(lo.z, lo.w, hi.x, hi.y, hi.z) : make_uint4(lo.z, lo.w, hi.x, hi.y);
    default: return half ? halves(lo.w, hi.x, hi.y, hi.z, hi.w) : make_uint4(lo.w, hi.x, hi.y, hi.z);
  }
}

// ------------------------------------------------------------------------------------ forward
// W warps take a row, V vectors a lane, all loaded before the first sum.  Bound by memory with many rows: 8192 x 4096 bf16 25.1 us (a copy
// takes 22.2); a few rows take the chain load, two sums, barrier, store.
__host__ __device__ constexpr int fwd_rows(int W) { return W == 1 ? 4 : 1; }

template <class T, int VEC, int V, int W, bool SHIFT>
__global__ void __launch_bounds__(32 * W * fwd_rows(W))
fwd_kernel(const T* __restrict__ x, const T* __restrict__ w, const T* __restrict__ b, T* __restrict__ y, float2* __restrict__ stats, int rows,
           int D, float eps) {
  __shared__ float4 red[W];
  const int lane = threadIdx.x & 31, warp = W > 1 ? threadIdx.x >> 5 : 0, i0 = warp * 32 + lane;
  const size_t row = (size_t)blockIdx.x * fwd_rows(W) + threadIdx.x / (32 * W);
  if (row >= (size_t)rows) return;                       // a whole warp of W == 1, never part of a row
  const Cut<T> cut((int)(row % Of<T>::N), D);            // SHIFT
  const int nv = SHIFT ? cut.nv : D / VEC, head = SHIFT ? cut.head : 0;
  const T* src = x + row * D + head;
  const int sc = SHIFT && warp == 0 ? cut.single(lane) : -1;
  float fs = 0.f, gs = 0.f, cs = 0.f;                    // a lane's single value, its weight and bias
  if constexpr (SHIFT) {
    if (sc >= 0) { fs = Of<T>::one(x[row * D + sc]); gs = Of<T>::one(w[sc]); cs = Of<T>::one(b[sc]); }
  }
  // the weights as well where a lane has few of them: a row alone on its SM then waits once
  constexpr bool AHEAD = V * VEC <= 16 && !SHIFT;
  float f[V][VEC], g[AHEAD ? V : 1][VEC], c[AHEAD ? V : 1][VEC];
  int n = 0;                                             // values of this warp
  float s = 0.f;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int i = i0 + 32 * W * v;
    n += min(max(nv - (warp * 32 + 32 * W * v), 0), 32) * VEC;
    if (i < nv) {
      load<T, VEC>(src, i, f[v]);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[v][j] = 0.f;
    }
  }
  if (AHEAD) {
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (i0 + 32 * W * v < nv) { load<T, VEC>(w, i0 + 32 * W * v, g[AHEAD ? v : 0]); load<T, VEC>(b, i0 + 32 * W * v, c[AHEAD ? v : 0]); }
  }
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int j = 0; j < VEC; ++j) s += f[v][j];
  if (SHIFT && warp == 0) { n += cut.head + cut.tail; s += fs; }
  s = warp_sum(s);
  float mean = n ? __fdividef(s, (float)n) : 0.f, m2 = 0.f;
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (i0 + 32 * W * v < nv) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) { const float d = f[v][j] - mean; m2 = fmaf(d, d, m2); }
    }
  if (SHIFT && sc >= 0) m2 = fmaf(fs - mean, fs - mean, m2);
  m2 = warp_sum(m2);
  if (W > 1) {                                           // the warps' results, one a lane: the same sums in every warp
    if (lane == 0) red[warp] = make_float4(s, m2, mean, (float)n);
    __syncthreads();
    const float4 k = red[lane % W];
    mean = k.x;
#pragma unroll
    for (int o = W / 2; o; o >>= 1) mean += __shfl_xor_sync(0xffffffffu, mean, o);
    mean = __fdividef(mean, (float)D);
    const float d = k.z - mean;
    m2 = fmaf(k.w * d, d, k.y);
#pragma unroll
    for (int o = W / 2; o; o >>= 1) m2 += __shfl_xor_sync(0xffffffffu, m2, o);
  }
  const float rstd = rsqrtf(__fdividef(m2, (float)D) + eps);
  if (stats && i0 == 0) stats[row] = make_float2(mean, rstd);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int i = i0 + 32 * W * v;
    if (i < nv) {
      const int k = AHEAD ? v : 0;
      if constexpr (SHIFT) { Of<T>::get(weights_at<T>(w, head + i * VEC, D), g[k]); Of<T>::get(weights_at<T>(b, head + i * VEC, D), c[k]); }
      else if (!AHEAD) { load<T, VEC>(w, i, g[k]); load<T, VEC>(b, i, c[k]); }
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[v][j] = fmaf((f[v][j] - mean) * rstd, g[k][j], c[k][j]);
      store<T, VEC>(y + row * D + head, i, f[v]);
    }
  }
  if constexpr (SHIFT) {
    if (sc >= 0) y[row * D + sc] = Of<T>::from(fmaf((fs - mean) * rstd, gs, cs));
  }
}

// Rows of up to LPR = 8 or 16 vectors: as many lanes a row.  262144 x 64 bf16: 17 us, 58 with a warp a row.
template <class T, int LPR>
__global__ void __launch_bounds__(256)
fwd_narrow_kernel(const T* __restrict__ x, const T* __restrict__ w, const T* __restrict__ b, T* __restrict__ y, float2* __restrict__ stats, int rows,
                  int D, float eps) {
  constexpr int N = Of<T>::N;
  const int i = threadIdx.x % LPR, row = blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  const bool have = row < rows && i < D / N;
  float f[N], g[N], c[N], s = 0.f, m2 = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j) f[j] = g[j] = c[j] = 0.f;
  if (have) {
    load<T, N>(x + (size_t)row * D, i, f);
    load<T, N>(w, i, g);
    load<T, N>(b, i, c);
  }
#pragma unroll
  for (int j = 0; j < N; ++j) s += f[j];
#pragma unroll
  for (int o = LPR / 2; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const float mean = __fdividef(s, (float)D);
#pragma unroll
  for (int j = 0; j < N; ++j) { const float d = have ? f[j] - mean : 0.f; m2 = fmaf(d, d, m2); }
#pragma unroll
  for (int o = LPR / 2; o; o >>= 1) m2 += __shfl_xor_sync(0xffffffffu, m2, o);
  const float rstd = rsqrtf(__fdividef(m2, (float)D) + eps);
  if (!have) return;
  if (stats && i == 0) stats[row] = make_float2(mean, rstd);
#pragma unroll
  for (int j = 0; j < N; ++j) f[j] = fmaf((f[j] - mean) * rstd, g[j], c[j]);
  store<T, N>(y + (size_t)row * D, i, f);
}

// ------------------------------------------------------------------------------------ backward
// A thread owns V vectors of columns and keeps their dw and db sums in registers; W warps share a row, a block holds several such groups
// and walks over the rows.  partial[block] = [dw | db] of the block's rows, added up by reduce_kernel in a fixed order.
//
// SHIFT: a group takes rows of one class, which are cut alike, so that it owns fixed columns all the same, single ones among them.
//
// The rows come through a ring in shared memory, R rows at a time and S of those ahead: a thread copies the 16 bytes of each row and
// tensor that it owns, nobody else reads them, so there is no barrier for them, only the thread's own wait.  8192 x 4096 bf16 with residual:
// 47.2 us with two rows at a time and two of those ahead (a copy of as many bytes takes 42.5), 48.7 with one row, 50.3 with four and none
// ahead; with scalar arithmetic, and x and dy kept in registers over the barrier (which spilled), 79.  Without residual 42.3 (32.3).
constexpr int BWD_THREADS = 512;

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ uint4 take(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}

// Sums of 2 R values over the W warps of a group, the same in all of its threads; `red` [W][2 R] floats of its own for every other call.
template <int R, int W16>
__device__ __forceinline__ void group_sums(float (&s)[2 * R], float* red, int warps, int bar, int wid, int lane) {
  const int W = W16 ? 16 : warps;
  constexpr int P = 2 * R;
  // halves of the values change lanes in the first steps: lane l ends with the warp's sum of value l / (32 / P)
  int o = 16;
#pragma unroll
  for (int n = P / 2; n; n >>= 1, o >>= 1) {
    const bool upper = lane & o;
#pragma unroll
    for (int k = 0; k < n; ++k) {
      const float got = __shfl_xor_sync(0xffffffffu, upper ? s[k] : s[k + n], o);
      s[k] = (upper ? s[k + n] : s[k]) + got;
    }
  }
  for (; o; o >>= 1) s[0] += __shfl_xor_sync(0xffffffffu, s[0], o);
  float t = s[0];
  if (W > 1) {
    constexpr int Q = 32 / P;                            // lanes per value
    if (lane % Q == 0) red[wid * P + lane / Q] = t;
    asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(32 * W) : "memory");
    t = 0.f;
#pragma unroll
    for (int k = 0; k < 16; k += Q) {
      const int at = k + lane % Q;
      if (W16 || at < W) t += red[at * P + lane / Q];
    }
#pragma unroll
    for (int d = Q / 2; d; d >>= 1) t += __shfl_xor_sync(0xffffffffu, t, d);
  }
#pragma unroll
  for (int k = 0; k < P; ++k) s[k] = __shfl_sync(0xffffffffu, t, k * (32 / P));
}

template <class T, int V, int R, int S, bool RES, bool W16, bool SHIFT, int THREADS>
__global__ void __launch_bounds__(THREADS, V == 1 ? 2 : 1)
bwd_kernel(const T* __restrict__ x, const T* __restrict__ w, const T* __restrict__ dy, const float2* __restrict__ stats,
           const T* __restrict__ gres, T* __restrict__ dx, float* __restrict__ partial, int rows, int D, int warps, int classes) {
  const int W = W16 ? 16 : warps;
  constexpr int N = Of<T>::N, NT = RES ? 3 : 2;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float red_all[2][16][2 * R];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, grp = warp / W, wid = warp - grp * W, gl = wid * 32 + lane;
  const int G = (blockDim.x >> 5) / W, group = blockIdx.x * G + grp, groups = gridDim.x * G;
  const int cls = SHIFT ? group % classes : 0;
  const Cut<T> cut(cls, D);
  const int nv = SHIFT ? cut.nv : D / N, head = SHIFT ? cut.head : 0;
  const int live_rows = SHIFT ? (rows - cls + classes - 1) / classes : rows, units = (live_rows + R - 1) / R;
  auto row_of = [&](int i) { return SHIFT ? cls + i * classes : i; };
  const int sc = SHIFT && wid == 0 ? cut.single(lane) : -1;
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + threadIdx.x * 16, part = blockDim.x * 16;
  auto slot = [&](int s, int r, int t, int v) { return ring + (((s * R + r) * NT + t) * V + v) * part; };
  auto fetch = [&](int u, int s) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int i = u * R + r;
      if (u < units && i < live_rows) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          if (gl + 32 * W * v < nv) {
            const size_t o = (size_t)row_of(i) * D + head + (gl + 32 * W * v) * N;
            copy16(slot(s, r, 0, v), x + o);
            copy16(slot(s, r, 1, v), dy + o);
            if (RES) copy16(slot(s, r, 2, v), gres + o);
          }
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  constexpr int M = N / 2;
  f2 wf[V][M], dwa[V][M], dba[V][M];
  const int step = SHIFT ? (groups - cls + classes - 1) / classes : groups;
  int u = SHIFT ? group / classes : group;
#pragma unroll
  for (int s = 0; s < S; ++s) fetch(u + s * step, s);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int i = gl + 32 * W * v;
    if (SHIFT) {
#pragma unroll
      for (int j = 0; j < M; ++j) {
        const int c = head + i * N + 2 * j;
        wf[v][j] = i < nv ? f2_pack(Of<T>::one(w[c]), Of<T>::one(w[c + 1])) : f2(0);
      }
    } else {
      get2<T>(i < nv ? reinterpret_cast<const uint4*>(w)[i] : make_uint4(0, 0, 0, 0), wf[v]);
    }
#pragma unroll
    for (int j = 0; j < M; ++j) dwa[v][j] = dba[v][j] = 0;
  }
  auto row_stats = [&](int un, float2 (&st)[R]) {
#pragma unroll
    for (int r = 0; r < R; ++r) st[r] = un < units && un * R + r < live_rows ? stats[row_of(un * R + r)] : make_float2(0.f, 0.f);
  };
  float2 next[R];                                        // of the next rows: as far away as they are
  row_stats(u, next);
  const float ws = SHIFT && sc >= 0 ? Of<T>::one(w[sc]) : 0.f;
  float dws = 0.f, dbs = 0.f;                            // a lane's single column
  T sx[R], sg[R], sr[R];
  auto singles = [&](int un) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      sx[r] = sg[r] = sr[r] = Of<T>::from(0.f);
      if (SHIFT && sc >= 0 && un < units && un * R + r < live_rows) {
        const size_t o = (size_t)row_of(un * R + r) * D + (unsigned)sc;
        sx[r] = x[o]; sg[r] = dy[o];
        if (RES) sr[r] = gres[o];
      }
    }
  };
  if (SHIFT) singles(u);
  const float inv = 1.f / D;
  int s = 0;
  for (int it = 0; u < units; u += step, ++it) {
    f2 rs[R], off[R];                                    // xh = x rstd - mean rstd
    float rstd[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float m = -next[r].x * next[r].y;
      rstd[r] = next[r].y;
      rs[r] = f2_pack(rstd[r], rstd[r]); off[r] = f2_pack(m, m);
    }
    row_stats(u + step, next);
    asm volatile("cp.async.wait_group %0;" ::"n"(S - 1) : "memory");
    float sums[2 * R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool live = u * R + r < live_rows;
      f2 a = 0, c = 0;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (live && gl + 32 * W * v < nv) {
          f2 xf[M], gf[M];
          get2<T>(take(slot(s, r, 0, v)), xf); get2<T>(take(slot(s, r, 1, v)), gf);
#pragma unroll
          for (int j = 0; j < M; ++j) {
            const f2 xh = f2_fma(xf[j], rs[r], off[r]), g = f2_mul(gf[j], wf[v][j]);
            dwa[v][j] = f2_fma(gf[j], xh, dwa[v][j]);
            dba[v][j] = f2_add(dba[v][j], gf[j]);
            a = f2_add(a, g);
            c = f2_fma(g, xh, c);
          }
        }
      }
      const float2 ta = f2_unpack(a), tc = f2_unpack(c);
      sums[2 * r] = ta.x + ta.y; sums[2 * r + 1] = tc.x + tc.y;
      if (SHIFT && sc >= 0 && live) {
        const float xh = fmaf(Of<T>::one(sx[r]), rstd[r], f2_unpack(off[r]).x), gf = Of<T>::one(sg[r]);
        dws = fmaf(gf, xh, dws);
        dbs += gf;
        sums[2 * r] = fmaf(gf, ws, sums[2 * r]);
        sums[2 * r + 1] = fmaf(gf * ws, xh, sums[2 * r + 1]);
      }
    }
    group_sums<R, W16>(sums, &red_all[it & 1][grp * W][0], W, 1 + grp, wid, lane);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (u * R + r >= live_rows) break;
      const float k1 = -rstd[r] * (sums[2 * r] * inv), k2 = -rstd[r] * (sums[2 * r + 1] * inv);
      const f2 c1 = f2_pack(k1, k1), c2 = f2_pack(k2, k2);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int i = gl + 32 * W * v;
        if (i < nv) {
          f2 xf[M], gf[M];
          get2<T>(take(slot(s, r, 0, v)), xf); get2<T>(take(slot(s, r, 1, v)), gf);
#pragma unroll
          for (int j = 0; j < M; ++j)
            xf[j] = f2_fma(f2_fma(xf[j], rs[r], off[r]), c2, f2_fma(f2_mul(gf[j], wf[v][j]), rs[r], c1));
          if (RES) {
            get2<T>(take(slot(s, r, 2, v)), gf);
#pragma unroll
            for (int j = 0; j < M; ++j) xf[j] = f2_add(xf[j], gf[j]);
          }
          reinterpret_cast<uint4*>(dx + (size_t)row_of(u * R + r) * D + head)[i] = put2<T>(xf);
        }
      }
      if (SHIFT && sc >= 0) {
        const float xh = fmaf(Of<T>::one(sx[r]), rstd[r], f2_unpack(off[r]).x);
        dx[(size_t)row_of(u * R + r) * D + (unsigned)sc] = Of<T>::from(fmaf(xh, k2, fmaf(Of<T>::one(sg[r]) * ws, rstd[r], k1)) + Of<T>::one(sr[r]));
      }
    }
    if (SHIFT) singles(u + step);
    fetch(u + S * step, s);                              // this thread has read the slot that it fills again
    if (++s == S) s = 0;
  }
  // the groups of a block in their order, through the ring, which nothing is copied into any more
  asm volatile("cp.async.wait_all;" ::: "memory");
  float* out = partial + (size_t)blockIdx.x * 2 * D;
  auto put_sums = [&](float* dst) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int i = gl + 32 * W * v;
      if (i < nv) {
#pragma unroll
        for (int j = 0; j < M; ++j) {
          const float2 pw = f2_unpack(dwa[v][j]), pb = f2_unpack(dba[v][j]);
          const int c = head + i * N + 2 * j;
          if (SHIFT) { dst[c] = pw.x; dst[c + 1] = pw.y; dst[D + c] = pb.x; dst[D + c + 1] = pb.y; }
          else { *reinterpret_cast<float2*>(dst + c) = pw; *reinterpret_cast<float2*>(dst + D + c) = pb; }
        }
      }
    }
    if (SHIFT && sc >= 0) { dst[sc] = dws; dst[D + sc] = dbs; }
  };
  if (G == 1) { put_sums(out); return; }
  __syncthreads();
  float* sh = reinterpret_cast<float*>(smem);
  put_sums(sh + (size_t)grp * 2 * D);
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * D; c += blockDim.x) {
    float t = 0.f;
    for (int g = 0; g < G; ++g) t += sh[(size_t)g * 2 * D + c];
    out[c] = t;
  }
}

// Tensors off a 16-byte boundary: a block per row, V single values a thread, the next row's on their way while this one is summed.
template <class T, int V>
__global__ void __launch_bounds__(V > 8 ? 1024 : 256)
bwd_any_kernel(const T* __restrict__ x, const T* __restrict__ w, const T* __restrict__ dy, const float2* __restrict__ stats,
               const T* __restrict__ gres, T* __restrict__ dx, float* __restrict__ partial, int rows, int D) {
  __shared__ float red[2][32][2];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, nw = blockDim.x >> 5;
  float wf[V], dwa[V], dba[V];
  T xn[V], gn[V], rn[V];
  auto fetch = [&](int row) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int i = threadIdx.x + v * blockDim.x;
      if (row < rows && i < D) {
        xn[v] = x[(size_t)row * D + i];
        gn[v] = dy[(size_t)row * D + i];
        if (gres) rn[v] = gres[(size_t)row * D + i];
      }
    }
  };
  int row = blockIdx.x;
  fetch(row);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int i = threadIdx.x + v * blockDim.x;
    wf[v] = i < D ? Of<T>::one(w[i]) : 0.f;
    dwa[v] = dba[v] = 0.f;
  }
  const float inv = 1.f / D;
  for (int it = 0; row < rows; row += gridDim.x, ++it) {
    const float2 st = stats[row];
    float xh[V], g[V], r[V], a = 0.f, c = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const bool have = (int)(threadIdx.x + v * blockDim.x) < D;
      const float gf = have ? Of<T>::one(gn[v]) : 0.f;
      xh[v] = have ? (Of<T>::one(xn[v]) - st.x) * st.y : 0.f;
      r[v] = have && gres ? Of<T>::one(rn[v]) : 0.f;
      g[v] = gf * wf[v];
      dwa[v] = fmaf(gf, xh[v], dwa[v]);
      dba[v] += gf;
      a += g[v];
      c = fmaf(g[v], xh[v], c);
    }
    fetch(row + gridDim.x);
    a = warp_sum(a); c = warp_sum(c);
    if (lane == 0) { red[it & 1][wid][0] = a; red[it & 1][wid][1] = c; }
    __syncthreads();
    a = warp_sum(lane < nw ? red[it & 1][lane][0] : 0.f) * inv;
    c = warp_sum(lane < nw ? red[it & 1][lane][1] : 0.f) * inv;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int i = threadIdx.x + v * blockDim.x;
      if (i < D) dx[(size_t)row * D + i] = Of<T>::from(st.y * (g[v] - a - xh[v] * c) + r[v]);
    }
  }
  float* out = partial + (size_t)blockIdx.x * 2 * D;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int i = threadIdx.x + v * blockDim.x;
    if (i < D) { out[i] = dwa[v]; out[D + i] = dba[v]; }
  }
}

// dw, db = sum over the blocks of partial [nblk][2][D]: a block takes 32 columns, its 32 thread rows split the partial rows.
template <class T>
__global__ void __launch_bounds__(1024)
reduce_kernel(const float* partial, T* dw, T* db, int nblk, int D) {
  __shared__ float sh[32][33];
  const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5, c = blockIdx.x * 32 + cx;
  wait_for_previous();
  float s = 0.f;
  if (c < 2 * D) {
#pragma unroll 4
    for (int k = ry; k < nblk; k += 32) s += partial[(size_t)k * 2 * D + c];
  }
  sh[ry][cx] = s;
  __syncthreads();
  const float t = warp_sum(sh[cx][ry]);                  // column ry of this block, its 32 parts over the lanes
  const int o = blockIdx.x * 32 + ry;
  if (cx == 0 && o < 2 * D) (o < D ? dw[o] : db[o - D]) = Of<T>::from(t);
}

// ------------------------------------------------------------------------------------ launchers
constexpr int MAX_D = 16384, MAX_ROWS = 1 << 30;

template <class T, int VEC, int V, int W, bool SHIFT = false>
static int launch_fwd(const void* x, const void* w, const void* b, void* y, float* stats, int rows, int D, float eps, cudaStream_t st) {
  const int per = fwd_rows(W);
  fwd_kernel<T, VEC, V, W, SHIFT><<<(rows + per - 1) / per, 32 * W * per, 0, st>>>((const T*)x, (const T*)w, (const T*)b, (T*)y, (float2*)stats, rows, D, eps);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

template <class T, int VEC>
static int forward(const void* x, const void* w, const void* b, void* y, float* stats, int rows, int D, float eps, cudaStream_t st) {
  // A warp alone on a row has no barrier and the fewest sums to join, and with many rows that is what counts; with few rows on an SM a row is
  // spread so that its loads and its sums are short.  us, more vectors a lane / fewer (bf16): D = 1024 200 rows 2.97 / 2.37, 8192 rows 8.6 / 12.4;
  // D = 2048 1000 rows 3.8 / 3.2, 4000 rows 8.8 / 10.8; D = 4096 200 rows 3.3 / 3.0, 1000 rows 5.4 / 7.8; D = 8192 8 rows 3.3 / 3.0, 200 rows
  // 3.7 / 4.5; D = 16384 1000 rows 17.9 / 17.3, 4000 rows 51.2 / 52.1.  Single values: D = 1027, 8192 rows 24.3 with 8 x 8, 26.9 with 16 x 4,
  // 34.9 with 4 x 16.
  const int lanes = (D / VEC + 31) / 32;                 // warps that hold a row with one vector a lane
  const int per_sm = (rows + num_sms() - 1) / num_sms();
#define LN_FWD(V, W) return launch_fwd<T, VEC, V, W>(x, w, b, y, stats, rows, D, eps, st)
  if constexpr (VEC == 1) {
    if (lanes <= 4) LN_FWD(4, 1);
    if (lanes <= 8) LN_FWD(8, 1);
    if (lanes <= 16) LN_FWD(8, 2);
    if (lanes <= 32) LN_FWD(8, 4);
    if (lanes <= 64) LN_FWD(8, 8);
    if (lanes <= 128) LN_FWD(16, 8);
    if (lanes <= 256) LN_FWD(8, 32);
    LN_FWD(16, 32);
  } else {
    if (D / VEC <= 16) {
      auto* kernel = D / VEC <= 8 ? fwd_narrow_kernel<T, 8> : fwd_narrow_kernel<T, 16>;
      const int per = D / VEC <= 8 ? 32 : 16;
      kernel<<<(rows + per - 1) / per, 256, 0, st>>>((const T*)x, (const T*)w, (const T*)b, (T*)y, (float2*)stats, rows, D, eps);
      return cudaGetLastError() == cudaSuccess ? 0 : -2;
    }
    if (lanes <= 1) LN_FWD(1, 1);
    if (lanes <= 2) { if (per_sm <= 4) LN_FWD(1, 2); LN_FWD(2, 1); }
    if (lanes <= 4) { if (per_sm <= 7) LN_FWD(1, 4); LN_FWD(4, 1); }
    if (lanes <= 8) { if (per_sm <= 7) LN_FWD(2, 4); LN_FWD(4, 2); }
    if (lanes <= 16) { if (per_sm <= 2) LN_FWD(2, 8); LN_FWD(4, 4); }
    if (lanes <= 32) { if (per_sm <= 1) LN_FWD(2, 16); LN_FWD(4, 8); }
    if (lanes <= 64) { if (per_sm <= 7) LN_FWD(4, 16); LN_FWD(8, 8); }
    LN_FWD(8, 16);
  }
#undef LN_FWD
}

struct Plan { int W, V, threads, grid, classes; };
// Groups of warps a row by vectors of n values.
static Plan plan_vec(int rows, int D, int n) {
  Plan p;
  p.classes = D % n == 0 ? 1 : D % 2 ? n : D % 4 ? n / 2 : 2;
  const int lanes = D < n ? 1 : (D / n + 31) / 32;       // 1 .. 128
  p.V = lanes <= 16 ? 1 : lanes <= 32 ? 2 : lanes <= 64 ? 4 : 8;
  p.W = p.V == 1 ? lanes : 16;
  const int G = p.V > 1 ? 1 : p.classes > 1 && p.W <= 12 ? 12 / p.W : 16 / p.W, R = p.V <= 2 ? 2 : 1;      // 384 threads have registers for the single values
  p.threads = 32 * p.W * G;
  const int units = (rows + R - 1) / R, blocks = (units + G - 1) / G, most = (p.V == 1 ? 2 : 1) * num_sms(), least = (p.classes + G - 1) / G;
  p.grid = blocks < most ? blocks : most;
  if (p.grid < least) p.grid = least;                    // a group for every class
  return p;
}
static Plan plan_any(int rows, int D) {
  Plan p;
  p.threads = D <= 2048 ? 256 : 1024;
  const int v = (D + p.threads - 1) / p.threads;
  p.V = p.threads == 256 ? (v <= 2 ? 2 : v <= 4 ? 4 : 8) : 16;
  p.W = p.threads / 32;
  const int most = (p.threads == 256 ? 4 : 1) * num_sms();
  p.grid = rows < most ? rows : most;
  return p;
}

template <class T>
static int forward_shift(const void* x, const void* w, const void* b, void* y, float* stats, int rows, int D, float eps, cudaStream_t st) {
  constexpr int N = Of<T>::N;
  const int lanes = (D / N + 31) / 32;
#define LN_FWD(V, W) if (lanes <= V * W) return launch_fwd<T, N, V, W, true>(x, w, b, y, stats, rows, D, eps, st)
  LN_FWD(1, 1); LN_FWD(2, 1); LN_FWD(3, 1); LN_FWD(4, 1);
  LN_FWD(3, 2); LN_FWD(4, 2);
  LN_FWD(3, 4); LN_FWD(4, 4);
  LN_FWD(3, 8); LN_FWD(4, 8);
  LN_FWD(3, 16); LN_FWD(4, 16);
  if constexpr (N == 4) LN_FWD(8, 16);
#undef LN_FWD
  return -3;
}

template <class T, int V, int R, int S, bool RES, bool W16, bool SHIFT, int THREADS = BWD_THREADS>
static int launch_bwd(const Plan& p, const void* x, const void* w, const void* dy, const float* stats, const void* gres, void* dx, float* partial,
                      int rows, int D, cudaStream_t st) {
  const int ring = S * R * (RES ? 3 : 2) * V * p.threads * 16;
  if (ring > 40 * 1024 && cudaFuncSetAttribute(bwd_kernel<T, V, R, S, RES, W16, SHIFT, THREADS>, cudaFuncAttributeMaxDynamicSharedMemorySize, ring) != cudaSuccess) return -2;
  bwd_kernel<T, V, R, S, RES, W16, SHIFT, THREADS><<<p.grid, p.threads, ring, st>>>((const T*)x, (const T*)w, (const T*)dy, (const float2*)stats, (const T*)gres, (T*)dx,
                                                               partial, rows, D, p.W, p.classes);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

template <class T>
static int backward(const void* x, const void* w, const void* dy, const float* stats, const void* gres, void* dx, void* dw, void* db, float* partial,
                    int rows, int D, bool vec, cudaStream_t st) {
  const Plan p = vec ? plan_vec(rows, D, Of<T>::N) : plan_any(rows, D);
  int rc = 0;
#define LN_ARGS p, x, w, dy, stats, gres, dx, partial, rows, D, st
#define LN_BWD(V, R, S, W16)                                                                                                              \
  rc = p.classes == 1 ? (gres ? launch_bwd<T, V, R, S, true, W16, false>(LN_ARGS) : launch_bwd<T, V, R, S, false, W16, false>(LN_ARGS)) \
                      : (gres ? launch_bwd<T, V, R, S, true, W16, true>(LN_ARGS) : launch_bwd<T, V, R, S, false, W16, true>(LN_ARGS))
#define LN_ANY(V) bwd_any_kernel<T, V><<<p.grid, p.threads, 0, st>>>((const T*)x, (const T*)w, (const T*)dy, (const float2*)stats, (const T*)gres, \
                                                                     (T*)dx, partial, rows, D)
  if (rows > 0) {
    if (vec) {
      if (p.V == 1 && p.W == 16) LN_BWD(1, 2, 2, true);
      else if (p.V == 1 && p.threads <= 384 && p.classes > 1)
        rc = gres ? launch_bwd<T, 1, 2, 2, true, false, true, 384>(LN_ARGS) : launch_bwd<T, 1, 2, 2, false, false, true, 384>(LN_ARGS);
      else if (p.V == 1) LN_BWD(1, 2, 2, false);
      else if (p.V == 2) LN_BWD(2, 2, 2, true);
      else if (p.V == 4) LN_BWD(4, 1, 2, true);
      else if constexpr (Of<T>::N == 4) LN_BWD(8, 1, 1, true);
      else return -3;
      if (rc) return rc;
    } else {
      if (p.V == 2) LN_ANY(2);
      else if (p.V == 4) LN_ANY(4);
      else if (p.V == 8) LN_ANY(8);
      else LN_ANY(16);
      if (cudaGetLastError() != cudaSuccess) return -2;
    }
  }
#undef LN_ARGS
#undef LN_BWD
#undef LN_ANY
  return launch_chained(false, reduce_kernel<T>, dim3((2 * D + 31) / 32), 1024, 0, st, (const float*)partial, (T*)dw, (T*)db, rows > 0 ? p.grid : 0, D);
}

static bool on16(std::initializer_list<const void*> ps) {
  uintptr_t a = 0;
  for (const void* p : ps) a |= reinterpret_cast<uintptr_t>(p);
  return (a & 15) == 0;
}

}  // namespace ln
}  // namespace sb

using namespace sb::ln;

// x, y [rows, D], w and b [D] of one type (0: bf16, 1: fp16, 2: fp32); stats [rows, 2] fp32 (mean, rstd) for the backward, or null.
extern "C" int sb_layernorm_fwd(const void* x, const void* w, const void* b, void* y, float* stats, int rows, int D, float eps, int type,
                                cudaStream_t st) {
  if (D < 1 || D > MAX_D || rows < 0 || rows > MAX_ROWS || type < 0 || type > 2) return -1;
  if (rows == 0) return 0;
  const int n = type == 2 ? 4 : 8;
  const bool vec = D % n == 0 && on16({x, w, b, y}), shift = D % n != 0 && on16({x, w, b, y});
  if (shift) return type == 0   ? forward_shift<bf16>(x, w, b, y, stats, rows, D, eps, st)
                    : type == 1 ? forward_shift<__half>(x, w, b, y, stats, rows, D, eps, st)
                                : forward_shift<float>(x, w, b, y, stats, rows, D, eps, st);
  if (type == 0) return vec ? forward<bf16, 8>(x, w, b, y, stats, rows, D, eps, st) : forward<bf16, 1>(x, w, b, y, stats, rows, D, eps, st);
  if (type == 1) return vec ? forward<__half, 8>(x, w, b, y, stats, rows, D, eps, st) : forward<__half, 1>(x, w, b, y, stats, rows, D, eps, st);
  return vec ? forward<float, 4>(x, w, b, y, stats, rows, D, eps, st) : forward<float, 1>(x, w, b, y, stats, rows, D, eps, st);
}

// Rows of 2 D floats that sb_layernorm_bwd needs as scratch.
extern "C" int sb_layernorm_bwd_blocks(int rows, int D, int type) {
  if (rows <= 0 || D < 1) return 1;
  const int n = type == 2 ? 4 : 8, any = plan_any(rows, D).grid, vec = plan_vec(rows, D, n).grid;
  return vec > any ? vec : any;
}

// dx [rows, D] (gres, the gradient that came along the residual branch, added; may be null), dw and db [D], written.  Two launches.
extern "C" int sb_layernorm_bwd(const void* x, const void* w, const void* dy, const float* stats, const void* gres, void* dx, void* dw, void* db,
                                float* partial, int rows, int D, int type, cudaStream_t st) {
  if (D < 1 || D > MAX_D || rows < 0 || rows > MAX_ROWS || type < 0 || type > 2) return -1;
  const int n = type == 2 ? 4 : 8;
  const bool vec = on16({x, dy, gres, dx}) && (D % n || on16({w}));
  if (type == 0) return backward<bf16>(x, w, dy, stats, gres, dx, dw, db, partial, rows, D, vec, st);
  if (type == 1) return backward<__half>(x, w, dy, stats, gres, dx, dw, db, partial, rows, D, vec, st);
  return backward<float>(x, w, dy, stats, gres, dx, dw, db, partial, rows, D, vec, st);
}
