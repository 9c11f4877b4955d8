// Operands of the block-scaled 8-bit products (gemm_fp8_block.cu) from 16- or 32-bit tensors, and back:
//
//   quantise   x [R, C] -> e4m3 with a scale for 128 values of a row, of a column, of both (two forms from one read), or of a 128 x 128 tile
//   norm       s = x + residual;  y = s / rms(s) * g  -> e4m3 with a scale for 128 values of a row; y itself is never rounded to 16 bits
//   dequantise
//
// Layouts.  Codes keep the shape of x; their rows are `ldq` bytes apart (a multiple of 16, what the tensor-core product's loads need).
// Scales lie with the direction that the product does not contract contiguous: [C / 128][R] for rows, [R / 128][C] for columns, both with the inner
// dimension rounded up to fours (the product fetches those of 128 neighbouring rows in copies of 16 bytes), [R / 128][C / 128] for tiles.
// Bound by memory, and where both forms are written by the instructions for them (some 20 a value).  us for bf16, in brackets those of a copy of as many
// bytes: 8192 x 12288 rows 51 (46), columns 55 (46), both 89 (62), tiles 47 (46); norm with residual 8192 x 4096 39 (36), its backward 58 (51), back to
// 16 bits 18 (15).  Of fp32, whose instances spill some 100 to 250 bytes: 8192 x 4096 rows 41 (27), columns 42 (27), both 50 (32), tiles 41 (27).
#include <type_traits>

#include "device_info.h"
#include "entries.h"
#include "fp8_block.cuh"
#include "pdl.cuh"

namespace sb {
namespace blk8 {

__host__ __device__ inline long long fours(long long n) { return (n + 3) / 4 * 4; }

// These kernels are programmatic dependents of whatever is before them (pdl.cuh, the second kind) and let the next one start once all that is
// complete: the product for few tokens, which follows, may then read weights ahead as the link of a chain behind an ordinary launch.
__device__ __forceinline__ void begin() {
  wait_for_previous();
  let_next_start();
}

// ------------------------------------------------------------------------------------------------ tiles of 128 x 128
// A block holds a tile in registers: sixteen threads eight columns each, eight rows a thread (four where both forms are written), all loads issued before
// the first value is used.  From there a row's largest magnitude is four shuffles away and a column's one exchange through shared memory, so the
// second form of the codes costs its writes alone.
struct QuantArgs {
  const void* x;
  long long ld, R;
  int C;
  long long ldq;                   // of both forms
  uint8_t* q_rows;                 // scales of rows, or of tiles
  float* s_rows;
  uint8_t* q_cols;
  float* s_cols;
  const float* a;                  // NORM: x * a[row] * g[column] is quantised
  const void* g;
  float* sums;                     // [R / 128][C] sums of x over a tile's rows (a bias gradient), or null
  long long col_tiles;
};

enum { ROWS = 1, COLS = 2, TILE = 4 };

// Threads of a block: with both forms, or a norm in front, half as many rows a thread, whose values and codes would otherwise leave room for two
// blocks on an SM.
__host__ __device__ constexpr int quant_threads(int form, bool norm) { return form == (ROWS | COLS) || norm ? 512 : 256; }
// Blocks of an SM that the registers are cut for: 64 a thread where one form is written, 80 for columns.
__host__ __device__ constexpr int quant_blocks(int form, bool norm) { return quant_threads(form, norm) == 512 ? 2 : form == COLS ? 3 : 4; }
template <class T, int FORM, bool NORM, bool VEC>
__global__ void __launch_bounds__(quant_threads(FORM, NORM), quant_blocks(FORM, NORM))
quantize_kernel(QuantArgs p) {
  constexpr int THREADS = quant_threads(FORM, NORM), HALVES = THREADS / 16, WARPS = THREADS / 32, RPT = BLOCK / HALVES;
  typedef typename std::conditional<NORM, float, T>::type M;          // what magnitudes are compared in
  constexpr int MW = sizeof(M) == 2 ? 4 : 8;
  __shared__ uint32_t part[WARPS][16][MW];                      // columns' largest magnitudes by warp
  __shared__ float sum_part[WARPS][BLOCK];
  __shared__ float row_scale[BLOCK];
  __shared__ uint32_t col_max[BLOCK];                       // tiles: by warp
  __shared__ __align__(16) float col_inv[BLOCK], col_minus[BLOCK];
  begin();
  const long long tile_r = blockIdx.x / p.col_tiles, tile_c = blockIdx.x - tile_r * p.col_tiles;
  const int l = threadIdx.x & 15, h = threadIdx.x >> 4, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long r0 = tile_r * BLOCK;
  const int c0 = int(tile_c) * BLOCK + l * 8;
  const int n = min(8, p.C - c0);                           // of the thread's columns
  const int rows = int(min((long long)BLOCK, p.R - r0));
  const T* x = static_cast<const T*>(p.x) + r0 * p.ld + c0;
  Eight<T> raw[RPT];
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int r = h + HALVES * i;
    raw[i] = fetch<VEC, T>(x + r * p.ld, r < rows ? n : 0);
  }
  f2 g[4];
  float a[RPT];
  if (NORM) {
    pairs(fetch<VEC, T>(static_cast<const T*>(p.g) + c0, n), g);
#pragma unroll
    for (int i = 0; i < RPT; ++i) a[i] = h + HALVES * i < rows ? p.a[r0 + h + HALVES * i] : 0.f;
  }
  auto values = [&](int i, f2 (&v)[4]) {
    pairs(raw[i], v);
    if (NORM) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = f2_mul(f2_mul(v[j], f2_pack(a[i], a[i])), g[j]);
    }
  };
  auto sizes = [&](int i) {
    if constexpr (NORM) {
      f2 v[4];
      values(i, v);
      return magnitudes(v);
    } else {
      return magnitudes(raw[i]);
    }
  };
  Magnitudes<M> most = {};                                  // of the thread's columns
  f2 cs[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
  for (int i = 0; i < RPT; i += 2) {
    const Magnitudes<M> m[2] = {sizes(i), sizes(i + 1)};
    if (FORM & (COLS | TILE)) {
#pragma unroll
      for (int j = 0; j < MW; ++j) most.w[j] = max_of<M>(most.w[j], max_of<M>(m[0].w[j], m[1].w[j]));
    }
    if ((FORM & COLS) && p.sums) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        f2 v[4];
        values(i + k, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) cs[j] = f2_add(cs[j], v[j]);
      }
    }
    if (FORM & ROWS) {
      uint32_t top[2];
      largest_of_rows(m[0], m[1], top[0], top[1]);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        // rows alone: the rounded reciprocal's branch keeps the rows' instructions apart, 8192 x 12288 in 51 us instead of 58; beside columns it costs
        // (103 instead of 89)
        const Coder c(top[k], FORM == ROWS);
        const int r = h + HALVES * (i + k);
        f2 v[4];
        values(i + k, v);
        if (r < rows && n > 0) *reinterpret_cast<uint2*>(p.q_rows + (r0 + r) * p.ldq + c0) = encode(c, v);
        if (l == 0) row_scale[r] = c.scale;
      }
    }
  }
  if (FORM & TILE) {
    uint32_t top = largest(most);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) col_max[warp] = top;
  }
  if (FORM & COLS) {
#pragma unroll
    for (int j = 0; j < MW; ++j) most.w[j] = max_of<M>(most.w[j], __shfl_xor_sync(0xffffffffu, most.w[j], 16));
    if (lane < 16) {
#pragma unroll
      for (int j = 0; j < MW; ++j) part[warp][l][j] = most.w[j];
    }
    if (p.sums) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 t = f2_unpack(cs[j]);
        const float u = t.x + __shfl_xor_sync(0xffffffffu, t.x, 16), v = t.y + __shfl_xor_sync(0xffffffffu, t.y, 16);
        if (lane < 16) { sum_part[warp][l * 8 + 2 * j] = u; sum_part[warp][l * 8 + 2 * j + 1] = v; }
      }
    }
  }
  __syncthreads();
  if ((FORM & ROWS) && threadIdx.x < rows) p.s_rows[tile_c * fours(p.R) + r0 + threadIdx.x] = row_scale[threadIdx.x];
  if (FORM & TILE) {
    uint32_t top = col_max[0];
#pragma unroll
    for (int k = 1; k < WARPS; ++k) top = max(top, col_max[k]);
    const Coder c(top);
    if (threadIdx.x == 0) p.s_rows[blockIdx.x] = c.scale;
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      const int r = h + HALVES * i;
      f2 v[4];
      values(i, v);
      if (r < rows && n > 0) *reinterpret_cast<uint2*>(p.q_rows + (r0 + r) * p.ldq + c0) = encode(c, v);
    }
  }
  if (FORM & COLS) {
    if (threadIdx.x < BLOCK) {                              // a column a thread
      const int who = threadIdx.x >> 3, j = threadIdx.x & 7;
      uint32_t top = 0;
#pragma unroll
      for (int k = 0; k < WARPS; ++k) {
        const uint32_t w = part[k][who][sizeof(M) == 2 ? j >> 1 : j];
        top = max(top, sizeof(M) == 2 ? (j & 1 ? w >> 16 : w & 0xffffu) : w);
      }
      const Coder coder(widen<M>(top));
      col_inv[threadIdx.x] = coder.inv;
      col_minus[threadIdx.x] = coder.minus_amax;
      const long long c = tile_c * BLOCK + threadIdx.x;
      if (c < p.C) {
        p.s_cols[tile_r * fours(p.C) + c] = coder.scale;
        if (p.sums) {
          float s = sum_part[0][threadIdx.x];
#pragma unroll
          for (int k = 1; k < WARPS; ++k) s += sum_part[k][threadIdx.x];
          p.sums[tile_r * p.C + c] = s;
        }
      }
    }
    __syncthreads();
    f2 inv[4], minus[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      inv[j] = *reinterpret_cast<const f2*>(&col_inv[l * 8 + 2 * j]);
      minus[j] = *reinterpret_cast<const f2*>(&col_minus[l * 8 + 2 * j]);
    }
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      const int r = h + HALVES * i;
      f2 v[4];
      values(i, v);
      if (r < rows && n > 0)
        *reinterpret_cast<uint2*>(p.q_cols + (r0 + r) * p.ldq + c0) =
            make_uint2(code2(v[0], inv[0], minus[0]) | code2(v[1], inv[1], minus[1]) << 16, code2(v[2], inv[2], minus[2]) | code2(v[3], inv[3], minus[3]) << 16);
    }
  }
}

// sums [tiles][C] -> out [C], in the order of the tiles
template <class T>
__global__ void __launch_bounds__(1024)
column_sum_kernel(const float* sums, T* out, long long tiles, int C) {
  __shared__ float part[32][33];
  begin();
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), k = threadIdx.x >> 5;
  float s = 0.f;
  if (c < C) {
#pragma unroll 8
    for (long long t = k; t < tiles; t += 32) s += sums[t * C + c];
  }
  part[k][threadIdx.x & 31] = s;
  __syncthreads();
  if (k == 0 && c < C) {
#pragma unroll
    for (int j = 1; j < 32; ++j) s += part[j][threadIdx.x];
    out[c] = down<T>(s);
  }
}

// ------------------------------------------------------------------------------------------------ norm
// One block a row, V times eight neighbouring columns a thread, held in registers between the sum of squares and the codes.  Sixteen threads
// share a scale.
struct NormArgs {
  const void *x, *res, *g;
  void* sum;                       // x + res, written where res is given
  uint8_t* q;
  float* scale;
  float* a;                        // 1 / rms of each row, or null
  long long ldx, ldr, ldq, T;
  int D, form;
  float eps;
};

template <class T, int V, bool VEC>
__global__ void __launch_bounds__(512)
norm_quantize_kernel(NormArgs p) {
  __shared__ float red[16];
  begin();
  const long long row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const T* res = p.res ? static_cast<const T*>(p.res) + row * p.ldr : nullptr;
  Eight<T> s[V], r[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = (threadIdx.x + v * blockDim.x) * 8;
    s[v] = fetch<VEC, T>(x + c, min(8, p.D - c));
    if (res) r[v] = fetch<VEC, T>(res + c, min(8, p.D - c));
  }
  f2 ss2 = 0ull;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    f2 f[4];
    pairs(s[v], f);
    if (res) {
      f2 t[4];
      pairs(r[v], t);
      float sum[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) { const float2 u = f2_unpack(f2_add(f[j], t[j])); sum[2 * j] = u.x; sum[2 * j + 1] = u.y; }
      s[v] = pack<T>(sum);                                // the norm is that of the sum as it is kept
      const int c = (threadIdx.x + v * blockDim.x) * 8;
      put<VEC, T>(static_cast<T*>(p.sum) + row * p.D + c, s[v], min(8, p.D - c));
      pairs(s[v], f);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) ss2 = f2_fma(f[j], f[j], ss2);
  }
  float ss = f2_unpack(ss2).x + f2_unpack(ss2).y;
#pragma unroll
  for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (blockDim.x > 32) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = ss;
    __syncthreads();
    ss = 0.f;
    for (int k = 0; k < int(blockDim.x >> 5); ++k) ss += red[k];
  }
  const float mean = ss / p.D;
  const float a = p.form == 0 ? rsqrtf(mean + p.eps) : 1.f / (sqrtf(mean) + p.eps);
  if (p.a && threadIdx.x == 0) p.a[row] = a;
  const f2 a2 = f2_pack(a, a);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = (threadIdx.x + v * blockDim.x) * 8;
    f2 f[4], g[4];
    pairs(s[v], f);
    pairs(fetch<VEC, T>(static_cast<const T*>(p.g) + c, min(8, p.D - c)), g);
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = f2_mul(f2_mul(f[j], a2), g[j]);
    uint32_t m = largest(magnitudes(f));
#pragma unroll
    for (int o = 8; o; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const Coder k(m);
    if (c < p.D) {
      *reinterpret_cast<uint2*>(p.q + row * p.ldq + c) = encode(k, f);
      if ((threadIdx.x & 15) == 0) p.scale[(c / BLOCK) * fours(p.T) + row] = k.scale;
    }
  }
}

// ------------------------------------------------------------------------------------------------ norm, backward
//   dx = a * (dn * g) - x * c * mean(dn * g * x) (+ ds),  dg = sum over the rows of dn * x * a
// a = 1 / sqrt(mean(x^2) + eps) and c = a^3 (form 0), or a = 1 / (rms + eps) and c = a^2 / rms (form 1).  dn is the input gradient of the projection in
// fp32, as its product leaves it: rounded to 16 bits it would cost dg, a sum over all rows, half as much again as its own rounding.  A block goes
// through rows with a stride of the grid, its threads keep their columns and add up dg for them; the next row's loads are on their way while this
// one's sum crosses the block.  us with ds, in brackets those of a copy of as many bytes: bf16 8192 x 4096 58 (53), 4096 x 8192 64 (53); above 8192 columns the
// sums and one row fill the 128 registers of 512 threads and 112 to 272 bytes spill, 4096 x 8200 84 (53), 2048 x 16384 75 (53).  fp32 spills from 2049
// columns on (128 to 360 bytes): 8192 x 2048 56 (43), 8192 x 4096 124 (83), 2048 x 16384 135 (83).
struct NormBackArgs {
  const void *x, *g, *ds;
  const float *a, *dn;
  void* dx;
  float* dg;                       // [blocks][D]
  long long T;
  int D, form;
  float eps;
};
template <class T, int V, bool VEC>
__global__ void __launch_bounds__(512, 1)
norm_backward_kernel(NormBackArgs p) {
  __shared__ float red[2][16];
  begin();
  // with four times eight columns a thread, the gain is read again for each row and nothing is fetched ahead: the registers would not do
  constexpr bool AHEAD = V < 4;
  struct Row { Eight<T> x[V], s[V]; Eight<float> dn[V]; } now, next;
  Eight<T> gain[AHEAD ? V : 1];
  f2 acc[V][4];
  auto column = [&](int v) { return int(threadIdx.x + v * blockDim.x) * 8; };
  auto load = [&](Row& r, long long row) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = column(v), n = row < p.T ? min(8, p.D - c) : 0;
      r.x[v] = fetch<VEC, T>(static_cast<const T*>(p.x) + row * p.D + c, n);
      r.dn[v] = fetch<VEC, float>(p.dn + row * p.D + c, n);
      if (p.ds) r.s[v] = fetch<VEC, T>(static_cast<const T*>(p.ds) + row * p.D + c, n);
    }
  };
  auto gains = [&](int v) { return fetch<VEC, T>(static_cast<const T*>(p.g) + column(v), min(8, p.D - column(v))); };
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if (AHEAD) gain[AHEAD ? v : 0] = gains(v);
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[v][j] = 0ull;
  }
  if (AHEAD) load(next, blockIdx.x);
  int turn = 0;
  for (long long row = blockIdx.x; row < p.T; row += gridDim.x, turn ^= 1) {
    const float a = p.a[row];
    const f2 a2 = f2_pack(a, a);
    if (AHEAD) {
      now = next;
      load(next, row + gridDim.x);
    } else {
      load(now, row);
    }
    f2 gv[V][4], dot = 0ull;                               // dn * g
#pragma unroll
    for (int v = 0; v < V; ++v) {
      f2 d[4], x[4], g[4];
      pairs(now.x[v], x);
      pairs(now.dn[v], d);
      pairs(AHEAD ? gain[AHEAD ? v : 0] : gains(v), g);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        gv[v][j] = f2_mul(d[j], g[j]);
        dot = f2_fma(gv[v][j], x[j], dot);
        acc[v][j] = f2_fma(d[j], f2_mul(x[j], a2), acc[v][j]);
      }
    }
    float sum = f2_unpack(dot).x + f2_unpack(dot).y;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (blockDim.x > 32) {
      if ((threadIdx.x & 31) == 0) red[turn][threadIdx.x >> 5] = sum;
      __syncthreads();
      sum = 0.f;
      for (int k = 0; k < int(blockDim.x >> 5); ++k) sum += red[turn][k];
    }
    float c = a * a * a;
    if (p.form == 1) {
      const float rms = 1.f / a - p.eps;
      c = rms > 0.f ? a * a / rms : 0.f;                   // a row of zeros
    }
    const float m = -c * (sum / p.D);
    const f2 m2 = f2_pack(m, m);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      f2 x[4], s[4];
      pairs(now.x[v], x);
      if (p.ds) pairs(now.s[v], s);
      float f[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f2 d = f2_fma(gv[v][j], a2, f2_mul(x[j], m2));
        if (p.ds) d = f2_add(d, s[j]);
        const float2 t = f2_unpack(d);
        f[2 * j] = t.x; f[2 * j + 1] = t.y;
      }
      put<VEC, T>(static_cast<T*>(p.dx) + row * p.D + column(v), pack<T>(f), min(8, p.D - column(v)));
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int n = min(8, p.D - column(v));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 t = f2_unpack(acc[v][j]);
      if (2 * j < n) p.dg[(long long)blockIdx.x * p.D + column(v) + 2 * j] = t.x;
      if (2 * j + 1 < n) p.dg[(long long)blockIdx.x * p.D + column(v) + 2 * j + 1] = t.y;
    }
  }
}

// ------------------------------------------------------------------------------------------------ back
// Eight values a thread and turn, two turns with both loads on their way before the first value is used.
template <class T, bool VEC>
__global__ void __launch_bounds__(256)
dequantize_kernel(const uint8_t* __restrict__ q, const float* __restrict__ scale, T* __restrict__ x, long long R, int C, long long ldq,
                  long long s_row, long long s_col, int tiles) {
  constexpr int TURNS = 2;
  const uint32_t per_row = (uint32_t(C) + 7) / 8;
  const long long total = R * per_row;
  uint32_t w[TURNS][2];
  float s[TURNS];
  long long row[TURNS];
  int c[TURNS];
#pragma unroll
  for (int u = 0; u < TURNS; ++u) {
    const long long i = ((long long)blockIdx.x * TURNS + u) * 256 + threadIdx.x;
    row[u] = i >= total ? -1 : total < 0x80000000LL ? (long long)(uint32_t(i) / per_row) : i / per_row;
    w[u][0] = w[u][1] = 0u;
    if (row[u] < 0) continue;
    c[u] = int(i - row[u] * per_row) * 8;
    s[u] = scale[(tiles ? row[u] / BLOCK : row[u]) * s_row + (c[u] / BLOCK) * s_col];
    const uint8_t* from = q + row[u] * ldq + c[u];
    if (VEC) {
      const uint2 t = *reinterpret_cast<const uint2*>(from);
      w[u][0] = t.x; w[u][1] = t.y;
    } else {
      for (int j = 0; j < min(8, C - c[u]); ++j) w[u][j >> 2] |= uint32_t(from[j]) << (8 * (j & 3));
    }
  }
#pragma unroll
  for (int u = 0; u < TURNS; ++u) {
    if (row[u] < 0) continue;
    float f[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 t = decode2(w[u][j >> 1] >> (16 * (j & 1)));
      f[2 * j] = t.x * s[u]; f[2 * j + 1] = t.y * s[u];
    }
    put<VEC, T>(x + row[u] * C + c[u], pack<T>(f), min(8, C - c[u]));
  }
}

template <class T> bool aligned16(const void* p, long long ld) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * (long long)sizeof(T) % 16 == 0;
}

template <class T, int FORM, bool NORM>
static int launch_quantize(const QuantArgs& p, cudaStream_t st) {
  const long long tiles = (p.R + BLOCK - 1) / BLOCK * p.col_tiles;
  if (tiles > 0x7fffffffLL) return -3;
  const bool vec = p.C % 8 == 0 && aligned16<T>(p.x, p.ld) && (!NORM || aligned16<T>(p.g, 8));
  return launch_chained(false, vec ? quantize_kernel<T, FORM, NORM, true> : quantize_kernel<T, FORM, NORM, false>, dim3((unsigned)tiles), quant_threads(FORM, NORM), 0, st, p);
}
template <class T>
static int launch_form(const QuantArgs& p, int form, cudaStream_t st) {
  if (p.a) return form == COLS ? launch_quantize<T, COLS, true>(p, st) : -3;
  switch (form) {
    case ROWS: return launch_quantize<T, ROWS, false>(p, st);
    case COLS: return launch_quantize<T, COLS, false>(p, st);
    case ROWS | COLS: return launch_quantize<T, ROWS | COLS, false>(p, st);
    case TILE: return launch_quantize<T, TILE, false>(p, st);
  }
  return -3;
}

template <class T, int V>
static int launch_norm_v(const NormArgs& p, int threads, cudaStream_t st) {
  const bool vec = p.D % 8 == 0 && aligned16<T>(p.x, p.ldx) && aligned16<T>(p.g, 8) && (!p.res || (aligned16<T>(p.res, p.ldr) && aligned16<T>(p.sum, 8)));
  return launch_chained(false, vec ? norm_quantize_kernel<T, V, true> : norm_quantize_kernel<T, V, false>, dim3((unsigned)p.T), threads, 0, st, p);
}
template <class T>
static int launch_norm(const NormArgs& p, cudaStream_t st) {
  const int groups = (p.D + 7) / 8;
  auto threads = [&](int v) { return ((groups + v - 1) / v + 31) / 32 * 32; };
  if (groups <= 128) return launch_norm_v<T, 1>(p, threads(1), st);
  if (groups <= 512) return launch_norm_v<T, 2>(p, threads(2), st);
  return launch_norm_v<T, 4>(p, threads(4), st);
}

// threads of the backward kernel and its columns of eight a thread
static int back_shape(int D, int& v) {
  const int groups = (D + 7) / 8;
  v = groups <= 256 ? 1 : groups <= 1024 ? 2 : 4;
  return ((groups + v - 1) / v + 31) / 32 * 32;
}
template <class T, int V>
static int launch_back_v(const NormBackArgs& p, int blocks, int threads, cudaStream_t st) {
  const bool vec = p.D % 8 == 0 && aligned16<T>(p.x, 8) && aligned16<T>(p.g, 8) && aligned16<float>(p.dn, 8) && aligned16<T>(p.dx, 8) && aligned16<T>(p.ds, 8);
  return launch_chained(false, vec ? norm_backward_kernel<T, V, true> : norm_backward_kernel<T, V, false>, dim3(blocks), threads, 0, st, p);
}
template <class T>
static int launch_back(const NormBackArgs& p, int blocks, cudaStream_t st) {
  int v;
  const int threads = back_shape(p.D, v);
  return v == 1 ? launch_back_v<T, 1>(p, blocks, threads, st) : v == 2 ? launch_back_v<T, 2>(p, blocks, threads, st) : launch_back_v<T, 4>(p, blocks, threads, st);
}

template <class T>
static int launch_dequantize(const void* q, const float* scale, void* x, long long R, int C, long long ldq, long long s_row, long long s_col,
                             int tiles, cudaStream_t st) {
  const long long blocks = (R * (((long long)C + 7) / 8) + 511) / 512;                // two turns of 256 threads
  if (blocks > 0x7fffffffLL) return -3;
  const bool vec = C % 8 == 0 && ldq % 8 == 0 && reinterpret_cast<uintptr_t>(q) % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  if (vec) dequantize_kernel<T, true><<<(unsigned)blocks, 256, 0, st>>>((const uint8_t*)q, scale, (T*)x, R, C, ldq, s_row, s_col, tiles);
  else dequantize_kernel<T, false><<<(unsigned)blocks, 256, 0, st>>>((const uint8_t*)q, scale, (T*)x, R, C, ldq, s_row, s_col, tiles);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

}  // namespace blk8
}  // namespace sb

// x [R, C] of type 0 bf16, 1 fp16, 2 fp32, rows `ld` apart.  form: 1 rows, 2 columns, 3 both, 4 tiles (codes and scales in q_rows, s_rows).
// a, g: form 2 of x * a[row] * g[column].  sums: column sums of each 128 rows (forms 2 and 3), or null.
extern "C" int sb_fp8_block_quantize(const void* x, long long ld, long long R, int C, int type, int form, void* q_rows, float* s_rows,
                                     void* q_cols, float* s_cols, long long ldq, const float* a, const void* g, float* sums,
                                     cudaStream_t st) {
  using namespace sb::blk8;
  if (R <= 0 || C <= 0) return 0;
  if (ldq % 16 || ldq < C) return -4;
  QuantArgs p{x, ld, R, C, ldq, (uint8_t*)q_rows, s_rows, (uint8_t*)q_cols, s_cols, a, g, sums, (C + BLOCK - 1) / BLOCK};
  return type == 0 ? launch_form<bf16>(p, form, st) : type == 1 ? launch_form<__half>(p, form, st) : launch_form<float>(p, form, st);
}

// sums [tiles][C] of sb_fp8_block_quantize -> out [C]
extern "C" int sb_fp8_block_column_sums(const float* sums, void* out, long long tiles, int C, int type, cudaStream_t st) {
  using namespace sb::blk8;
  if (C <= 0) return 0;
  const int grid = (C + 31) / 32;
  if (type == 0) return sb::launch_chained(false, column_sum_kernel<bf16>, dim3(grid), 1024, 0, st, sums, (bf16*)out, tiles, C);
  if (type == 1) return sb::launch_chained(false, column_sum_kernel<__half>, dim3(grid), 1024, 0, st, sums, (__half*)out, tiles, C);
  return sb::launch_chained(false, column_sum_kernel<float>, dim3(grid), 1024, 0, st, sums, (float*)out, tiles, C);
}

// D up to 16384.  res and sum: both or neither.  form 0: eps under the root, 1: beside it.  a: 1 / rms [T], or null.
extern "C" int sb_fp8_block_norm(const void* x, long long ldx, const void* res, long long ldr, const void* g, void* sum, void* q, long long ldq,
                                 float* scale, float* a, long long T, int D, float eps, int form, int type, cudaStream_t st) {
  using namespace sb::blk8;
  if (T <= 0 || D <= 0) return 0;
  if (D > 16384 || T > 0x7fffffffLL) return -3;
  if (ldq % 16 || ldq < D || !res != !sum) return -4;
  NormArgs p{x, res, g, sum, (uint8_t*)q, scale, a, ldx, ldr, ldq, T, D, form, eps};
  return type == 0 ? launch_norm<bf16>(p, st) : type == 1 ? launch_norm<__half>(p, st) : launch_norm<float>(p, st);
}

// Blocks of the backward kernel: rows of its dg.
extern "C" int sb_fp8_block_norm_back_blocks(long long T, int D) {
  int v;
  const int threads = sb::blk8::back_shape(D, v), per_sm = threads >= 512 ? 1 : 512 / threads < 4 ? 512 / threads : 4;
  const long long most = (long long)sb::num_sms() * per_sm;
  return int(T < most ? T : most);
}
// x, dx, ds (or null) [T, D] and g [D] of `type`, dense; dn fp32 [T, D]; a [T] of sb_fp8_block_norm; dg fp32 [sb_fp8_block_norm_back_blocks][D], whose
// column sums are the gain's gradient
extern "C" int sb_fp8_block_norm_back(const void* x, const void* g, const float* a, const float* dn, const void* ds, void* dx, float* dg, long long T, int D,
                                      float eps, int form, int type, cudaStream_t st) {
  using namespace sb::blk8;
  if (T <= 0 || D <= 0) return 0;
  if (D > 16384) return -3;
  const int blocks = sb_fp8_block_norm_back_blocks(T, D);
  NormBackArgs p{x, g, ds, a, dn, dx, dg, T, D, form, eps};
  return type == 0 ? launch_back<bf16>(p, blocks, st) : type == 1 ? launch_back<__half>(p, blocks, st) : launch_back<float>(p, blocks, st);
}

// q [R, C], rows ldq apart, times scale[row * s_row + (column / 128) * s_col] (tiles: row / 128) -> x [R, C] of `type`
extern "C" int sb_fp8_block_dequantize(const void* q, long long ldq, const float* scale, long long s_row, long long s_col, int tiles, void* x,
                                       long long R, int C, int type, cudaStream_t st) {
  using namespace sb::blk8;
  if (R <= 0 || C <= 0) return 0;
  return type == 0   ? launch_dequantize<bf16>(q, scale, x, R, C, ldq, s_row, s_col, tiles, st)
         : type == 1 ? launch_dequantize<__half>(q, scale, x, R, C, ldq, s_row, s_col, tiles, st)
                     : launch_dequantize<float>(q, scale, x, R, C, ldq, s_row, s_col, tiles, st);
}
