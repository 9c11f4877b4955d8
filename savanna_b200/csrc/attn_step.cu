// Attention of one new token of every sequence over its cached keys and values, with a bias by relative position:
//
//   s_j = q k_j / sqrt(hd) + scale table[bucket(len - 1 - j), h],  o = sum_j softmax(s)_j v_j  over the sequence's len keys (0 of them: o = 0)
//
// Every key and value is read once, so memory bounds it, and with few heads or short caches the latency of one block's chain.  A key's hd values
// lie over hd / 8 lanes with a 16-byte load each; such a group takes four keys at a time, all of whose loads are under way together, keeps its own
// running maximum and sum, and the groups are joined at the end.  A row (sequence and head) is split over so many blocks that all SMs read: up
// to eight in a cluster, joined through distributed shared memory; more than that leave their results in scratch and a second kernel joins them.
//
// One sequence of 32768 keys, 32 heads of 128, bf16: 82.8 us for 537 MB, the rate of a copy.  Eight warps a block instead of four: 101 -> 82 us there;
// reading the first keys before the query and the bias, two or eight keys a group, or a limit on registers for more blocks gained nothing.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "device_info.h"
#include "entries.h"
#include "pdl.cuh"

namespace sb {
namespace step {
namespace cg = cooperative_groups;
typedef __nv_bfloat16 bf16;

constexpr int WARPS = 8, THREADS = 32 * WARPS;
constexpr int U = 4;                     // keys of a group under way
constexpr int MAX_HD = 256, MAX_T = 1 << 30;             // indexes of keys run a little past T in 32 bits
constexpr float LOG2E = 1.4426950408889634f;

struct Args {
  const void *q, *k, *v;
  void* out;                             // [B, H, hd]
  long long q_sb, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh;      // element strides
  const int* lengths;                    // [B], or null: T everywhere
  const void* table;                     // [nb, H] of type table_type (0 bf16, 1 fp16, 2 fp32)
  const int* buckets;                    // [far + 1]
  float* part;                           // of the form with a second kernel: (maximum, sum) [B, H, splits], then [B, H, splits, hd]
  int T, H, hd, nb, far, table_type, splits;
  float scale_log2, bias_log2;           // 1 / sqrt(hd) and the bias' scale, times log2(e)
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint4 stream16(const void* p) {             // read once by this block: not into L1
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
template <class T> __device__ __forceinline__ void eight(const uint4& v, float (&f)[8]);
template <> __device__ __forceinline__ void eight<bf16>(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
template <> __device__ __forceinline__ void eight<__half>(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    f[2 * i] = t.x; f[2 * i + 1] = t.y;
  }
}
__device__ __forceinline__ bf16 to(float v, bf16) { return __float2bfloat16_rn(v); }
__device__ __forceinline__ __half to(float v, __half) { return __float2half_rn(v); }

// log2(e) * bias at distance d >= 0; a bucket that does not exist has none
__device__ __forceinline__ float bias(const Args& a, int h, int d) {
  const int b = __ldg(a.buckets + min(d, a.far));
  const bool ok = b >= 0 && b < a.nb;
  const size_t i = ok ? (size_t)b * a.H + h : h;
  const float t = a.table_type == 2 ? static_cast<const float*>(a.table)[i]
                  : a.table_type == 1 ? __half2float(static_cast<const __half*>(a.table)[i]) : __bfloat162float(static_cast<const bf16*>(a.table)[i]);
  return ok ? t * a.bias_log2 : 0.f;
}

// A weighted sum under a maximum: what joins two of them.
__device__ __forceinline__ void weights(float m1, float m2, float& m, float& w1, float& w2) {
  m = fmaxf(m1, m2);
  const float r = m == -INFINITY ? 0.f : m;
  w1 = ex2(m1 - r);
  w2 = ex2(m2 - r);
}

// LPK lanes a key: hd <= 8 LPK.  EARLY: the biases of a group's keys are read beside the keys themselves.
template <class T, int LPK, bool EARLY>
__global__ void __launch_bounds__(THREADS, 4)
step_kernel(const Args a) {
  constexpr int G = 32 / LPK;              // groups of a warp
  __shared__ float wm[WARPS], wl[WARPS], wo[WARPS][8 * LPK];
  __shared__ float cm, cl, co[8 * LPK];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, grp = lane / LPK, c0 = (lane % LPK) * 8;
  const int split = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.T) : a.T;
  const int chunk = ((len + a.splits - 1) / a.splits + U - 1) / U * U, j0 = min(len, split * chunk), j1 = min(len, j0 + chunk);
  const bool have = c0 < a.hd;
  const T* kp = static_cast<const T*>(a.k) + b * a.k_sb + h * a.k_sh + (have ? c0 : 0);
  const T* vp = static_cast<const T*>(a.v) + b * a.v_sb + h * a.v_sh + (have ? c0 : 0);
  float q[8], o[8], m = -INFINITY, l = 0.f;
  eight<T>(have ? *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + b * a.q_sb + h * a.q_sh + c0) : make_uint4(0, 0, 0, 0), q);
#pragma unroll
  for (int i = 0; i < 8; ++i) { q[i] *= a.scale_log2; o[i] = 0.f; }
  const float far_bias = EARLY ? 0.f : bias(a, h, a.far);
  for (int j = j0 + (warp * G + grp) * U; __any_sync(0xffffffffu, j < j1); j += WARPS * G * U) {
    uint4 kr[U], vr[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {          // a key beyond the last reads the last one again
      const long long at = max(min(j + u, j1 - 1), j0);
      kr[u] = stream16(kp + at * a.k_st);
      vr[u] = stream16(vp + at * a.v_st);
    }
    float bs[U];
    if (EARLY) {
      if (j + U > len - a.far) {           // some of them nearer than far
#pragma unroll
        for (int u = 0; u < U; ++u) bs[u] = bias(a, h, max(len - 1 - (j + u), 0));
      } else {
        const float t = bias(a, h, a.far);
#pragma unroll
        for (int u = 0; u < U; ++u) bs[u] = t;
      }
    }
    float s[U], mx = m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[8];
      eight<T>(kr[u], f);
      s[u] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s[u] = fmaf(q[i], f[i], s[u]);
      if (!have) s[u] = 0.f;               // columns that this lane has not: 0 * inf of others' would be NaN
    }
#pragma unroll
    for (int d = LPK / 2; d; d >>= 1)
#pragma unroll
      for (int u = 0; u < U; ++u) s[u] += __shfl_xor_sync(0xffffffffu, s[u], d);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int d = len - 1 - (j + u);
      s[u] = j + u < j1 ? s[u] + (EARLY ? bs[u] : d >= a.far ? far_bias : bias(a, h, d)) : -INFINITY;
      mx = fmaxf(mx, s[u]);
    }
    const float ref = mx == -INFINITY ? 0.f : mx, al = ex2(m - ref);
    m = mx;
    l *= al;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] *= al;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float p = ex2(s[u] - ref);
      float f[8];
      eight<T>(vr[u], f);
      l += p;
      if (j + u < j1) {
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = fmaf(p, f[i], o[i]);
      }
    }
  }
  // the groups of a warp, the warps of a block, the blocks of a cluster
#pragma unroll
  for (int d = LPK; d < 32; d <<= 1) {
    float mm, w1, w2;
    weights(m, __shfl_xor_sync(0xffffffffu, m, d), mm, w1, w2);
    m = mm;
    l = l * w1 + __shfl_xor_sync(0xffffffffu, l, d) * w2;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = o[i] * w1 + __shfl_xor_sync(0xffffffffu, o[i], d) * w2;
  }
  if (grp == 0) {
    if (lane == 0) { wm[warp] = m; wl[warp] = l; }
#pragma unroll
    for (int i = 0; i < 8; ++i) wo[warp][c0 + i] = o[i];
  }
  __syncthreads();
  float bm = wm[0];
#pragma unroll
  for (int w = 1; w < WARPS; ++w) bm = fmaxf(bm, wm[w]);
  float e[WARPS], bl = 0.f;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) { e[w] = ex2(wm[w] - (bm == -INFINITY ? 0.f : bm)); bl += e[w] * wl[w]; }
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = cluster.num_blocks();
  const long long row = (long long)b * a.H + h;
  T* out = static_cast<T*>(a.out) + row * a.hd;
  for (int c = threadIdx.x; c < a.hd; c += THREADS) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) t += e[w] * wo[w][c];
    if (a.splits == 1) out[c] = to(bl == 0.f ? 0.f : t / bl, T());     // 0: no keys; NaN stays
    else if (blocks > 1) co[c] = t;
    else a.part[(long long)gridDim.z * a.H * a.splits * 2 + (row * a.splits + split) * a.hd + c] = t;
  }
  if (a.splits == 1) return;
  if (threadIdx.x == 0) {
    if (blocks > 1) { cm = bm; cl = bl; }
    else reinterpret_cast<float2*>(a.part)[row * a.splits + split] = make_float2(bm, bl);
  }
  if (blocks == 1) return;
  cluster.sync();
  if (cluster.block_rank() == 0) {
    float pm[8], tm = -INFINITY, tl = 0.f;
#pragma unroll
    for (int r = 0; r < 8; ++r) { pm[r] = r < blocks ? *cluster.map_shared_rank(&cm, r) : -INFINITY; tm = fmaxf(tm, pm[r]); }
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      pm[r] = ex2(pm[r] - (tm == -INFINITY ? 0.f : tm));
      if (r < blocks) tl += pm[r] * *cluster.map_shared_rank(&cl, r);
    }
    for (int c = threadIdx.x; c < a.hd; c += THREADS) {
      float t = 0.f;
#pragma unroll
      for (int r = 0; r < 8; ++r) if (r < blocks) t += pm[r] * *cluster.map_shared_rank(&co[c], r);
      out[c] = to(tl == 0.f ? 0.f : t / tl, T());
    }
  }
  cluster.sync();                          // the others' shared memory stays until it has been read
}

// Joins the splits of a row: a block a row, two columns a thread, the splits in as many groups as there are threads for.
constexpr int JOIN_THREADS = 512;
template <class T>
__global__ void __launch_bounds__(JOIN_THREADS)
join_kernel(const float* part, T* out, long long rows, int splits, int hd) {
  extern __shared__ float e[];             // [splits], then [JOIN_THREADS][2]
  __shared__ float red[JOIN_THREADS / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, cols = hd / 2, groups = JOIN_THREADS / cols, g = tid / cols;
  const float2* ml = reinterpret_cast<const float2*>(part) + (long long)blockIdx.x * splits;
  const float2* o = reinterpret_cast<const float2*>(part) + rows * splits + (long long)blockIdx.x * splits * cols + tid - g * cols;
  auto block = [&](float v, bool sum) {
#pragma unroll
    for (int d = 16; d; d >>= 1) { const float w = __shfl_xor_sync(0xffffffffu, v, d); v = sum ? v + w : fmaxf(v, w); }
    __syncthreads();
    if (lane == 0) red[warp] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int k = 1; k < JOIN_THREADS / 32; ++k) v = sum ? v + red[k] : fmaxf(v, red[k]);
    return v;
  };
  wait_for_previous();
  float m = -INFINITY, l = 0.f;
  for (int s = tid; s < splits; s += JOIN_THREADS) m = fmaxf(m, ml[s].x);
  m = block(m, false);
  const float ref = m == -INFINITY ? 0.f : m;
  for (int s = tid; s < splits; s += JOIN_THREADS) {
    const float2 v = ml[s];
    const float w = ex2(v.x - ref);
    e[s] = w;
    l += w * v.y;
  }
  l = block(l, true);                      // and e is there
  float2 t = make_float2(0.f, 0.f);
  if (g < groups) {
#pragma unroll 8
    for (int s = g; s < splits; s += groups) { const float2 v = o[(long long)s * cols]; t.x += e[s] * v.x; t.y += e[s] * v.y; }
  }
  float2* sh = reinterpret_cast<float2*>(e + (splits + 1) / 2 * 2);
  sh[tid] = t;
  __syncthreads();
  if (tid < cols) {
    for (int k = 1; k < groups; ++k) { t.x += sh[tid + k * cols].x; t.y += sh[tid + k * cols].y; }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* dst = out + (long long)blockIdx.x * hd + 2 * tid;
    dst[0] = to(t.x * inv, T());
    dst[1] = to(t.y * inv, T());
  }
}

// Blocks a row: so many that there are four on a SM (no more: they would run one after the other), each with 64 keys or more.  Up to eight are a
// cluster; more, with a second kernel, where a row is so long that eight blocks would leave SMs idle for longer than that kernel takes.  us, by
// blocks a row: one sequence of 32768, 32 heads of 128 8: 93, 16: 82.4, 18: 81.7, 24: 87.5; twelve of up to 1500, 16 heads of 64 1: 19, 2: 15.9,
// 4: 19.9; one of 1000, 32 heads 4: 10, 8: 8, 16: 11; 64 of 512, 16 heads 1: 36, 2: 47; one of 65536, 2 heads 8: 280, 64: 28, 128: 20, 256: 21.5.
static int choose_splits(long long rows, int T) {
  const long long want = 4LL * num_sms() / rows, keys = (T + 63) / 64;
  int s = 1;
  while (s < 8 && 2 * s <= want && s < keys) s *= 2;
  if (s < 8 || want <= 8 || T < 8192) return s;
  const long long longest = T / 256;
  return (int)(want < longest ? want : longest);
}

template <class T>
static int launch(const Args& a, int B, cudaStream_t st) {
  const dim3 grid(a.splits, a.H, B);
  // A block's chain counts where it is short, or where lengths differ and the longest sequences' blocks end last: the biases are read early then.
  // With long blocks on all SMs alike the reads of the far bias in every step cost more.  us, late / early: 8 sequences of 300, 32 heads of 128
  // 13.4 / 12.4; of up to 2000 28.9 / 25.4, of 2000 each 43.3 / 43.8; 12 of up to 1500, 16 heads of 64 15.7 / 14.1; one of 7000 28.4 / 25.2, of
  // 16000 44.1 / 44.9, of 32768 82.9 / 87.5; 8 of 16384, 16 heads of 64 82.8 / 93, of up to 16384 50.5 / 45.4.
  // The lengths are on the device: a batch that passes them is taken for one of unequal sequences, and where they are equal and long it goes
  // without the late form's gain.
  const bool early = (a.lengths && B > 1) || a.T <= 1024 * a.splits;
  auto* kernel = early ? a.hd <= 64 ? step_kernel<T, 8, true> : a.hd <= 128 ? step_kernel<T, 16, true> : step_kernel<T, 32, true>
                       : a.hd <= 64 ? step_kernel<T, 8, false> : a.hd <= 128 ? step_kernel<T, 16, false> : step_kernel<T, 32, false>;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = a.splits;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(THREADS);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = a.splits > 1 && a.splits <= 8 ? 1 : 0;
  if (cudaLaunchKernelEx(&cfg, kernel, a) != cudaSuccess) { (void)cudaGetLastError(); return -2; }
  if (a.splits <= 8) return 0;
  return launch_chained(false, join_kernel<T>, dim3((unsigned)(B * a.H)), JOIN_THREADS, (a.splits + 1) / 2 * 8 + JOIN_THREADS * 8, st,
                        (const float*)a.part, (T*)a.out, (long long)B * a.H, a.splits, a.hd);
}

}  // namespace step
}  // namespace sb

using namespace sb::step;

// Blocks a row of sb_attn_step; above eight it needs scratch of B * H * splits * (hd + 2) floats.
extern "C" int sb_attn_step_splits(int B, int H, int T) { return B < 1 || H < 1 || T < 1 ? 1 : choose_splits((long long)B * H, T); }

// q [B, H, hd], k and v [B, T, H, hd] (type 0 bf16, 1 fp16; 16-byte boundaries, strides in elements multiples of 8, unit inner stride), out
// [B, H, hd] contiguous.  lengths [B] int32 (clamped to 0 .. T) or null; table [nb, H] of table_type (0, 1 or 2: fp32), buckets [far + 1] int32
// of the distances 0 .. far.  T <= 2^30.
extern "C" int sb_attn_step(const void* q, const void* k, const void* v, void* out, const int* lengths, int B, int T, int H, int hd,
                            const long long* q_str, const long long* k_str, const long long* v_str, int type, const void* table, int table_type,
                            const int* buckets, int nb, int far, float scale, float bias_scale, float* part, int splits, cudaStream_t st) {
  if (hd < 8 || hd > MAX_HD || hd % 8 || nb < 1 || far < 0 || type < 0 || type > 1 || splits < 1 || splits > 8192 || (splits > 8 && !part)) return -1;
  if (splits != 1 && splits != 2 && splits != 4 && splits < 8) return -1;
  if (B < 0 || H < 0 || T < 0 || T > MAX_T || B > 65535 || H > 65535) return -1;
  if (B == 0 || H == 0) return 0;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) return -4;
  if ((q_str[0] | q_str[1] | k_str[0] | k_str[1] | k_str[2] | v_str[0] | v_str[1] | v_str[2]) & 7) return -4;
  const Args a{q, k, v, out, q_str[0], q_str[1], k_str[0], k_str[1], k_str[2], v_str[0], v_str[1], v_str[2], lengths, table, buckets, part, T, H, hd, nb,
               far, table_type, splits, scale * LOG2E, bias_scale * LOG2E};
  return type == 0 ? launch<bf16>(a, B, st) : launch<__half>(a, B, st);
}
