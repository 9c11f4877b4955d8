// Matrix product of e4m3 operands with fp32 scales for blocks of 128 along the contraction:
//
//   C[m, n] = sum_kb sa[m, kb] * sb[n, kb] * (sum over the block's 128 k of A[m, k] * B[n, k])  (+ bias[n]) (+ residual[m, n]) (+ C[m, n])
//
// sb is given for 128 n at once (weights: tiles of 128 x 128) or for each n (the weight gradient's operand).  The tensor cores form the inner
// sum; their accumulator cannot be scaled on the way, so each k-block's product is a fresh accumulator in TMEM that the epilogue warps read and
// add, scaled, to sums in their registers (fp32, the k-blocks in order).  This is the whole design:
//
//   warp 0     TMA producer: a k-block's operands, 32 KB a CTA and stage
//   warp 1     MMA issuer: four products of 32 k a k-block, each k-block into the next of the TMEM buffers
//   warp 2     the scales into a ring in shared memory (asynchronous copies of 16 bytes, or of 4 for any strides), eight k-blocks deep, handed over by fours
//   warps 4-11 a lane owns a row and half of the tile's columns: tcgen05.ld of 32 columns twice, packed multiply-adds on the one while the next of the
//              other are on their way; after the last k-block the sums leave by bulk stores beside the next tile's products
//
// Two tiles: 256 x 256 on a CTA pair (cta_group::2; two buffers of 256 columns, 128 sums a thread) and 128 x 128 on one CTA (four buffers of
// 128, 64 sums), for outputs that leave the chip idle in the larger one.
//
// 8192 x 4096 x 12288: 324 us forward, 313 input gradient, 526 weight gradient (2540, 2630, 1570 TFLOP/s; the per-tensor kernel 261 to 271).  A k-block
// of a pair takes 0.48 us, some 840 cycles (thousands of products back to back: 392 us at 1.43 GHz under the power cap) where its products need 512:
// reading 256 columns of TMEM and a multiply-add for each value, in warps that also wait for every accumulator; the weight gradient, whose values have
// a factor for their column too, 1330 (549 us at 1.70 GHz).  Without the multiply-adds the forward takes 250.
// The single-CTA tile is bound by the 32 KB of operands that a k-block takes from L2.
//
// A programmatic dependent of the kernel before it (pdl.cuh, the second kind).  All waits are bounded (sm100.cuh).
#include "entries.h"
#include "f32x2.cuh"
#include "fp8_block.cuh"
#include "pdl.cuh"
#include "sm100.cuh"

namespace sb {

int make_tmap_2d_bf16(CUtensorMap* out, const void* base, uint64_t inner, uint64_t outer, uint64_t ld, uint32_t box_inner, uint32_t box_outer);
int make_tmap_2d_u8(CUtensorMap* out, const void* base, uint64_t inner, uint64_t outer, uint64_t ld, uint32_t box_inner, uint32_t box_outer);

namespace blk8 {

struct GemmArgs {
  void* C;
  const void *bias, *residual;
  const float *sa, *sb;
  long long sa_m, sa_k, sb_n, sb_k;      // strides; sb_n counts blocks of 128 n where the scale is theirs
  long long ldc, ldr;
  int M, N, K, type, beta;
  bool boxes;                            // results, and what is added, on 16-byte boundaries: stored in boxes
  bool runs;                             // scales of neighbouring rows (and columns, where those have their own) lie together, on 16-byte boundaries
  uint32_t* status;
};

constexpr int EPI_WARPS = 8, NUM_THREADS = 128 + 32 * EPI_WARPS;
// Registers: 168 a thread at launch (384 threads), of which the first four warps keep 56 and each of the other eight gets 224:
// 128 * 56 + 256 * 224 = 384 * 168.
constexpr int REGS_FEW = 56, REGS_MANY = 224;
static_assert(128 * REGS_FEW + 32 * EPI_WARPS * REGS_MANY <= NUM_THREADS * 168, "registers of a block");
constexpr int OPERAND = 128 * 128, STAGE_BYTES = 2 * OPERAND;
// Scales of a k-block, rows and columns.  They change hands by GROUP k-blocks: a barrier for each cost the epilogue 200 cycles of 1000.
constexpr int GROUP = 4, SLOTS = 2 * GROUP, SLOT_BYTES = (128 + 256) * 4;
// Shared memory: operand stages; the tile on its way out, 32 rows x 64 columns of 16 bits a box, a box or two a warp; scales; barriers.
template <bool PAIR> struct Space {
  static constexpr int STAGES = PAIR ? 4 : 5, BOXES = PAIR ? 2 : 1, BOX = 32 * 128;
  static constexpr int OUT = STAGES * STAGE_BYTES, SLOT = OUT + EPI_WARPS * BOXES * BOX, BAR = SLOT + SLOTS * SLOT_BYTES, BYTES = BAR + 256 + 1024;
  static_assert(BYTES <= 232448, "shared memory of a block");
};
constexpr int GROUP_M = 8;               // raster: m-tiles that share the concurrently running n-tiles

__device__ __forceinline__ void raster(int tile, int m_tiles, int n_tiles, int& mt, int& nt) {
  const int per_group = GROUP_M * n_tiles, g = tile / per_group, first = g * GROUP_M, size = min(GROUP_M, m_tiles - first), r = tile - g * per_group;
  mt = first + r % size;
  nt = r / size;
}

// acc += (a, b) * s.  Volatile, as the loads and their wait are: it stays behind the wait for a and b.
__device__ __forceinline__ void add_scaled(f2& acc, uint32_t a, uint32_t b, f2 s) {
  asm volatile("{\n\t.reg .b64 t;\n\tmov.b64 t, {%1, %2};\n\tfma.rn.f32x2 %0, t, %3, %0;\n\t}" : "+l"(acc) : "r"(a), "r"(b), "l"(s));
}
__device__ __forceinline__ f2 scaled(uint32_t a, uint32_t b, f2 s) {
  f2 v;
  asm volatile("{\n\t.reg .b64 t;\n\tmov.b64 t, {%1, %2};\n\tmul.rn.f32x2 %0, t, %3;\n\t}" : "=l"(v) : "r"(a), "r"(b), "l"(s));
  return v;
}
// 32 rows x 32 columns of TMEM, spread as the tensor cores spread a fragment: of each 8 columns a lane has two neighbouring ones,
// 2 (lane % 4), of rows lane / 4, + 8 (r[4 i ..]), + 16, + 24 (r[16 + 4 i ..])
__device__ __forceinline__ void load_fragments(uint32_t taddr, uint32_t (&r)[32]) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[16 * h]), "=r"(r[16 * h + 1]), "=r"(r[16 * h + 2]), "=r"(r[16 * h + 3]), "=r"(r[16 * h + 4]), "=r"(r[16 * h + 5]), "=r"(r[16 * h + 6]),
          "=r"(r[16 * h + 7]), "=r"(r[16 * h + 8]), "=r"(r[16 * h + 9]), "=r"(r[16 * h + 10]), "=r"(r[16 * h + 11]), "=r"(r[16 * h + 12]),
          "=r"(r[16 * h + 13]), "=r"(r[16 * h + 14]), "=r"(r[16 * h + 15])
        : "r"(taddr + (uint32_t(16 * h) << 16))
        : "memory");
}
__device__ __forceinline__ void put2(uint32_t at, float2 v) {
  asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(at), "f"(v.x), "f"(v.y) : "memory");
}
__device__ __forceinline__ f2 get2(uint32_t at) {
  f2 v;
  asm volatile("ld.shared.b64 %0, [%1];" : "=l"(v) : "r"(at) : "memory");
  return v;
}
// The arrival that frees a TMEM buffer hands over no memory (what was read is in registers), so it orders none: a releasing one would wait for
// the loads of the next scales too, and took four fifths of a k-block's time.
__device__ __forceinline__ void arrive_relaxed(uint32_t cluster_addr, bool one) {
  asm volatile("{\n\t.reg .pred P;\n\tsetp.ne.b32 P, %1, 0;\n\t@P mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];\n\t}"
               ::"r"(cluster_addr), "r"(uint32_t(one)) : "memory");
}

// four bytes to shared memory, or zeros
__device__ __forceinline__ void copy4(uint32_t dst, const float* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(__cvta_generic_to_global(src)), "r"(there ? 4 : 0) : "memory");
}
// up to four values there are, zeros for the others
__device__ __forceinline__ void copy16(uint32_t dst, const float* src, int there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(__cvta_generic_to_global(src)), "r"(min(max(there, 0), 4) * 4) : "memory");
}
// the thread's copies so far arrive once they have landed
__device__ __forceinline__ void copies_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ float get1(uint32_t at) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

__device__ __forceinline__ float2 two(uint32_t w, bf16) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
__device__ __forceinline__ float2 two(uint32_t w, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ uint32_t word(float a, float b, bf16) { return pack_bf2(a, b); }
__device__ __forceinline__ uint32_t word(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void tma_store_2d(const void* tmap, uint32_t src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"(src) : "memory");
}
template <class T> __device__ __forceinline__ void add8(const T* p, float (&f)[16], int at) {
  float t[8];
  unpack(*reinterpret_cast<const Eight<T>*>(p), t);
#pragma unroll
  for (int j = 0; j < 8; ++j) f[at + j] += t[j];
}
// A warp's 32 rows of 16-bit results by way of shared memory (128-byte rows, 128-byte swizzle) and a bulk store that runs beside the next
// tile.  Stored from the registers a tile of 256 x 256 held its warps up for 2 us.  FRAGMENTS: the sums are spread as load_fragments leaves
// them.  The sum of what is added to the product is formed in fp32.
template <int COLS, class T, bool FRAGMENTS>
__device__ __forceinline__ void store_boxes(const GemmArgs& p, const CUtensorMap* tmC, uint32_t space, const f2* acc, int row0, int col0, int lane) {
  if (lane == 0) bulk_wait_read<0>();              // the last tile has left
  __syncwarp();
  if (FRAGMENTS) {
#pragma unroll
    for (int c = 0; c < COLS / 8; ++c)             // 8 columns each
#pragma unroll
      for (int k = 0; k < 4; ++k) {                // rows lane / 4 + 8 k
        const int r = (lane >> 2) + 8 * k, row = row0 + r, col = col0 + 8 * c + 2 * (lane & 3);
        float2 f = f2_unpack(acc[(c >> 2) * 16 + (k >> 1) * 8 + (c & 3) * 2 + (k & 1)]);
        if (p.beta && row < p.M && col < p.N) {
          const float2 o = two(*reinterpret_cast<const uint32_t*>(static_cast<const T*>(p.C) + row * p.ldc + col), T());
          f.x += o.x; f.y += o.y;
        }
        const uint32_t at = space + (c >> 3) * (32 * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4) + (lane & 3) * 4;
        asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(word(f.x, f.y, T())) : "memory");
      }
  } else {
    const int row = row0 + lane;
    const bool extra = (p.bias || p.residual || p.beta) && row < p.M;
#pragma unroll
    for (int c = 0; c < COLS / 16; ++c) {
      float f[16];
#pragma unroll
      for (int j = 0; j < 8; ++j) { const float2 t = f2_unpack(acc[c * 8 + j]); f[2 * j] = t.x; f[2 * j + 1] = t.y; }
      if (extra) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int col = col0 + c * 16 + 8 * h;
          if (col < p.N) {
            if (p.bias) add8(static_cast<const T*>(p.bias) + col, f, 8 * h);
            if (p.residual) add8(static_cast<const T*>(p.residual) + row * p.ldr + col, f, 8 * h);
            if (p.beta) add8(static_cast<const T*>(p.C) + row * p.ldc + col, f, 8 * h);
          }
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t at = space + (c >> 2) * (32 * 128) + lane * 128 + (((2 * (c & 3) + h) ^ (lane & 7)) << 4);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(word(f[8 * h], f[8 * h + 1], T())), "r"(word(f[8 * h + 2], f[8 * h + 3], T())),
                     "r"(word(f[8 * h + 4], f[8 * h + 5], T())), "r"(word(f[8 * h + 6], f[8 * h + 7], T())) : "memory");
      }
    }
  }
  fence_proxy_async();
  __syncwarp();
  if (lane == 0 && row0 < p.M) {
#pragma unroll
    for (int b = 0; b < COLS / 64; ++b)
      if (col0 + 64 * b < p.N) tma_store_2d(tmC, space + b * (32 * 128), col0 + 64 * b, row0);
    bulk_commit();
  }
}
// fp32 results: boxes of 32 columns, half of the warp's columns at a time
template <int COLS>
__device__ __forceinline__ void store_boxes_f32(const GemmArgs& p, const CUtensorMap* tmC, uint32_t space, const f2* acc, int row0, int col0, int lane) {
  constexpr int BOXES = COLS / 64;
  const int row = row0 + lane;
  const bool extra = (p.bias || p.residual || p.beta) && row < p.M;
#pragma unroll
  for (int round = 0; round < 2; ++round) {
    if (lane == 0) bulk_wait_read<0>();
    __syncwarp();
#pragma unroll
    for (int c = 0; c < 4 * BOXES; ++c) {          // 8 columns each
      const int first = round * 32 * BOXES + 8 * c, col = col0 + first;
      float f[16];
#pragma unroll
      for (int j = 0; j < 4; ++j) { const float2 t = f2_unpack(acc[first / 2 + j]); f[2 * j] = t.x; f[2 * j + 1] = t.y; }
      if (extra && col < p.N) {
        if (p.bias) add8(static_cast<const float*>(p.bias) + col, f, 0);
        if (p.residual) add8(static_cast<const float*>(p.residual) + row * p.ldr + col, f, 0);
        if (p.beta) add8(static_cast<const float*>(p.C) + row * p.ldc + col, f, 0);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t at = space + (c >> 2) * (32 * 128) + lane * 128 + (((2 * (c & 3) + h) ^ (lane & 7)) << 4);
        asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(f[4 * h]), "f"(f[4 * h + 1]), "f"(f[4 * h + 2]), "f"(f[4 * h + 3]) : "memory");
      }
    }
    fence_proxy_async();
    __syncwarp();
    if (lane == 0 && row0 < p.M) {
#pragma unroll
      for (int b = 0; b < BOXES; ++b) {
        const int col = col0 + round * 32 * BOXES + 32 * b;
        if (col < p.N) tma_store_2d(tmC, space + b * (32 * 128), 2 * col, row0);      // the map counts 16-bit halves
      }
      bulk_commit();
    }
  }
}
template <class T> __device__ __forceinline__ void store_one(const GemmArgs& p, int row, int col, float f) {
  T* c = static_cast<T*>(p.C) + row * p.ldc + col;
  if (p.bias) f += up(static_cast<const T*>(p.bias)[col]);
  if (p.residual) f += up(static_cast<const T*>(p.residual)[row * p.ldr + col]);
  if (p.beta) f += up(*c);
  *c = down<T>(f);
}
// Everything else (rows off 16-byte boundaries, fp32 sums in fragments): 16 columns at a time, a half-warp a row.
template <int COLS, class T, bool FRAGMENTS>
__device__ __forceinline__ void store_values(const GemmArgs& p, uint32_t space, const f2* acc, int row0, int col0, int lane) {
#pragma unroll
  for (int c = 0; c < COLS / 16; ++c) {
    __syncwarp();
    if (FRAGMENTS) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = (lane >> 2) + 8 * k;
          put2(space + r * 64 + (8 * i + 2 * (lane & 3)) * 4, f2_unpack(acc[(c >> 1) * 16 + (k >> 1) * 8 + (2 * (c & 1) + i) * 2 + (k & 1)]));
        }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) put2(space + lane * 64 + 8 * j, f2_unpack(acc[c * 8 + j]));
    }
    __syncwarp();
    const int col = col0 + c * 16 + (lane & 15);
#pragma unroll 4
    for (int r = lane >> 4; r < 32; r += 2)
      if (col < p.N && row0 + r < p.M) store_one<T>(p, row0 + r, col, get1(space + r * 64 + (lane & 15) * 4));
  }
  __syncwarp();
}
template <int COLS, bool FRAGMENTS>
__device__ __forceinline__ void store_tile(const GemmArgs& p, const CUtensorMap* tmC, uint32_t space, const f2* acc, int row0, int col0, int lane) {
  if constexpr (!FRAGMENTS) {
    if (p.boxes && p.type == 2) return store_boxes_f32<COLS>(p, tmC, space, acc, row0, col0, lane);
  }
  if (p.boxes && p.type == 0) store_boxes<COLS, bf16, FRAGMENTS>(p, tmC, space, acc, row0, col0, lane);
  else if (p.boxes) store_boxes<COLS, __half, FRAGMENTS>(p, tmC, space, acc, row0, col0, lane);
  else if (p.type == 0) store_values<COLS, bf16, FRAGMENTS>(p, space, acc, row0, col0, lane);
  else if (p.type == 1) store_values<COLS, __half, FRAGMENTS>(p, space, acc, row0, col0, lane);
  else store_values<COLS, float, FRAGMENTS>(p, space, acc, row0, col0, lane);
}

__device__ __forceinline__ bool spin_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, uint32_t* status, uint32_t code) {
  for (int i = 0; i < 64; ++i)
    if (mbar_test(bar, parity)) return true;
  return mbar_wait(bar, parity, abort_flag, status, code);
}
template <bool PAIR, int A_MN, int B_MN, bool SB_ROWS>
__global__ void __launch_bounds__(NUM_THREADS, 1)
gemm_fp8_block_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmC, GemmArgs p) {
  typedef Space<PAIR> S;
  constexpr int STAGES = S::STAGES;
  constexpr int TM = PAIR ? 256 : 128, TN = PAIR ? 256 : 128, BUFS = 512 / TN, COLS = TN / 2;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t bar_base = smem_base + S::BAR;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (STAGES + s); };
  auto tfull_bar = [&](int b) { return bar_base + 8u * (2 * STAGES + b); };
  auto tempty_bar = [&](int b) { return bar_base + 8u * (2 * STAGES + 4 + b); };
  auto sfull_bar = [&](int g) { return bar_base + 8u * (2 * STAGES + 8 + g); };
  auto sempty_bar = [&](int g) { return bar_base + 8u * (2 * STAGES + 10 + g); };
  constexpr int FLAGS = S::BAR + 8 * (2 * STAGES + 12);
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem_gen + FLAGS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem_gen + FLAGS + 8);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0u;             // 0 issues the products, 1 is its partner
  const int worker = PAIR ? blockIdx.x >> 1 : blockIdx.x, workers = PAIR ? gridDim.x >> 1 : gridDim.x;
  const int m_tiles = (p.M + TM - 1) / TM, n_tiles = (p.N + TN - 1) / TN, num_tiles = m_tiles * n_tiles;
  const int num_kb = (p.K + BLOCK - 1) / BLOCK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 1); }
    for (int b = 0; b < BUFS; ++b) { mbar_init(tfull_bar(b), 1); mbar_init(tempty_bar(b), (PAIR ? 2 : 1) * EPI_WARPS); }
    for (int g = 0; g < 2; ++g) { mbar_init(sfull_bar(g), 32); mbar_init(sempty_bar(g), EPI_WARPS); }
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmB);
    if (p.boxes) prefetch_tmap(&tmC);
  }
  if (warp == 1) {
    if (PAIR) { tmem_alloc_pair(smem_u32(const_cast<uint32_t*>(tmem_slot)), 512); tmem_relinquish_pair(); }
    else { tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), 512); tmem_relinquish(); }
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) { cluster_arrive(); cluster_wait(); }                  // barriers of both CTAs are there before either signals the other
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  wait_for_previous();

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_FEW));
    if (warp == 0 && elect_one()) {
      int stage = 0; uint32_t phase = 0;
      bool ok = true;
      for (int tile = worker; tile < num_tiles && ok; tile += workers) {
        int mt, nt; raster(tile, m_tiles, n_tiles, mt, nt);
        const int m0 = mt * TM + int(rank) * 128, n0 = nt * TN + int(rank) * 128;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, p.status, ST_FP8_BLOCK + 1)) { ok = false; break; }
          const uint32_t a_dst = smem_base + stage * STAGE_BYTES, b_dst = a_dst + OPERAND;
          const int k0 = kb * BLOCK;
          if (PAIR) {
            const uint32_t bar = map_to_cta(full_bar(stage), 0);   // the even CTA counts both CTAs' bytes
            if (rank == 0) mbar_expect_tx(full_bar(stage), 2 * STAGE_BYTES);
            tma_load_2d_pair(a_dst, &tmA, A_MN ? m0 : k0, A_MN ? k0 : m0, bar);
            tma_load_2d_pair(b_dst, &tmB, B_MN ? n0 : k0, B_MN ? k0 : n0, bar);
          } else {
            mbar_expect_tx(full_bar(stage), STAGE_BYTES);
            tma_load_2d(a_dst, &tmA, A_MN ? m0 : k0, A_MN ? k0 : m0, full_bar(stage));
            tma_load_2d(b_dst, &tmB, B_MN ? n0 : k0, B_MN ? k0 : n0, full_bar(stage));
          }
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
      }
      if (!ok) {                                                   // copies in flight land before the block ends
        const unsigned long long t0 = globaltimer();
        while (globaltimer() - t0 < 200000ull) { __nanosleep(1000); }
      }
    }
    if (warp == 1 && rank == 0 && elect_one()) {
      constexpr uint32_t idesc = umma_idesc_fp8(TM, TN, A_MN, B_MN, 0, 0);
      constexpr uint32_t a_lbo = A_MN ? OPERAND : 16, a_step = A_MN ? (32 * 128) >> 4 : 2;
      constexpr uint32_t b_lbo = B_MN ? OPERAND : 16, b_step = B_MN ? (32 * 128) >> 4 : 2;
      int stage = 0, buf = 0; uint32_t phase = 0, buf_phase = 0;
      bool ok = true;
      for (int tile = worker; tile < num_tiles && ok; tile += workers)
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!spin_wait(full_bar(stage), phase, abort_flag, p.status, ST_FP8_BLOCK + 3)) { ok = false; break; }
          const uint32_t a_addr = smem_base + stage * STAGE_BYTES;
          const uint64_t adesc = umma_smem_desc(a_addr, a_lbo, 1024u), bdesc = umma_smem_desc(a_addr + OPERAND, b_lbo, 1024u);
          if (!spin_wait(tempty_bar(buf), buf_phase ^ 1u, abort_flag, p.status, ST_FP8_BLOCK + 2)) { ok = false; break; }
          tc_fence_after();
          const uint32_t d = tmem_base + buf * TN;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (PAIR) umma_fp8_pair(d, adesc + k * a_step, bdesc + k * b_step, idesc, k != 0);
            else umma_fp8(d, adesc + k * a_step, bdesc + k * b_step, idesc, k != 0);
          }
          if (PAIR) { umma_commit_pair(tfull_bar(buf)); umma_commit_pair(empty_bar(stage)); }
          else { umma_commit(tfull_bar(buf)); umma_commit(empty_bar(stage)); }
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
          if (++buf == BUFS) { buf = 0; buf_phase ^= 1u; }
        }
    }
    if (warp == 2) {
      int n = 0;                                                   // k-blocks so far, over all tiles
      bool ok = true;
      for (int tile = worker; tile < num_tiles && ok; tile += workers) {
        int mt, nt; raster(tile, m_tiles, n_tiles, mt, nt);
        const int m0 = mt * TM + int(rank) * 128, n0 = nt * TN;
        for (int kb = 0; kb < num_kb; ++kb, ++n) {
          const int group = n / GROUP & 1;
          if (n % GROUP == 0 && !mbar_wait(sempty_bar(group), (n / SLOTS & 1) ^ 1, abort_flag, p.status, ST_FP8_BLOCK + 5)) { ok = false; break; }
          const uint32_t at = smem_base + S::SLOT + (n % SLOTS) * SLOT_BYTES;
          const float *sa = p.sa + kb * p.sa_k, *sb = p.sb + kb * p.sb_k;
          if (p.runs) {
            const int m = m0 + 4 * lane;
            copy16(at + 16 * lane, m < p.M ? sa + m : sa, p.M - m);
            if (SB_ROWS) {
#pragma unroll
              for (int j = 0; j < TN / 128; ++j) {
                const int c = n0 + 128 * j + 4 * lane;
                copy16(at + (128 + 128 * j) * 4 + 16 * lane, c < p.N ? sb + c : sb, p.N - c);
              }
            }
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int m = m0 + 32 * j + lane;
              copy4(at + (32 * j + lane) * 4, m < p.M ? sa + m * p.sa_m : sa, m < p.M);
            }
            if (SB_ROWS) {
#pragma unroll
              for (int j = 0; j < TN / 32; ++j) {
                const int c = n0 + 32 * j + lane;
                copy4(at + (128 + 32 * j + lane) * 4, c < p.N ? sb + c * p.sb_n : sb, c < p.N);
              }
            }
          }
          if (!SB_ROWS && lane < TN / 128) {
            const int c = n0 + 128 * lane;
            copy4(at + (128 + lane) * 4, c < p.N ? sb + (c / BLOCK) * p.sb_n : sb, c < p.N);
          }
          if (n % GROUP == GROUP - 1) copies_arrive(sfull_bar(group));
        }
      }
      if (n % GROUP) copies_arrive(sfull_bar(n / GROUP & 1));      // the last group may be a short one
      asm volatile("cp.async.wait_all;" ::: "memory");
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_MANY));
    const int q = warp & 3, half = (warp - 4) >> 2;
    const uint32_t space = smem_base + S::OUT + (warp - 4) * (S::BOXES * S::BOX);
    const uint32_t t_warp = tmem_base + (uint32_t(q * 32) << 16) + half * COLS;
    const uint32_t tempty_0 = map_to_cta(tempty_bar(0), 0);        // the even CTA's
    int buf = 0, n = 0; uint32_t buf_phase = 0;                    // n: k-blocks so far, over all tiles
    const uint32_t slot_0 = smem_base + S::SLOT;
    bool ok = true;
    for (int tile = worker; tile < num_tiles && ok; tile += workers) {
      int mt, nt; raster(tile, m_tiles, n_tiles, mt, nt);
      const int row0 = mt * TM + int(rank) * 128 + q * 32, col0 = nt * TN + half * COLS;
      f2 acc[COLS / 2];
#pragma unroll
      for (int j = 0; j < COLS / 2; ++j) acc[j] = 0ull;
      for (int kb = 0; kb < num_kb; ++kb) {
        const int group = n / GROUP & 1;
        if (n % GROUP == 0 && !spin_wait(sfull_bar(group), n / SLOTS & 1, abort_flag, p.status, ST_FP8_BLOCK + 6)) { ok = false; break; }
        const uint32_t at = slot_0 + (n % SLOTS) * SLOT_BYTES, sb_k = at + (128 + half * COLS) * 4;
        f2 s[SB_ROWS ? 4 : 1];                                     // scales of the lane's rows
        if (SB_ROWS) {
#pragma unroll
          for (int k = 0; k < 4; ++k) { const float v = get1(at + (q * 32 + (lane >> 2) + 8 * k) * 4); s[k] = f2_pack(v, v); }
        } else {
          const float v = get1(at + (q * 32 + lane) * 4) * get1(at + (128 + (PAIR ? half : 0)) * 4);
          s[0] = f2_pack(v, v);
        }
        const uint32_t t = t_warp + buf * TN;
        uint32_t r0[32], r1[32];
        auto load = [&](int c, uint32_t (&r)[32]) {
          if (SB_ROWS) load_fragments(t + 32 * c, r);
          else tmem_ld_32x32(t + 32 * c, r);
        };
        // scales of the lane's two columns of eight, fetched one eight ahead
        const uint32_t sb_lane = sb_k + 2 * (lane & 3) * 4;
        f2 b_next = SB_ROWS ? get2(sb_lane) : 0ull;
        auto add = [&](int c, const uint32_t (&r)[32]) {
          if (SB_ROWS) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const f2 b = b_next;
              if (c * 4 + i + 1 < COLS / 8) b_next = get2(sb_lane + (c * 4 + i + 1) * 32);
              f2 v[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) v[k] = scaled(r[(k >> 1) * 16 + i * 4 + (k & 1) * 2], r[(k >> 1) * 16 + i * 4 + (k & 1) * 2 + 1], b);
#pragma unroll
              for (int k = 0; k < 4; ++k) acc[c * 16 + (k >> 1) * 8 + i * 2 + (k & 1)] = f2_fma(v[k], s[SB_ROWS ? k : 0], acc[c * 16 + (k >> 1) * 8 + i * 2 + (k & 1)]);
            }
          } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) add_scaled(acc[c * 16 + j], r[2 * j], r[2 * j + 1], s[0]);
          }
        };
        if (!spin_wait(tfull_bar(buf), buf_phase, abort_flag, p.status, ST_FP8_BLOCK + 4)) { ok = false; break; }
        __syncwarp();
        tc_fence_after();
        load(0, r0);
        load(1, r1);
        tmem_wait_ld();
        if (COLS == 128) {
          add(0, r0);
          load(2, r0);
          add(1, r1);
          load(3, r1);
          tmem_wait_ld();
        }
        tc_fence_before();
        __syncwarp();
        arrive_relaxed(tempty_0 + 8u * buf, lane == 0);            // all read: the buffer is free again
        add(COLS / 32 - 2, r0);
        add(COLS / 32 - 1, r1);
        if (n % GROUP == GROUP - 1) {                              // this group's scales have been read by the whole warp
          __syncwarp();
          if (lane == 0) mbar_arrive(sempty_bar(group));
        }
        if (++buf == BUFS) { buf = 0; buf_phase ^= 1u; }
        ++n;
      }
      if (!ok) break;
      store_tile<COLS, SB_ROWS>(p, &tmC, space, acc, row0, col0, lane);
    }
    if (lane == 0) bulk_wait<0>();
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) { cluster_arrive(); cluster_wait(); }                  // neither CTA leaves while its partner can still signal it or read its memory
  if (warp == 1) {
    tc_fence_after();
    if (PAIR) tmem_dealloc_pair(tmem_base, 512);
    else tmem_dealloc(tmem_base, 512);
  }
}

// Whether an [M, N] product goes by 256 x 256 tiles on CTA pairs: where 128 x 128 tiles need more than 1.4 times as many waves, for a weight gradient
// (scales for single columns) 1.7 times.  Fitted to, us in a graph, pairs and single (waves):
//   forward, K = 4096   2304 x 2304 32.8, 32.6 (2, 3)   3712 x 3712 59.4, 61.4 (4, 6)   4480 x 4224 74.8, 82.4 (5, 8)   4096 x 4096 63.3, 72.9 (4, 7)
//                       512 x 4096 19.0, 14.0 (1, 1)    1100 x 2100 32.8, 35.1 (1, 2)   8192 x 12288 342, 435 (21, 42); input gradients alike
//   weight, K = 8192    2304 x 2304 90.9, 80.5 (2, 3)   3712 x 3712 176, 158 (4, 6)     4480 x 4224 220, 208 (5, 8)     4096 x 4096 179, 182 (4, 7)
//                       1024 x 1024 48.1, 29.0 (1, 1)   2048 x 2048 50.0, 55.9 (1, 2)   12288 x 4096 493, 581 (11, 21)
// Short contractions would want the smaller tiles up to 1.75 times the waves (forward, K = 1024: 2304 x 2304 14.4, 12.0; 4096 x 4096 24.4, 24.5).
static bool goes_by_pairs(int M, int N, bool columns, int sms) {
  auto waves = [](long long tiles, long long slots) { return (tiles + slots - 1) / slots; };
  const long long pair = waves((long long)((M + 255) / 256) * ((N + 255) / 256), sms / 2),
                  single = waves((long long)((M + 127) / 128) * ((N + 127) / 128), sms);
  return 10 * single > (columns ? 17 : 14) * pair;
}

template <bool PAIR, int A_MN, int B_MN, bool SB_ROWS>
static int launch(const CUtensorMap& tmA, const CUtensorMap& tmB, const CUtensorMap& tmC, const GemmArgs& p, cudaStream_t stream) {
  auto kern = gemm_fp8_block_kernel<PAIR, A_MN, B_MN, SB_ROWS>;
  static std::atomic<unsigned long long> allowed{0};       // devices that know the kernel's shared memory
  if (!allow_shared(allowed, kern, Space<PAIR>::BYTES)) return -5;
  // the split of the registers waits for good where a block has fewer of them than it deals out
  static const int regs = [] {
    cudaFuncAttributes a;
    return cudaFuncGetAttributes(&a, gemm_fp8_block_kernel<PAIR, A_MN, B_MN, SB_ROWS>) == cudaSuccess ? a.numRegs : 0;
  }();
  if (regs * NUM_THREADS < 128 * REGS_FEW + 32 * EPI_WARPS * REGS_MANY) return -7;
  constexpr int T = PAIR ? 256 : 128;
  const long long tiles = (long long)((p.M + T - 1) / T) * ((p.N + T - 1) / T), slots = PAIR ? num_sms() / 2 : num_sms();
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned((tiles < slots ? tiles : slots) * (PAIR ? 2 : 1)));
  cfg.blockDim = dim3(NUM_THREADS);
  cfg.dynamicSmemBytes = Space<PAIR>::BYTES;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = PAIR ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, kern, tmA, tmB, tmC, p) == cudaSuccess) return 0;
  (void)cudaGetLastError();
  return -6;
}

}  // namespace blk8
}  // namespace sb

// Whether an [M, N] product, or a weight gradient, goes by 256 x 256 tiles on CTA pairs.
extern "C" int sb_gemm_fp8_block_goes_by_pairs(int M, int N) { return sb::blk8::goes_by_pairs(M, N, false, sb::num_sms()); }
extern "C" int sb_gemm_fp8_block_weight_goes_by_pairs(int M, int N) { return sb::blk8::goes_by_pairs(M, N, true, sb::num_sms()); }

// C [M, N] of type 0 bf16, 1 fp16, 2 fp32 (bias, residual and a C that is added to: of the same type).  A: [M, K], or stored as [K, M] (a_mn);
// B: [N, K] or [K, N] (b_mn); bytes, rows lda / ldb apart, 16-byte boundaries.  Scale of A at sa[m * sa_m + (k / 128) * sa_k], of B at
// sb[n * sb_n + (k / 128) * sb_k] (sb_rows) or sb[(n / 128) * sb_n + (k / 128) * sb_k].  Forms: neither operand transposed, B, or both with sb_rows
// (a weight gradient's: without bias and residual).
extern "C" int sb_gemm_fp8_block(const void* A, const float* sa, long long sa_m, long long sa_k, const void* B, const float* sb, long long sb_n,
                                 long long sb_k, int sb_rows, void* C, const void* bias, const void* residual, int M, int N, int K,
                                 long long lda, long long ldb, long long ldc, long long ldr, int a_mn, int b_mn, int type, int beta, unsigned int* status,
                                 cudaStream_t stream) {
  using namespace sb;
  using namespace sb::blk8;
  if (M <= 0 || N <= 0) return 0;
  if (K <= 0 || (sb_rows && (bias || residual))) return -3;
  if (!bind_context()) return -5;                        // the tensor-map encoder needs a current context
  if ((lda % 16) || (ldb % 16) || ((reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(B)) & 15)) return -4;
  if ((long long)((M + 127) / 128) * ((N + 127) / 128) > 0x7fffffffLL) return -3;
  CUtensorMap tmA, tmB, tmC = {};
  int rc;
  if ((rc = a_mn ? make_tmap_2d_u8(&tmA, A, M, K, lda, 128, 128) : make_tmap_2d_u8(&tmA, A, K, M, lda, 128, 128))) return rc;
  if ((rc = b_mn ? make_tmap_2d_u8(&tmB, B, N, K, ldb, 128, 128) : make_tmap_2d_u8(&tmB, B, K, N, ldb, 128, 128))) return rc;
  const int size = type == 2 ? 4 : 2;
  const auto on16 = [](const void* at, long long row_bytes) { return !((reinterpret_cast<uintptr_t>(at) | row_bytes) & 15); };
  const bool boxes = !(type == 2 && sb_rows) && N % 8 == 0 && N < (1 << 30) && on16(C, ldc * size) && on16(bias, 0) && (!residual || on16(residual, ldr * size));
  const bool runs = sa_m == 1 && on16(sa, sa_k * 4) && (!sb_rows || (sb_n == 1 && on16(sb, sb_k * 4)));
  const int halves = size / 2;                           // the map is in 16-bit units, whatever the type
  if (boxes && (rc = make_tmap_2d_bf16(&tmC, C, (uint64_t)N * halves, M, ldc * halves, 64, 32))) return rc;
  GemmArgs p{C, bias, residual, sa, sb, sa_m, sa_k, sb_n, sb_k, ldc, ldr, M, N, K, type, beta, boxes, runs, status};
  const bool pair = goes_by_pairs(M, N, sb_rows != 0, num_sms());
  if (!a_mn && !b_mn && !sb_rows) return pair ? launch<true, 0, 0, false>(tmA, tmB, tmC, p, stream) : launch<false, 0, 0, false>(tmA, tmB, tmC, p, stream);
  if (!a_mn && b_mn && !sb_rows) return pair ? launch<true, 0, 1, false>(tmA, tmB, tmC, p, stream) : launch<false, 0, 1, false>(tmA, tmB, tmC, p, stream);
  if (a_mn && b_mn && sb_rows) return pair ? launch<true, 1, 1, true>(tmA, tmB, tmC, p, stream) : launch<false, 1, 1, true>(tmA, tmB, tmC, p, stream);
  return -3;
}
