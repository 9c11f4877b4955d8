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
//   warps 4-11 a lane owns a row and half of the tile's columns: tcgen05.ld of 16 columns, eight packed multiply-adds, while the next 16 are on
//              their way; after the last k-block the sums leave through shared memory in whole sectors
//
// Two tiles: 256 x 256 on a CTA pair (cta_group::2; two buffers of 256 columns, 128 sums a thread) and 128 x 128 on one CTA (four buffers of
// 128, 64 sums), for outputs that leave the chip idle in the larger one.
//
// A programmatic dependent of the kernel before it (pdl.cuh, the second kind).  All waits are bounded (sm100.cuh).
#include "entries.h"
#include "f32x2.cuh"
#include "fp8_block.cuh"
#include "pdl.cuh"
#include "sm100.cuh"

namespace sb {

int make_tmap_2d_u8(CUtensorMap* out, const void* base, uint64_t inner, uint64_t outer, uint64_t ld, uint32_t box_inner, uint32_t box_outer);

namespace blk8 {

struct GemmArgs {
  void* C;
  const void *bias, *residual;
  const float *sa, *sb;
  long long sa_m, sa_k, sb_n, sb_k;      // strides; sb_n counts blocks of 128 n where the scale is theirs
  long long ldc, ldr;
  int M, N, K, type, beta, vec;          // vec: rows of C and residual on 16-byte boundaries
  uint32_t* status;
};

constexpr int EPI_WARPS = 8, NUM_THREADS = 128 + 32 * EPI_WARPS;
// Registers: 168 a thread at launch (384 threads), of which the first four warps keep 40 and each of the other eight gets 232:
// 128 * 40 + 256 * 232 = 384 * 168.
constexpr int REGS_FEW = 40, REGS_MANY = 232;
static_assert(128 * REGS_FEW + 32 * EPI_WARPS * REGS_MANY <= NUM_THREADS * 168, "registers of a block");
constexpr int STAGES = 6, OPERAND = 128 * 128, STAGE_BYTES = 2 * OPERAND;
constexpr int BAR_OFF = STAGES * STAGE_BYTES, OUT_OFF = BAR_OFF + 256, OUT_BYTES = 32 * 64;      // a warp's 32 rows x 16 fp32 on their way out
constexpr int SB_OFF = OUT_OFF + EPI_WARPS * OUT_BYTES, SB_BYTES = 2 * 128 * 4;                  // a warp's column scales of two k-blocks
constexpr int SMEM_BYTES = SB_OFF + EPI_WARPS * SB_BYTES + 1024;
static_assert(SMEM_BYTES <= 232448, "shared memory of a block");
constexpr int GROUP_M = 8;               // raster: m-tiles that share the concurrently running n-tiles

__device__ __forceinline__ void raster(int tile, int m_tiles, int n_tiles, int& mt, int& nt) {
  const int per_group = GROUP_M * n_tiles, g = tile / per_group, first = g * GROUP_M, size = min(GROUP_M, m_tiles - first), r = tile - g * per_group;
  mt = first + r % size;
  nt = r / size;
}

__device__ __forceinline__ void load16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// the registers pass through the wait: nothing that uses them can move ahead of it
__device__ __forceinline__ void arrived(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                 "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}
__device__ __forceinline__ f2 pair_of(uint32_t a, uint32_t b) { return f2_pack(__uint_as_float(a), __uint_as_float(b)); }
__device__ __forceinline__ void put4(uint32_t at, float a, float b, float c, float d) {
  asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}
__device__ __forceinline__ float4 get4(uint32_t at) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
  return v;
}

template <class T>
__device__ __forceinline__ void add8(const T* p, int n, bool vec, float (&f)[8]) {
  float t[8];
  unpack(vec && n == 8 ? fetch<true, T>(p, 8) : fetch<false, T>(p, n), t);
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] += t[j];
}
// n of the eight sums of one row from column col on
template <class T>
__device__ __forceinline__ void finish8(const GemmArgs& p, int row, int col, int n, float (&f)[8]) {
  T* c = static_cast<T*>(p.C) + row * p.ldc + col;
  if (p.bias) add8(static_cast<const T*>(p.bias) + col, n, false, f);
  if (p.residual) add8(static_cast<const T*>(p.residual) + row * p.ldr + col, n, p.vec, f);
  if (p.beta) add8(c, n, p.vec, f);
  if (p.vec && n == 8) put<true, T>(c, pack<T>(f), 8);
  else put<false, T>(c, pack<T>(f), n);
}
// 16 sums of each of the warp's 32 rows, a lane a row, to memory.  Chunks of 16 bytes are permuted so that neither side meets a bank twice.
__device__ __forceinline__ void store16(const GemmArgs& p, uint32_t stage, const f2* acc, int row0, int col0, int lane) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const float2 a = f2_unpack(acc[2 * c]), b = f2_unpack(acc[2 * c + 1]);
    put4(stage + lane * 64 + ((c ^ (lane >> 1 & 3)) << 4), a.x, a.y, b.x, b.y);
  }
  __syncwarp();
  const int g = lane & 1, col = col0 + 8 * g, n = min(8, p.N - col);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 16 * i + (lane >> 1), x = r >> 1 & 3;
    const float4 a = get4(stage + r * 64 + ((2 * g ^ x) << 4)), b = get4(stage + r * 64 + (((2 * g + 1) ^ x) << 4));
    float f[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    if (row0 + r < p.M && n > 0) {
      if (p.type == 0) finish8<bf16>(p, row0 + r, col, n, f);
      else if (p.type == 1) finish8<__half>(p, row0 + r, col, n, f);
      else finish8<float>(p, row0 + r, col, n, f);
    }
  }
  __syncwarp();
}

template <bool PAIR, int A_MN, int B_MN, bool SB_ROWS>
__global__ void __launch_bounds__(NUM_THREADS, 1)
gemm_fp8_block_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, GemmArgs p) {
  constexpr int TM = PAIR ? 256 : 128, TN = PAIR ? 256 : 128, BUFS = 512 / TN, COLS = TN / 2;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t bar_base = smem_base + BAR_OFF;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (STAGES + s); };
  auto tfull_bar = [&](int b) { return bar_base + 8u * (2 * STAGES + b); };
  auto tempty_bar = [&](int b) { return bar_base + 8u * (2 * STAGES + 4 + b); };
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem_gen + BAR_OFF + 8 * (2 * STAGES + 8));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem_gen + BAR_OFF + 8 * (2 * STAGES + 8) + 8);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0u;             // 0 issues the products, 1 is its partner
  const int worker = PAIR ? blockIdx.x >> 1 : blockIdx.x, workers = PAIR ? gridDim.x >> 1 : gridDim.x;
  const int m_tiles = (p.M + TM - 1) / TM, n_tiles = (p.N + TN - 1) / TN, num_tiles = m_tiles * n_tiles;
  const int num_kb = (p.K + BLOCK - 1) / BLOCK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 1); }
    for (int b = 0; b < BUFS; ++b) { mbar_init(tfull_bar(b), 1); mbar_init(tempty_bar(b), (PAIR ? 2 : 1) * EPI_WARPS); }
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmB);
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
          if (!mbar_wait(tempty_bar(buf), buf_phase ^ 1u, abort_flag, p.status, ST_FP8_BLOCK + 2) ||
              !mbar_wait(full_bar(stage), phase, abort_flag, p.status, ST_FP8_BLOCK + 3)) { ok = false; break; }
          tc_fence_after();
          const uint32_t a_addr = smem_base + stage * STAGE_BYTES;
          const uint64_t adesc = umma_smem_desc(a_addr, a_lbo, 1024u), bdesc = umma_smem_desc(a_addr + OPERAND, b_lbo, 1024u);
          const uint32_t d = tmem_base + buf * TN;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (PAIR) umma_fp8_pair(d, adesc + k * a_step, bdesc + k * b_step, idesc, k != 0);
            else umma_fp8(d, adesc + k * a_step, bdesc + k * b_step, idesc, k != 0);
          }
          if (PAIR) { umma_commit_pair(empty_bar(stage)); umma_commit_pair(tfull_bar(buf)); }
          else { umma_commit(empty_bar(stage)); umma_commit(tfull_bar(buf)); }
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
          if (++buf == BUFS) { buf = 0; buf_phase ^= 1u; }
        }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_MANY));
    const int q = warp & 3, half = (warp - 4) >> 2;
    const uint32_t stage_w = smem_base + OUT_OFF + (warp - 4) * OUT_BYTES, sb_w = smem_base + SB_OFF + (warp - 4) * SB_BYTES;
    int buf = 0; uint32_t buf_phase = 0;
    bool ok = true;
    for (int tile = worker; tile < num_tiles && ok; tile += workers) {
      int mt, nt; raster(tile, m_tiles, n_tiles, mt, nt);
      const int row0 = mt * TM + int(rank) * 128 + q * 32, col0 = nt * TN + half * COLS;
      const float* sa = p.sa + (long long)min(row0 + lane, p.M - 1) * p.sa_m;
      const float* sb = SB_ROWS ? p.sb : p.sb + (min(col0, p.N - 1) / BLOCK) * p.sb_n;
      // the scales of a k-block are fetched two k-blocks ahead
      float a_next[2], b_next[2];
      float c_next[COLS / 32];
      auto columns = [&](int kb) {
#pragma unroll
        for (int j = 0; j < COLS / 32; ++j) {
          const int c = col0 + lane + 32 * j;
          c_next[j] = c < p.N && kb < num_kb ? sb[c * p.sb_n + kb * p.sb_k] : 0.f;
        }
      };
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        a_next[k] = k < num_kb ? sa[k * p.sa_k] : 0.f;
        b_next[k] = !SB_ROWS && k < num_kb ? sb[k * p.sb_k] : 0.f;
      }
      if (SB_ROWS) columns(0);
      f2 acc[COLS / 2];
#pragma unroll
      for (int j = 0; j < COLS / 2; ++j) acc[j] = 0ull;
      for (int kb = 0; kb < num_kb; ++kb) {
        float s = a_next[0];
        const uint32_t sb_k = sb_w + (kb & 1) * (SB_BYTES / 2);
        if (SB_ROWS) {
#pragma unroll
          for (int j = 0; j < COLS / 32; ++j) asm volatile("st.shared.f32 [%0], %1;" ::"r"(sb_k + (lane + 32 * j) * 4), "f"(c_next[j]) : "memory");
          __syncwarp();
          columns(kb + 1);
        } else {
          s *= b_next[0];
        }
        a_next[0] = a_next[1]; b_next[0] = b_next[1];
        if (kb + 2 < num_kb) {
          a_next[1] = sa[(kb + 2) * p.sa_k];
          if (!SB_ROWS) b_next[1] = sb[(kb + 2) * p.sb_k];
        }
        const f2 s2 = f2_pack(s, s);
        if (!mbar_wait(tfull_bar(buf), buf_phase, abort_flag, p.status, ST_FP8_BLOCK + 4)) { ok = false; break; }
        tc_fence_after();
        const uint32_t t = tmem_base + (uint32_t(q * 32) << 16) + buf * TN + half * COLS;
        auto add = [&](int c, const uint32_t (&r)[16]) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (SB_ROWS) {
              const float4 b = get4(sb_k + (c * 16 + 4 * j) * 4);
              acc[c * 8 + 2 * j] = f2_fma(pair_of(r[4 * j], r[4 * j + 1]), f2_mul(f2_pack(b.x, b.y), s2), acc[c * 8 + 2 * j]);
              acc[c * 8 + 2 * j + 1] = f2_fma(pair_of(r[4 * j + 2], r[4 * j + 3]), f2_mul(f2_pack(b.z, b.w), s2), acc[c * 8 + 2 * j + 1]);
            } else {
              acc[c * 8 + 2 * j] = f2_fma(pair_of(r[4 * j], r[4 * j + 1]), s2, acc[c * 8 + 2 * j]);
              acc[c * 8 + 2 * j + 1] = f2_fma(pair_of(r[4 * j + 2], r[4 * j + 3]), s2, acc[c * 8 + 2 * j + 1]);
            }
          }
        };
        uint32_t r0[16], r1[16];
        load16(t, r0);
#pragma unroll
        for (int c = 0; c < COLS / 16; c += 2) {
          arrived(r0);
          load16(t + (c + 1) * 16, r1);
          add(c, r0);
          arrived(r1);
          if (c + 2 < COLS / 16) load16(t + (c + 2) * 16, r0);
          else {                                                   // all read: the buffer is free again
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              if (PAIR) mbar_arrive_cluster(map_to_cta(tempty_bar(buf), 0));
              else mbar_arrive(tempty_bar(buf));
            }
          }
          add(c + 1, r1);
        }
        if (++buf == BUFS) { buf = 0; buf_phase ^= 1u; }
      }
      if (!ok) break;
#pragma unroll
      for (int c = 0; c < COLS / 16; ++c)
        if (col0 + c * 16 < p.N) store16(p, stage_w, acc + c * 8, row0, col0 + c * 16, lane);
    }
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

// Whether an [M, N] product goes by 256 x 256 tiles on CTA pairs: waves of either tile times what a k-block of it takes.
static bool goes_by_pairs(int M, int N, int sms) {
  auto waves = [](long long tiles, long long slots) { return (tiles + slots - 1) / slots; };
  const long long pair = waves((long long)((M + 255) / 256) * ((N + 255) / 256), sms / 2) * 512,
                  single = waves((long long)((M + 127) / 128) * ((N + 127) / 128), sms) * 320;
  return 8 * single > 7 * pair;
}

template <bool PAIR, int A_MN, int B_MN, bool SB_ROWS>
static int launch(const CUtensorMap& tmA, const CUtensorMap& tmB, const GemmArgs& p, cudaStream_t stream) {
  auto kern = gemm_fp8_block_kernel<PAIR, A_MN, B_MN, SB_ROWS>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES) != cudaSuccess) return -5;
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
  cfg.dynamicSmemBytes = SMEM_BYTES;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = PAIR ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, kern, tmA, tmB, p) == cudaSuccess) return 0;
  (void)cudaGetLastError();
  return -6;
}

}  // namespace blk8
}  // namespace sb

// C [M, N] of type 0 bf16, 1 fp16, 2 fp32 (bias, residual and a C that is added to: of the same type).  A: [M, K], or stored as [K, M] (a_mn);
// B: [N, K] or [K, N] (b_mn); bytes, rows lda / ldb apart, 16-byte boundaries.  Scale of A at sa[m * sa_m + (k / 128) * sa_k], of B at
// sb[n * sb_n + (k / 128) * sb_k] (sb_rows) or sb[(n / 128) * sb_n + (k / 128) * sb_k].  Forms: neither operand transposed, B, or both with sb_rows.
extern "C" int sb_gemm_fp8_block(const void* A, const float* sa, long long sa_m, long long sa_k, const void* B, const float* sb, long long sb_n,
                                 long long sb_k, int sb_rows, void* C, const void* bias, const void* residual, int M, int N, int K,
                                 long long lda, long long ldb, long long ldc, long long ldr, int a_mn, int b_mn, int type, int beta, unsigned int* status,
                                 cudaStream_t stream) {
  using namespace sb;
  using namespace sb::blk8;
  if (M <= 0 || N <= 0) return 0;
  if (K <= 0) return -3;
  static thread_local bool ctx_bound = false;            // the tensor-map encoder needs a current context
  if (!ctx_bound) { cudaFree(0); ctx_bound = true; }
  if ((lda % 16) || (ldb % 16) || ((reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(B)) & 15)) return -4;
  if ((long long)((M + 127) / 128) * ((N + 127) / 128) > 0x7fffffffLL) return -3;
  CUtensorMap tmA, tmB;
  int rc;
  if ((rc = a_mn ? make_tmap_2d_u8(&tmA, A, M, K, lda, 128, 128) : make_tmap_2d_u8(&tmA, A, K, M, lda, 128, 128))) return rc;
  if ((rc = b_mn ? make_tmap_2d_u8(&tmB, B, N, K, ldb, 128, 128) : make_tmap_2d_u8(&tmB, B, K, N, ldb, 128, 128))) return rc;
  const int size = type == 2 ? 4 : 2;
  const bool vec = reinterpret_cast<uintptr_t>(C) % 16 == 0 && ldc * size % 16 == 0 &&
                   (!residual || (reinterpret_cast<uintptr_t>(residual) % 16 == 0 && ldr * size % 16 == 0));
  GemmArgs p{C, bias, residual, sa, sb, sa_m, sa_k, sb_n, sb_k, ldc, ldr, M, N, K, type, beta, vec, status};
  const bool pair = goes_by_pairs(M, N, num_sms());
  if (!a_mn && !b_mn && !sb_rows) return pair ? launch<true, 0, 0, false>(tmA, tmB, p, stream) : launch<false, 0, 0, false>(tmA, tmB, p, stream);
  if (!a_mn && b_mn && !sb_rows) return pair ? launch<true, 0, 1, false>(tmA, tmB, p, stream) : launch<false, 0, 1, false>(tmA, tmB, p, stream);
  if (a_mn && b_mn && sb_rows) return pair ? launch<true, 1, 1, true>(tmA, tmB, p, stream) : launch<false, 1, 1, true>(tmA, tmB, p, stream);
  return -3;
}
