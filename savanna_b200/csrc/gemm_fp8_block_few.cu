// The block-scaled product (gemm_fp8_block.cu) for few tokens, a decode step's or a short prompt's:
//
//   y[t, n] = sum_kb sx[t, kb] * sw[n / 128, kb] * (sum over the block's 128 k of X[t, k] * W[n, k])  (+ bias[n]) (+ residual[t, n])
//
// Bound by reading the weights once, one byte each.  The weights are the tensor cores' rows (128 of them a tile) and the tokens their
// columns (TOK = 16, 32 or 64), so that nothing but weights takes room in the stages; with the tokens as rows, 16 of 128 would be in use.
// The CTAs of a cluster share a tile's k-blocks (as many of them as it takes to give every SM work), two CTAs fit on an SM, and each has
// 80 to 100 KB of operands on their way.  A k-block's product is read from TMEM and added, scaled, in fp32; the CTAs' sums are joined through
// distributed shared memory in a fixed order.
//
// 1 x 4096 x 12288: 12.7 us back to back on the same weights, 14.4 with others each time (the bytes alone 7.7), 13.6 on the same with the quantiser before it.
// What is left: an uneven share (with two parts 44 SMs have two CTAs and 104 one, so that the fullest reads 524 KB of weights where an even share is 340),
// a launch, barriers and tensor memory, the first loads' way and the join.  More parts than it takes to reach every SM cost more than they give (2 parts
// 12.5 us, 3 17, 4 15.4, 8 19.0; one 13.0); so do clusters that do not all find room at once (34 to 36 tiles in eight parts, 72 and 73 in four: T = 1, K = 4096,
// 33 tiles 8.2 us, 34 11.4, 37 8.5; 71 10.6, 72 14.5, 74 11.9).
//
// A link of a chain (pdl.cuh, the first kind) behind the kernel that quantises X, which lets it start when all before itself is complete: the first
// stages' weights, which do not depend on that kernel, are on their way before it has ended.  All waits are bounded (sm100.cuh).
#include "entries.h"
#include "fp8_block.cuh"
#include "pdl.cuh"
#include "sm100.cuh"

namespace sb {

int make_tmap_2d_u8(CUtensorMap* out, const void* base, uint64_t inner, uint64_t outer, uint64_t ld, uint32_t box_inner, uint32_t box_outer);

namespace blk8 {

struct FewArgs {
  const float *sx, *sw;
  long long sx_m, sx_k, sw_n, sw_k, ldc, ldr;
  void* y;
  const void *bias, *residual;
  int M, N, K, type;
  uint32_t* status;
};

template <int TOK> struct FewSpace {
  static constexpr int STAGES = TOK == 64 ? 4 : 5, W = 128 * 128, STAGE = W + TOK * 128, GROUP = 16;
  static constexpr int SCALES = STAGES * STAGE, BAR = SCALES + GROUP * TOK * 4, BYTES = BAR + 256 + 1024;
  static constexpr int BUFS = TOK == 64 ? 4 : 8;
  static_assert(2 * (BYTES + 1024) <= 233472 && TOK * 512 <= SCALES, "two blocks of an SM; the sums fit where the stages were");
};

__device__ __forceinline__ void epilogue_barrier() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ float4 peer_floats(uint32_t cluster_addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(cluster_addr) : "memory");
  return v;
}
template <int TOK> __device__ __forceinline__ void load_columns(uint32_t taddr, uint32_t (&r)[TOK]) {
#pragma unroll
  for (int c = 0; c < TOK; c += 16)
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[c]), "=r"(r[c + 1]), "=r"(r[c + 2]), "=r"(r[c + 3]), "=r"(r[c + 4]), "=r"(r[c + 5]), "=r"(r[c + 6]), "=r"(r[c + 7]), "=r"(r[c + 8]),
          "=r"(r[c + 9]), "=r"(r[c + 10]), "=r"(r[c + 11]), "=r"(r[c + 12]), "=r"(r[c + 13]), "=r"(r[c + 14]), "=r"(r[c + 15])
        : "r"(taddr + c)
        : "memory");
}
// four results of token t from row n on
template <class T> __device__ __forceinline__ void finish(const FewArgs& p, int t, int n, const float (&f)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (n + j >= p.N) return;
    float v = f[j];
    if (p.bias) v += up(static_cast<const T*>(p.bias)[n + j]);
    if (p.residual) v += up(static_cast<const T*>(p.residual)[t * p.ldr + n + j]);
    static_cast<T*>(p.y)[t * p.ldc + n + j] = down<T>(v);
  }
}

template <int TOK>
__global__ void __launch_bounds__(192, 2)
gemm_fp8_block_few_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, FewArgs p, int parts) {
  typedef FewSpace<TOK> S;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t bar_base = smem_base + S::BAR;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (S::STAGES + s); };
  auto tfull_bar = [&](int b) { return bar_base + 8u * (2 * S::STAGES + b); };
  auto tempty_bar = [&](int b) { return bar_base + 8u * (2 * S::STAGES + S::BUFS + b); };
  constexpr int FLAGS = S::BAR + 8 * (2 * S::STAGES + 2 * S::BUFS);
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem_gen + FLAGS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem_gen + FLAGS + 8);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = blockIdx.x % parts, n0 = (blockIdx.x / parts) * 128;
  const int kbs = (p.K + BLOCK - 1) / BLOCK, kb0 = int((long long)kbs * part / parts), kb1 = int((long long)kbs * (part + 1) / parts);

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::STAGES; ++s) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 1); }
    for (int b = 0; b < S::BUFS; ++b) { mbar_init(tfull_bar(b), 1); mbar_init(tempty_bar(b), 4); }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), 256);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (elect_one()) {
      // the weights of the first stages, then what the kernel before this one wrote
      const int ahead = min(S::STAGES, kb1 - kb0);
      for (int i = 0; i < ahead; ++i) {
        mbar_expect_tx(full_bar(i), S::STAGE);
        tma_load_2d(smem_base + i * S::STAGE, &tmW, (kb0 + i) * BLOCK, n0, full_bar(i));
      }
      wait_for_previous();
      for (int i = 0; i < ahead; ++i) tma_load_2d(smem_base + i * S::STAGE + S::W, &tmX, (kb0 + i) * BLOCK, 0, full_bar(i));
      int stage = 0; uint32_t phase = 0;
      for (int kb = kb0 + ahead; kb < kb1; ++kb) {
        if (!mbar_wait(empty_bar(stage), phase, abort_flag, p.status, ST_FP8_FEW + 1)) {
          const unsigned long long t0 = globaltimer();             // copies in flight land before the block ends
          while (globaltimer() - t0 < 200000ull) { __nanosleep(1000); }
          break;
        }
        mbar_expect_tx(full_bar(stage), S::STAGE);
        tma_load_2d(smem_base + stage * S::STAGE, &tmW, kb * BLOCK, n0, full_bar(stage));
        tma_load_2d(smem_base + stage * S::STAGE + S::W, &tmX, kb * BLOCK, 0, full_bar(stage));
        if (++stage == S::STAGES) { stage = 0; phase ^= 1u; }
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t idesc = umma_idesc_fp8(128, TOK, 0, 0, 0, 0);
      int stage = 0, buf = 0; uint32_t phase = 0, buf_phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(full_bar(stage), phase, abort_flag, p.status, ST_FP8_FEW + 2) ||
            !mbar_wait(tempty_bar(buf), buf_phase ^ 1u, abort_flag, p.status, ST_FP8_FEW + 3)) break;
        tc_fence_after();
        const uint32_t at = smem_base + stage * S::STAGE;
        const uint64_t wdesc = umma_smem_desc(at, 16u, 1024u), xdesc = umma_smem_desc(at + S::W, 16u, 1024u);
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_fp8(tmem_base + buf * TOK, wdesc + k * 2, xdesc + k * 2, idesc, k != 0);
        umma_commit(tfull_bar(buf));
        umma_commit(empty_bar(stage));
        if (++stage == S::STAGES) { stage = 0; phase ^= 1u; }
        if (++buf == S::BUFS) { buf = 0; buf_phase ^= 1u; }
      }
    }
  } else {
    wait_for_previous();
    const int q = warp & 3, thread = threadIdx.x - 64, n = q * 32 + lane;
    float* scales = reinterpret_cast<float*>(smem_gen + S::SCALES);
    float* sums = reinterpret_cast<float*>(smem_gen);              // [TOK][128], once the stages have been read
    float acc[TOK];
#pragma unroll
    for (int t = 0; t < TOK; ++t) acc[t] = 0.f;
    int buf = 0; uint32_t buf_phase = 0;
    bool ok = true;
    for (int kb = kb0; kb < kb1; ++kb) {
      const int g = (kb - kb0) % S::GROUP;
      if (g == 0) {                                                // scales of the next k-blocks: of a token's values times the weights'
        if (kb > kb0) epilogue_barrier();
        const int count = min(S::GROUP, kb1 - kb);
        float x[S::GROUP * TOK / 128], w[S::GROUP * TOK / 128];
#pragma unroll
        for (int j = 0; j < S::GROUP * TOK / 128; ++j) {           // all on their way before the first is used
          const int i = thread + 128 * j, t = i % TOK, k = kb + i / TOK;
          const bool there = i < count * TOK && t < p.M;
          x[j] = there ? p.sx[t * p.sx_m + k * p.sx_k] : 0.f;
          w[j] = there ? p.sw[(n0 / BLOCK) * p.sw_n + k * p.sw_k] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < S::GROUP * TOK / 128; ++j) scales[thread + 128 * j] = x[j] * w[j];
        epilogue_barrier();
      }
      // every warp goes on to the barriers above and below, also when it has given up
      ok = ok && mbar_wait(tfull_bar(buf), buf_phase, abort_flag, p.status, ST_FP8_FEW + 4);
      ok = __all_sync(0xffffffffu, ok);
      if (ok) {
        tc_fence_after();
        uint32_t r[TOK];
        load_columns<TOK>(tmem_base + (uint32_t(q * 32) << 16) + buf * TOK, r);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(tempty_bar(buf));
        const float4* s = reinterpret_cast<const float4*>(scales + g * TOK);
#pragma unroll
        for (int t = 0; t < TOK; t += 4) {
          const float4 v = s[t >> 2];
          acc[t] = fmaf(__uint_as_float(r[t]), v.x, acc[t]);
          acc[t + 1] = fmaf(__uint_as_float(r[t + 1]), v.y, acc[t + 1]);
          acc[t + 2] = fmaf(__uint_as_float(r[t + 2]), v.z, acc[t + 2]);
          acc[t + 3] = fmaf(__uint_as_float(r[t + 3]), v.w, acc[t + 3]);
        }
        if (++buf == S::BUFS) { buf = 0; buf_phase ^= 1u; }
      }
    }
    // the last k-block's product is there, so all stages have been read by the tensor cores
    epilogue_barrier();
#pragma unroll
    for (int t = 0; t < TOK; ++t) sums[t * 128 + n] = acc[t];
  }
  let_next_start();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 256);
  }
  if (parts > 1) { cluster_arrive(); cluster_wait(); }             // every part's sums are there
  // this part's share of the tokens: a warp a token, four rows a lane
  if (!*abort_flag && n0 + 4 * lane < p.N) {
    for (int t = part + parts * warp; t < p.M; t += parts * 6) {
      float4 v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < parts) v[k] = peer_floats(map_to_cta(smem_base + (t * 128 + 4 * lane) * 4, k));
      float f[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < parts) { f[0] += v[k].x; f[1] += v[k].y; f[2] += v[k].z; f[3] += v[k].w; }
      if (p.type == 0) finish<bf16>(p, t, n0 + 4 * lane, f);
      else if (p.type == 1) finish<__half>(p, t, n0 + 4 * lane, f);
      else finish<float>(p, t, n0 + 4 * lane, f);
    }
  }
  if (parts > 1) { cluster_arrive(); cluster_wait(); }             // no part leaves while its sums are read
}

// As many parts of the contraction as give every SM a CTA, and two k-blocks each.
static int few_parts(int N, int K) {
  const int tiles = (N + 127) / 128, kbs = (K + 127) / 128;
  int parts = 1;
  while (parts < 8 && (long long)tiles * parts < num_sms() && 4 * parts <= kbs) parts *= 2;
  return parts;
}
template <int TOK>
static int launch_few(const CUtensorMap& tmW, const CUtensorMap& tmX, const FewArgs& p, bool chained, cudaStream_t stream) {
  auto kern = gemm_fp8_block_few_kernel<TOK>;
  static std::atomic<unsigned long long> allowed{0};       // devices that know the kernel's shared memory
  if (!allow_shared(allowed, kern, FewSpace<TOK>::BYTES)) return -5;
  const int tiles = (p.N + 127) / 128, parts = few_parts(p.N, p.K);
  if ((long long)tiles * parts > 0x7fffffffLL) return -3;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (chained) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (parts > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = parts; attr[n].val.clusterDim.y = 1; attr[n++].val.clusterDim.z = 1;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(tiles * parts));
  cfg.blockDim = dim3(192);
  cfg.dynamicSmemBytes = FewSpace<TOK>::BYTES;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = n;
  if (cudaLaunchKernelEx(&cfg, kern, tmW, tmX, p, parts) == cudaSuccess) return 0;
  (void)cudaGetLastError();
  return -6;
}

}  // namespace blk8
}  // namespace sb

// Whether a product of M tokens goes by this kernel.  With more tokens their tiles weigh as much as the weights', which the 128 x 128 tiles of the
// other kernel read once for 128 tokens; but those leave SMs idle where there are fewer tiles of weights than 7 for 16 SMs, and take a quarter longer for
// tokens that end inside of 32.  us, this kernel and the other, weights from memory:
//   K = 4096    N = 4096      8192        9472        12288       22528
//   T = 17       8.7, 12.6   11.0, 17.7  13.0, 18.2  15.2, 18.9  21.0, 29.6
//   T = 31                   11.4, 17.3  13.2, 17.1  15.6, 18.5  21.9, 29.9
//   T = 32       9.2, 12.7   11.5, 13.3  13.5, 13.4  15.7, 14.4  21.9, 25.9
//   T = 64      11.2, 12.8   12.9, 13.3  15.2, 13.7  18.2, 14.8  25.4, 26.1
// (K = 1024, N = 12288: T = 17 8.0, 7.8; T = 64 10.5, 7.5.  K = 11264: T = 17 28.7, 30.8; T = 64 32.0, 31.5.)
extern "C" int sb_gemm_fp8_block_takes_few(int M, int N) { return M < 32 || (M <= 64 && (N + 127) / 128 * 16 <= 7 * sb::num_sms()); }

// CTAs that share a tile's k-blocks.
extern "C" int sb_gemm_fp8_block_few_parts(int N, int K) { return sb::blk8::few_parts(N, K); }

// As sb_gemm_fp8_block with neither operand transposed and tiles of 128 x 128 in W; up to 64 rows of X.  chained: the launch before it on the
// stream was that of sb_fp8_block_quantize or sb_fp8_block_norm, which wrote X and sx and not W or sw.
extern "C" int sb_gemm_fp8_block_few(const void* X, const float* sx, long long sx_m, long long sx_k, const void* W, const float* sw, long long sw_n,
                                     long long sw_k, void* y, const void* bias, const void* residual, int M, int N, int K, long long ldx,
                                     long long ldw, long long ldc, long long ldr, int type, int chained, unsigned int* status, cudaStream_t stream) {
  using namespace sb;
  using namespace sb::blk8;
  if (M <= 0 || N <= 0) return 0;
  if (M > 64 || K <= 0) return -3;
  if (!bind_context()) return -5;                        // the tensor-map encoder needs a current context
  if ((ldx % 16) || (ldw % 16) || ((reinterpret_cast<uintptr_t>(X) | reinterpret_cast<uintptr_t>(W)) & 15)) return -4;
  const int tok = M <= 16 ? 16 : M <= 32 ? 32 : 64;
  CUtensorMap tmW, tmX;
  int rc;
  if ((rc = make_tmap_2d_u8(&tmW, W, K, N, ldw, 128, 128))) return rc;
  if ((rc = make_tmap_2d_u8(&tmX, X, K, M, ldx, 128, tok))) return rc;
  FewArgs p{sx, sw, sx_m, sx_k, sw_n, sw_k, ldc, ldr, y, bias, residual, M, N, K, type, status};
  return tok == 16 ? launch_few<16>(tmW, tmX, p, chained, stream) : tok == 32 ? launch_few<32>(tmW, tmX, p, chained, stream)
                                                                              : launch_few<64>(tmW, tmX, p, chained, stream);
}
