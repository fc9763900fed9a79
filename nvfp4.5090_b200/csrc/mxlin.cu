// MXFP4 linear layer for few tokens (B200, sm_100a): y = Q(x) . W^T + bias
// with W held in MXFP4.
//
// With few tokens the product is a stream of the weights (17/32 byte per
// element, each read once); the 256 x 256 pair tiles of the general GEMM spread
// an n of 4096 over 32 of the 148 SMs and fill 255 of 256 rows with zeros for
// one token.  Here the roles are swapped: 128 weight rows are the MMA's M, the
// tokens (16, 32, 64 or 128 columns) its N, and K is cut over the CTAs of a
// cluster, so that 128-row tiles x K parts fill the SMs.  The parts' fp32 sums
// meet through distributed shared memory in one fixed order.
//
//   grid (tiles * parts, token blocks), cluster (parts, 1): CTA rank r of a
//     cluster takes every stage (256 k) of its share of K for 128 weight rows;
//   warp 0      producer: weights (one 128-byte-swizzled TMA box of 128 rows x
//               128 bytes, and their 2 scale atoms) and tokens (N x 128 bytes,
//               2 atoms) per stage, into a ring of up to 8 stages;
//   warp 1      MMA issuer: 4 tcgen05.mma.cta_group::1 kind::mxf4 128 x N x 64
//               per stage and the copies of the scale atoms to TMEM;
//   all 4 warps epilogue: TMEM -> shared memory as [token][row]; after a
//               cluster barrier the CTA of rank r adds up the parts of tokens
//               r, r + parts, .. and writes them with the bias.
// The tokens are quantized by the row quantizer just before; this kernel is
// its programmatic dependent, so the weights' first stages are under way (they
// need nothing of it) while the tokens are being quantized.
//
// Every wait is bounded; a timeout sets the library's device error word.
#include "bulk.cuh"

#include <cuda.h>

#include <algorithm>
#include <mutex>

namespace nvfp4b200 {

int mx_quant_rows_async(const void* x, void* q, void* s, int64_t rows, int64_t cols, int64_t ldx, cudaStream_t st);

namespace mxlin {

__device__ int g_error = 0;

constexpr int TILE_ROWS = 128;
constexpr int BK = 256, BK_BYTES = BK / 2;
constexpr int A_BYTES = TILE_ROWS * BK_BYTES;     // 16 KB
constexpr int SF_BYTES = 1024;                    // two atoms: 128 rows x 8 scales
constexpr int THREADS = 128;
constexpr int MAX_STAGES = 8;
constexpr int MAX_PARTS = 8;
constexpr int SMEM_SM = 227 * 1024;

struct Args {
  const uint8_t *sfw, *sfx;     // scale atoms of the weights and of the tokens
  const uint16_t* bias;         // bf16 [n] or null
  uint16_t* y;                  // bf16 [m, n]
  int64_t m, n, k;
  int atoms;                    // scale atoms per 128 rows: ceil(k / 128)
  int k_stages;                 // ceil(k / 256)
  int stages;                   // ring depth
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_cluster(uint32_t local_addr, uint32_t rank) {
  float v;
  asm volatile(
      "{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.f32 %0, [a];\n\t}"
      : "=f"(v)
      : "r"(local_addr), "r"(rank)
      : "memory");
  return v;
}
__device__ __forceinline__ void tma_2d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          bulk::addr(dst)),
      "l"(map), "r"(x), "r"(y), "r"(bulk::addr(bar))
      : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bulk::addr(bar))
               : "memory");
}
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// K-major operand with 128-byte swizzle: 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t operand_desc(uint32_t saddr) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// One 512-byte scale atom: 32 rows of 16 bytes, 8-row groups 128 bytes apart.
__device__ __forceinline__ uint64_t atom_desc(uint32_t saddr) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (8ull << 32) | (1ull << 46);
}
// kind::mxf4, E2M1 operands, UE8M0 scales, M = 128.  `byte` (0 or 2): where the
// MMA's two scales per row start in a 4-byte scale cell.
__device__ __forceinline__ void mma(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t n, uint32_t sfa, uint32_t sfb,
                                    uint32_t byte, bool accumulate) {
  const uint32_t idesc =
      (1u << 7) | (1u << 10) | ((n >> 3) << 17) | (1u << 23) | (1u << 27) | (byte << 29) | (byte << 4);
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}\n" ::"r"(d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"((uint32_t)accumulate), "r"(sfa | (byte << 30)), "r"(sfb | (byte << 30))
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

template <int N>
constexpr int stage_bytes() { return A_BYTES + N * BK_BYTES + 2 * SF_BYTES; }
template <int N>
constexpr int tmem_cols() { return 2 * N; }   // N accumulator columns, 8 + 8 of scales; a power of two, at least 32

template <int N>
__global__ void __launch_bounds__(THREADS) mx_linear_kernel(const __grid_constant__ CUtensorMap wmap,
                                                            const __grid_constant__ CUtensorMap xmap, const Args a) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  // ring: operands of every stage (1024-byte aligned), then the scales
  uint8_t* s_a = smem;
  uint8_t* s_b = s_a + a.stages * A_BYTES;
  uint8_t* s_sfa = s_b + a.stages * N * BK_BYTES;
  uint8_t* s_sfb = s_sfa + a.stages * SF_BYTES;
  __shared__ __align__(8) uint64_t full[MAX_STAGES], empty[MAX_STAGES], done;
  __shared__ uint32_t tmem_slot;
  __shared__ int gave_up;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_rank(), parts = (int)cluster_size();
  const int tile = blockIdx.x / parts;
  const int tok0 = blockIdx.y * N;
  const int k_lo = (int)((int64_t)a.k_stages * rank / parts), k_hi = (int)((int64_t)a.k_stages * (rank + 1) / parts);
  const int steps = k_hi - k_lo;

  if (threadIdx.x == 0) {
    gave_up = 0;
    bulk::init(full, MAX_STAGES);
    bulk::init(empty, MAX_STAGES);
    bulk::init(&done, 1);
    asm volatile("prefetch.tensormap [%0];" ::"l"(&wmap) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&xmap) : "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(bulk::addr(&tmem_slot)),
                 "r"(tmem_cols<N>())
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_slot;

  int issued = 0;   // thread 0: stages whose copies it issued
  if (warp == 0 && lane == 0) {
    // ---- producer ----
    auto sf_bytes = [&](int i) { return (uint32_t)min(2, a.atoms - 2 * (k_lo + i)) * 512u; };
    auto weights = [&](int i, int st) {
      const uint32_t sf = sf_bytes(i);
      bulk::expect(&full[st], (uint32_t)(A_BYTES + N * BK_BYTES) + 2 * sf);
      tma_2d(s_a + st * A_BYTES, &wmap, &full[st], (k_lo + i) * BK_BYTES, tile * TILE_ROWS);
      bulk::copy(s_sfa + st * SF_BYTES, a.sfw + ((int64_t)tile * a.atoms + 2 * (k_lo + i)) * 512, sf, &full[st]);
    };
    auto tokens = [&](int i, int st) {
      tma_2d(s_b + st * N * BK_BYTES, &xmap, &full[st], (k_lo + i) * BK_BYTES, tok0);
      bulk::copy(s_sfb + st * SF_BYTES, a.sfx + ((int64_t)(tok0 / 128) * a.atoms + 2 * (k_lo + i)) * 512, sf_bytes(i),
                 &full[st]);
    };
    const int first = min(steps, a.stages);
    for (int i = 0; i < first; ++i) weights(i, i);
    asm volatile("griddepcontrol.wait;" ::: "memory");   // the tokens are quantized from here on
    for (int i = 0; i < first; ++i) tokens(i, i);
    issued = first;
    int st = 0;
    uint32_t phase = 0;
    for (int i = first; i < steps; ++i) {
      if (!bulk::wait(&empty[st], phase)) {
        gave_up = 1;
        break;
      }
      weights(i, st);
      tokens(i, st);
      ++issued;
      if (++st == a.stages) {
        st = 0;
        phase ^= 1u;
      }
    }
  } else if (warp == 1 && lane == 0) {
    // ---- MMA issuer ----
    int st = 0;
    uint32_t phase = 0;
    bool ok = true;
    const uint32_t sfa = tmem + N, sfb = sfa + 8;
    for (int i = 0; i < steps; ++i) {
      if (!bulk::wait(&full[st], phase)) {
        ok = false;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const int64_t rem = a.k - (int64_t)(k_lo + i) * BK;
      const int kb = (int)imin64(4, (rem + 63) / 64);
      const uint64_t ad = operand_desc(bulk::addr(s_a + st * A_BYTES)), bd = operand_desc(bulk::addr(s_b + st * N * BK_BYTES));
      const uint64_t sad = atom_desc(bulk::addr(s_sfa + st * SF_BYTES)), sbd = atom_desc(bulk::addr(s_sfb + st * SF_BYTES));
      // the scale cells are reused by every stage: one thread's tcgen05
      // operations execute in the order it issues them
      for (int j = 0; j < kb; ++j) {
        const int c = j >> 1;
        if ((j & 1) == 0) {
          copy_scales(sfa + 4 * c, sad + 32 * c);
          copy_scales(sfb + 4 * c, sbd + 32 * c);
        }
        mma(tmem, ad + 2 * j, bd + 2 * j, N, sfa + 4 * c, sfb + 4 * c, 2u * (j & 1), (i | j) != 0);
      }
      commit(&empty[st]);
      if (++st == a.stages) {
        st = 0;
        phase ^= 1u;
      }
    }
    commit(&done);
    if (!bulk::wait(&done, 0)) ok = false;
    if (!ok) gave_up = 1;
  }
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (gave_up && threadIdx.x == 0) {
    atomicExch(&g_error, NVFP4B200_ERR_TIMEOUT);
    // let the copies that were issued land: the last fill of every stage
    for (int st = 0; st < a.stages; ++st) {
      const int fills = issued > st ? (issued - 1 - st) / a.stages + 1 : 0;
      if (fills) bulk::wait(&full[st], (uint32_t)(fills - 1) & 1u);
    }
  }
  // ---- epilogue: this part's sums as [token][row], over the ring (every MMA has read it) ----
  float* part = reinterpret_cast<float*>(smem);
  const int tokens_here = (int)imin64(N, a.m - tok0);
  for (int t = 0; t < tokens_here; t += 16) {
    uint32_t v[16];
    tmem_ld16(tmem + ((uint32_t)(warp * 32) << 16) + t, v);
#pragma unroll
    for (int j = 0; j < 16; ++j) part[(t + j) * TILE_ROWS + threadIdx.x] = __uint_as_float(v[j]);
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(tmem_cols<N>()) : "memory");
  __syncwarp();
  if (parts > 1) cluster_sync();
  const int64_t row = (int64_t)tile * TILE_ROWS + threadIdx.x;
  if (row < a.n && !gave_up) {
    const float bias = a.bias ? __uint_as_float((uint32_t)__ldg(a.bias + row) << 16) : 0.0f;
    for (int t = rank; t < tokens_here; t += parts) {
      const uint32_t at = bulk::addr(part + t * TILE_ROWS + threadIdx.x);
      float s = 0.0f;
      for (int r = 0; r < parts; ++r) s += parts > 1 ? ld_cluster(at, (uint32_t)r) : part[t * TILE_ROWS + threadIdx.x];
      a.y[(int64_t)(tok0 + t) * a.n + row] = __bfloat16_as_ushort(__float2bfloat16_rn(s + bias));
    }
  }
  if (parts > 1) cluster_sync();   // no CTA leaves while another reads its sums
}

// ---- host ----------------------------------------------------------------

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                             const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                             CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Packed operand [rows, row_bytes], boxes of 128 bytes x box_rows, 128-byte swizzle; past the end reads zeros.
static bool operand_map(CUtensorMap* map, const void* base, int64_t rows, int64_t row_bytes, int box_rows) {
  static EncodeFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeFn>(ptr);
  });
  if (!fn) return false;
  cuuint64_t dims[2] = {(cuuint64_t)row_bytes, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)row_bytes};
  cuuint32_t box[2] = {(cuuint32_t)BK_BYTES, (cuuint32_t)box_rows}, one[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, one,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int N>
static int launch(const void* qw, const void* qx, Args a, int sms, cudaStream_t st) {
  CUtensorMap wm, xm;
  if (!operand_map(&wm, qw, a.n, a.k / 2, TILE_ROWS) || !operand_map(&xm, qx, a.m, a.k / 2, N)) return NVFP4B200_ERR_CUDA;
  const int64_t tiles = ceil_div(a.n, TILE_ROWS), blocks = ceil_div(a.m, N);
  // K parts: double them while that leaves every CTA at least 2 stages and
  // the grid under two CTAs per SM
  int parts = 1;
  while (parts < MAX_PARTS && a.k_stages >= 4 * parts && tiles * blocks * parts * 2 <= 2 * sms) parts *= 2;
  const int most = (int)ceil_div(a.k_stages, parts);
  // two CTAs per SM share its memory; the [N][128] sums reuse the ring
  const int fit = (SMEM_SM / 2 - 2048) / stage_bytes<N>();
  a.stages = std::max(1, std::min({most, fit, MAX_STAGES}));
  const int smem = std::max(a.stages * stage_bytes<N>(), N * TILE_ROWS * 4) + 1024;
  auto* fn = mx_linear_kernel<N>;
  if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return NVFP4B200_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * parts), (unsigned)blocks, 1);
  cfg.blockDim = dim3(THREADS, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, fn, wm, xm, a) != cudaSuccess) {
    cudaGetLastError();
    return NVFP4B200_ERR_LAUNCH;
  }
  return launch_status();
}

}  // namespace mxlin

int take_mxlin_device_error() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, mxlin::g_error, sizeof(int)) != cudaSuccess) return NVFP4B200_ERR_CUDA;
  if (v && cudaMemcpyToSymbol(mxlin::g_error, &zero, sizeof(int)) != cudaSuccess) return NVFP4B200_ERR_CUDA;
  return v;
}

}  // namespace nvfp4b200

using namespace nvfp4b200;

extern "C" int nvfp4b200_mx_linear(const void* x, const void* qw, const void* sfw, const void* bias, void* qx, void* sfx,
                                   void* y, int64_t m, int64_t n, int64_t k, int64_t ldx, void* stream) {
  if (!x || !qw || !sfw || !qx || !sfx || !y) return NVFP4B200_ERR_INVALID_ARG;
  if (m < 0 || n < 0 || n % 8 || k <= 0 || k % 32 || ldx < k || ldx % 8 || m > (1ll << 30) || n > (1ll << 30) ||
      k > (1ll << 30))
    return NVFP4B200_ERR_BAD_SHAPE;
  for (const void* p : {x, qw, sfw, bias, (const void*)qx, (const void*)sfx, (const void*)y})
    if (p && !aligned(p, 16)) return NVFP4B200_ERR_MISALIGNED;
  int rc = check_device();
  if (rc) return rc;
  if (m == 0 || n == 0) return NVFP4B200_OK;
  cudaStream_t st = (cudaStream_t)stream;
  rc = mx_quant_rows_async(x, qx, sfx, m, k, ldx, st);
  if (rc) return rc;
  if (m > 128) return nvfp4b200_mx_gemm(qx, qw, sfx, sfw, bias, nullptr, y, NVFP4B200_BF16, 0, NVFP4B200_EPI_NONE, m, n, k, n, stream);
  mxlin::Args a;
  a.sfw = static_cast<const uint8_t*>(sfw);
  a.sfx = static_cast<const uint8_t*>(sfx);
  a.bias = static_cast<const uint16_t*>(bias);
  a.y = static_cast<uint16_t*>(y);
  a.m = m;
  a.n = n;
  a.k = k;
  a.atoms = (int)ceil_div(k, 128);
  a.k_stages = (int)ceil_div(k, mxlin::BK);
  a.stages = 0;
  const int sms = sm_count_current();
  if (m <= 16) return mxlin::launch<16>(qw, qx, a, sms, st);
  if (m <= 32) return mxlin::launch<32>(qw, qx, a, sms, st);
  if (m <= 64) return mxlin::launch<64>(qw, qx, a, sms, st);
  return mxlin::launch<128>(qw, qx, a, sms, st);
}
