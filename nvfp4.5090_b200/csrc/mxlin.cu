// MXFP4 linear layer for few tokens, or few outputs (B200, sm_100a): y = Q(x) . W^T + bias
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
//   grid (tiles * parts, blocks of N tokens), cluster (parts): CTA rank r of a cluster takes every
//     stage (256 k) of its share of K for 128 weight rows;
//   warp 0      producer: weights (one 128-byte-swizzled TMA box of 128 rows x
//               128 bytes, and their 2 scale atoms) per stage into a ring of up
//               to 8 stages, and the quantized tokens (N x 128 bytes, 2 atoms);
//   warp 1      MMA issuer: 4 tcgen05.mma.cta_group::1 kind::mxf4 128 x N x 64
//               per stage and the copies of the scale atoms to TMEM;
//   all 8 warps epilogue: TMEM -> shared memory as [token][row]; after a
//               cluster barrier the CTA of rank r adds up the parts of tokens
//               r, r + parts, .. and writes them with the bias.
// Up to 12 tokens are quantized here (FUSED): warps 2-7 read a token's 256 k
// of a stage, a warp each, and write nibbles and scale codes where the MMA
// reads them, while the weights are still under way; one launch, no
// workspace.  More tokens would make every 128-row tile's CTA spend longer on
// them than on its weights: they are quantized once by the row quantizer just
// before, and this kernel is its programmatic dependent, so its first weights
// load meanwhile (they were complete before the quantizer, an ordinary launch,
// began).  At 12 tokens the two forms are level: 17.5 against 17.7 us through
// 28672 x 4096; at 16 it is 21.5 against 17.7, at 1 it is 14.7 against 16.5.
// FUSED is launched as a dependent too, of whatever comes before it:
// only its set-up runs early, it reads nothing before that is complete.
//
// Every wait is bounded; a timeout sets the library's device error word.
#include "bulk.cuh"
#include "mx.cuh"

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
constexpr int THREADS = 256;
constexpr int FUSED_TOKENS = 12;
constexpr int FUSED_STEPS = 16;                   // stages of tokens that stay in shared memory (48 KB)
constexpr int MAX_STAGES = 8;
constexpr int MAX_PARTS = 8;
constexpr int SMEM_SM = 227 * 1024;

struct Args {
  const uint8_t *sfw, *sfx;     // scale atoms of the weights and (not FUSED) of the tokens
  const uint16_t* x;            // FUSED: bf16 [m, k], row stride ldx
  int64_t ldx;
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
// The barrier's aligned form takes whole warps: lanes that parted before it meet first.
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 ld_cluster(uint32_t local_addr, uint32_t rank) {
  float4 v;
  asm volatile(
      "{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %4, %5;\n\tld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n\t}"
      : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
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

// Ring stage: weights, and unless they are quantized here the tokens, each with scale atoms.
template <int N, bool FUSED>
constexpr int stage_bytes() { return A_BYTES + SF_BYTES + (FUSED ? 0 : N * BK_BYTES + SF_BYTES); }
template <int N>
constexpr int tmem_cols() { return 2 * N; }   // N accumulator columns, 8 + 8 of scales; a power of two, at least 32

template <int N, bool FUSED>
__global__ void __launch_bounds__(THREADS) mx_linear_kernel(const __grid_constant__ CUtensorMap wmap,
                                                            const __grid_constant__ CUtensorMap xmap, const Args a) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t full[MAX_STAGES], empty[MAX_STAGES], tok[FUSED_STEPS], done;
  __shared__ uint32_t tmem_slot;
  __shared__ int gave_up;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_rank(), parts = (int)cluster_size();
  const int tile = blockIdx.x / parts;
  const int tok0 = blockIdx.y * N;   // N = 128 where there is more than one block of tokens
  const int k_lo = (int)((int64_t)a.k_stages * rank / parts), k_hi = (int)((int64_t)a.k_stages * (rank + 1) / parts);
  const int steps = k_hi - k_lo;
  // weights of every stage and tokens (1024-byte aligned), then the scales; the
  // tokens sit in the ring, or (FUSED) all steps of them stay
  const int tok_slots = FUSED ? steps : a.stages;
  uint8_t* s_a = smem;
  uint8_t* s_b = s_a + a.stages * A_BYTES;
  uint8_t* s_sfa = s_b + tok_slots * N * BK_BYTES;
  uint8_t* s_sfb = s_sfa + a.stages * SF_BYTES;

  if (threadIdx.x == 0) {
    gave_up = 0;
    bulk::init(full, MAX_STAGES);
    bulk::init(empty, MAX_STAGES);
    bulk::init(&done, 1);
    if (FUSED)
      for (int i = 0; i < FUSED_STEPS; ++i) bulk::init(tok + i, 1, (uint32_t)a.m);
    asm volatile("prefetch.tensormap [%0];" ::"l"(&wmap) : "memory");
    if (!FUSED) asm volatile("prefetch.tensormap [%0];" ::"l"(&xmap) : "memory");
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
      bulk::expect(&full[st], (uint32_t)A_BYTES + sf + (FUSED ? 0u : N * BK_BYTES + sf));
      tma_2d(s_a + st * A_BYTES, &wmap, &full[st], (k_lo + i) * BK_BYTES, tile * TILE_ROWS);
      bulk::copy(s_sfa + st * SF_BYTES, a.sfw + ((int64_t)tile * a.atoms + 2 * (k_lo + i)) * 512, sf, &full[st]);
    };
    auto tokens = [&](int i, int st) {
      if (FUSED) return;
      tma_2d(s_b + st * N * BK_BYTES, &xmap, &full[st], (k_lo + i) * BK_BYTES, tok0);
      bulk::copy(s_sfb + st * SF_BYTES, a.sfx + ((int64_t)blockIdx.y * a.atoms + 2 * (k_lo + i)) * 512, sf_bytes(i), &full[st]);
    };
    const int first = min(steps, a.stages);
    // FUSED: whatever ran before may have written the weights themselves
    if (FUSED) asm volatile("griddepcontrol.wait;" ::: "memory");
    for (int i = 0; i < first; ++i) weights(i, i);
    if (!FUSED) {
      asm volatile("griddepcontrol.wait;" ::: "memory");   // the tokens are quantized from here on
      for (int i = 0; i < first; ++i) tokens(i, i);
    }
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
    // every load is under way: a next call's CTAs may set themselves up
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  } else if (warp == 1 && lane == 0) {
    // ---- MMA issuer ----
    int st = 0;
    uint32_t phase = 0;
    bool ok = true;
    const uint32_t sfa = tmem + N, sfb = sfa + 8;
    for (int i = 0; i < steps; ++i) {
      if ((FUSED && !bulk::wait(&tok[i], 0)) || !bulk::wait(&full[st], phase)) {
        ok = false;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const int64_t rem = a.k - (int64_t)(k_lo + i) * BK;
      const int kb = (int)imin64(4, (rem + 63) / 64);
      const int bs = FUSED ? i : st;
      const uint64_t ad = operand_desc(bulk::addr(s_a + st * A_BYTES)), bd = operand_desc(bulk::addr(s_b + bs * N * BK_BYTES));
      const uint64_t sad = atom_desc(bulk::addr(s_sfa + st * SF_BYTES)), sbd = atom_desc(bulk::addr(s_sfb + bs * SF_BYTES));
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
  } else if (FUSED && warp >= 2) {
    // ---- tokens: a warp quantizes 256 k of one token, 8 values a lane, 4 lanes a block ----
    // Rows past m are left as they are: they are columns of the product that nobody reads.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    constexpr int WARPS = THREADS / 32 - 2, AHEAD = 4;   // reads in flight per warp
    const int m = (int)a.m, tasks = steps * m;
    for (int t0 = warp - 2; t0 < tasks; t0 += WARPS * AHEAD) {
      uint4 raw[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int task = t0 + u * WARPS, i = task / m, t = task - i * m;
        const int64_t c = (int64_t)(k_lo + i) * BK + 8 * lane;
        raw[u] = make_uint4(0, 0, 0, 0);
        if (task < tasks && c < a.k) raw[u] = __ldg(reinterpret_cast<const uint4*>(a.x + t * a.ldx + c));
      }
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int task = t0 + u * WARPS, i = task / m, t = task - i * m;
        if (task >= tasks) break;
        const uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
        uint32_t top = 0;
        float f[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          top = __vmaxu2(top, w[j] & 0x7FFF7FFFu);
          f[2 * j] = bf16lo(w[j]);
          f[2 * j + 1] = bf16hi(w[j]);
        }
        top = max(top & 0xFFFFu, top >> 16);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        uint32_t code;
        float inv;
        mx::block_scale(__uint_as_float(top << 16), code, inv);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] *= inv;
        const uint32_t nib = mx::encode8(f);
        const int j = lane >> 2;   // the stage's block, a 16-byte piece of the swizzled row
        *reinterpret_cast<uint32_t*>(s_b + i * N * BK_BYTES + t * BK_BYTES + ((j ^ (t & 7)) << 4) + 4 * (lane & 3)) = nib;
        if ((lane & 3) == 0) s_sfb[i * SF_BYTES + (j >> 2) * 512 + atom_offset(t, j & 3)] = (uint8_t)code;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the MMA reads through the async proxy
        __syncwarp();
        if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bulk::addr(&tok[i])) : "memory");
      }
    }
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
  __syncthreads();
  float* part = reinterpret_cast<float*>(smem);
  const int m = (int)imin64(N, a.m - tok0);   // tokens of this block
  __syncwarp();
  {
    const int row = 32 * (warp & 3) + lane;   // a warp reads the TMEM lanes of its quarter
    for (int t = 16 * (warp >> 2); t < m; t += 32) {
      uint32_t v[16];
      tmem_ld16(tmem + ((uint32_t)(32 * (warp & 3)) << 16) + t, v);
#pragma unroll
      for (int j = 0; j < 16; ++j) part[(t + j) * TILE_ROWS + row] = __uint_as_float(v[j]);
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  __syncwarp();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(tmem_cols<N>()) : "memory");
  if (parts > 1) cluster_sync();
  const int64_t row = (int64_t)tile * TILE_ROWS + 4 * lane;   // n % 8 == 0: all four rows or none
  if (row < a.n && !gave_up) {
    float bias[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (a.bias) {
      const uint2 w = __ldg(reinterpret_cast<const uint2*>(a.bias + row));
      bias[0] = bf16lo(w.x); bias[1] = bf16hi(w.x); bias[2] = bf16lo(w.y); bias[3] = bf16hi(w.y);
    }
#pragma unroll 2
    for (int t = rank + parts * warp; t < m; t += parts * (THREADS / 32)) {
      const float* at = part + t * TILE_ROWS + 4 * lane;
      float4 v[MAX_PARTS];
      if (parts == 1) {
        v[0] = *reinterpret_cast<const float4*>(at);
      } else {
#pragma unroll
        for (int r = 0; r < MAX_PARTS; ++r)
          if (r < parts) v[r] = ld_cluster(bulk::addr(at), (uint32_t)r);
      }
      float4 s = v[0];   // the parts in order
#pragma unroll
      for (int r = 1; r < MAX_PARTS; ++r)
        if (r < parts) {
          s.x += v[r].x;
          s.y += v[r].y;
          s.z += v[r].z;
          s.w += v[r].w;
        }
      const __nv_bfloat162 lo = __floats2bfloat162_rn(s.x + bias[0], s.y + bias[1]);
      const __nv_bfloat162 hi = __floats2bfloat162_rn(s.z + bias[2], s.w + bias[3]);
      *reinterpret_cast<uint2*>(a.y + (int64_t)(tok0 + t) * a.n + row) =
          make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
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

// K parts: doubled while that leaves every CTA at least 2 stages and the grid
// at most two CTAs per SM (what its memory holds).  One token: 11.0 us so at
// 4096 x 14336, 12.5 with half the CTAs; 11.2 at 8192 x 8192, 13.6 with half and
// 15.0 with twice as many.
static int parts_for(int64_t tiles, int k_stages, int sms) {
  int parts = 1;
  while (parts < MAX_PARTS && k_stages >= 4 * parts && tiles * parts * 2 <= 2 * sms) parts *= 2;
  return parts;
}

template <int N, bool FUSED>
static int launch(const void* qw, const void* qx, Args a, int parts, cudaStream_t st) {
  CUtensorMap wm, xm;
  if (!operand_map(&wm, qw, a.n, a.k / 2, TILE_ROWS)) return NVFP4B200_ERR_CUDA;
  if (FUSED) xm = wm;   // not used
  else if (!operand_map(&xm, qx, a.m, a.k / 2, N)) return NVFP4B200_ERR_CUDA;
  const int64_t tiles = ceil_div(a.n, TILE_ROWS);
  const int most = (int)ceil_div(a.k_stages, parts);
  const int held = FUSED ? most * (N * BK_BYTES + SF_BYTES) : 0;
  // two CTAs per SM share its memory; the [N][128] sums reuse the ring
  const int fit = (SMEM_SM / 2 - 2048 - held) / stage_bytes<N, FUSED>();
  a.stages = std::max(1, std::min({most, fit, MAX_STAGES}));
  const int smem = std::max(a.stages * stage_bytes<N, FUSED>() + held, N * TILE_ROWS * 4) + 1024;
  constexpr int MOST = SMEM_SM / 2;   // of the ring (above) and of the sums
  static_assert(N * TILE_ROWS * 4 + 1024 <= MOST && stage_bytes<N, FUSED>() + (FUSED ? FUSED_STEPS * (N * BK_BYTES + SF_BYTES) : 0) + 1024 <= MOST,
                "shared memory of one CTA of two");
  auto* fn = mx_linear_kernel<N, FUSED>;
  if (!allow_smem(fn, MOST)) return NVFP4B200_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * parts), (unsigned)ceil_div(a.m, N), 1);
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

// Whether to take the 128-row tiles, times blocks of 128 tokens, and not the 256 x
// 256 pair tiles of the general GEMM: for one block of tokens, and while there is
// an SM for each tile.  Both ways in us (quantizer included, replayed from a graph
// over weights that come from HBM), weights as n x k:
//   tokens            16          64          96         128         256
//   28672 x 4096   16.8/23.8   17.7/23.6   19.4/23.9   19.8/24.6   26.3/26.0 *
//   14336 x 4096   12.5/14.7   13.7/14.9   14.9/15.2   15.9/15.6   16.4/16.5 *
//   4096 x 14336   12.6/25.6   14.3/25.9   15.6/26.3   17.7/26.7   18.8/27.3
//   4096 x 4096     8.3/12.9   10.9/13.3   13.0/13.6   15.1/14.1   12.9/14.1
//   57344 x 8192   51.0/66.0   51.5/62.5   55.6/64.0   58.0/65.2   68.6/68.6 *
// (*: the rule takes the general GEMM.)  So the rule costs up to 7% at 97 to 128
// tokens of a small weight, where K is in four parts.  512 tokens 14.2/15.1 at
// 4096 x 4096 (128 tiles), 768 tokens 17.5/15.7 there (192 tiles).
static bool few_tokens(int64_t m, int64_t tiles, int sms) { return m <= 128 || tiles * ceil_div(m, 128) <= sms; }

extern "C" {

int nvfp4b200_mx_linear_fused(int64_t m, int64_t n, int64_t k) {
  if (m < 1 || m > mxlin::FUSED_TOKENS || n < 1 || k < 1) return 0;
  // K parts that hold their tokens in shared memory: 8 parts of 16 stages at most
  return ceil_div(k, mxlin::BK) <= mxlin::MAX_PARTS * mxlin::FUSED_STEPS;
}

int nvfp4b200_mx_linear(const void* x, const void* qw, const void* sfw, const void* bias, void* qx, void* sfx, void* y,
                        int64_t m, int64_t n, int64_t k, int64_t ldx, void* stream) {
  const bool fused = nvfp4b200_mx_linear_fused(m, n, k);
  if (!x || !qw || !sfw || (!fused && (!qx || !sfx)) || !y) return NVFP4B200_ERR_INVALID_ARG;
  if (m < 0 || n < 0 || n % 8 || k <= 0 || k % 32 || ldx < k || ldx % 8 || m > (1ll << 30) || n > (1ll << 30) ||
      k > (1ll << 30))
    return NVFP4B200_ERR_BAD_SHAPE;
  for (const void* p : {x, qw, sfw, bias, (const void*)qx, (const void*)sfx, (const void*)y})
    if (p && !aligned(p, 16)) return NVFP4B200_ERR_MISALIGNED;
  int rc = check_device();
  if (rc) return rc;
  if (m == 0 || n == 0) return NVFP4B200_OK;
  cudaStream_t st = (cudaStream_t)stream;
  const int sms = sm_count_current();
  const int64_t tiles = ceil_div(n, mxlin::TILE_ROWS);
  mxlin::Args a;
  a.sfw = static_cast<const uint8_t*>(sfw);
  a.sfx = static_cast<const uint8_t*>(sfx);
  a.x = static_cast<const uint16_t*>(x);
  a.ldx = ldx;
  a.bias = static_cast<const uint16_t*>(bias);
  a.y = static_cast<uint16_t*>(y);
  a.m = m;
  a.n = n;
  a.k = k;
  a.atoms = (int)ceil_div(k, 128);
  a.k_stages = (int)ceil_div(k, mxlin::BK);
  a.stages = 0;
  int parts = mxlin::parts_for(tiles * ceil_div(m, 128), a.k_stages, sms);
  if (fused) {
    while (ceil_div(a.k_stages, parts) > mxlin::FUSED_STEPS) parts *= 2;
    return mxlin::launch<16, true>(qw, nullptr, a, parts, st);
  }
  rc = mx_quant_rows_async(x, qx, sfx, m, k, ldx, st);
  if (rc) return rc;
  if (!few_tokens(m, tiles, sms))
    return nvfp4b200_mx_gemm(qx, qw, sfx, sfw, bias, nullptr, y, NVFP4B200_BF16, 0, NVFP4B200_EPI_NONE, m, n, k, n,
                             stream);
  if (m <= 16) return mxlin::launch<16, false>(qw, qx, a, parts, st);
  if (m <= 32) return mxlin::launch<32, false>(qw, qx, a, parts, st);
  if (m <= 64) return mxlin::launch<64, false>(qw, qx, a, parts, st);
  return mxlin::launch<128, false>(qw, qx, a, parts, st);
}

}  // extern "C"
