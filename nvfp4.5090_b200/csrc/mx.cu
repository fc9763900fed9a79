// MXFP4 operands for B200 (sm_100a): quantizers along rows, along columns and
// in both orientations from one read, and the way back.
//
// A block of 32 values v shares one power of two.  With amax the largest |v|
// and E2M1's largest exponent 2 (6 = 1.5 * 2^2),
//     code = clamp(floor(log2 amax) - 2, -127, ..) + 127        (UE8M0 byte)
//     q    = e2m1_rn(v * 2^(127 - code))                        (4 bits)
// where e2m1_rn rounds to the nearest of {0, .5, 1, 1.5, 2, 3, 4, 6}, ties to
// the even code, and saturates (v * 2^-e < 8).  floor(log2 amax) is the
// exponent field of amax as fp32, so code = max(field - 2, 0); a field of 0
// (zero or fp32-subnormal amax) gives 0.  The multiply is exact: a power of
// two, and a product that underflows is far below half the first grid step.
// A block that holds an infinity or a NaN gets code 0xFF, UE8M0's NaN, so it
// shows in every product that meets it; its nibbles mean nothing then.
//
// Every kernel is bound by HBM: 2 bytes read and 17/32 written per bf16
// element and orientation.
#include "mx.cuh"
#include "vec.cuh"

#include <algorithm>

namespace nvfp4b200 {

int sm_count_current() {
  static int cache[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return 148;
  if (cache[dev] == 0) cudaDeviceGetAttribute(&cache[dev], cudaDevAttrMultiProcessorCount, dev);
  return cache[dev] > 0 ? cache[dev] : 148;
}

namespace mx {

__device__ __forceinline__ uint32_t absbits(float f) { return __float_as_uint(f) & 0x7FFFFFFFu; }

// ---------------------------------------------------------------------------
// quantizer: one CTA per 128 x 128 tile, which is one 512-byte scale atom of
// either orientation (128 rows x 4 blocks of 32 columns, 128 columns x 4
// blocks of 32 rows)
// ---------------------------------------------------------------------------
// Rows: 16 lanes read a row of the tile (8 elements each), a block is 4 lanes.
// Columns: the tile is kept in shared memory; a thread owns two neighbouring
// columns of one 32-row block and reads them down, conflict-free because
// lanes own neighbouring words.  The columns' nibbles are staged in shared
// memory and written as 64-byte segments.
constexpr int TILE = 128;
constexpr int QTHREADS = 256;

struct QuantArgs {
  const void* x;
  const float* row_scale;     // [rows] or null
  const uint16_t* gamma;      // bf16 [cols] or null
  uint8_t* q;                 // [rows, cols/2]
  uint8_t* s;                 // atoms of (rows, cols)
  uint8_t* qt;                // [cols, prows/2], prows = rows rounded up to 32
  uint8_t* st;                // atoms of (cols, prows)
  int64_t rows, cols, ldx, prows;
  int64_t col_tiles, row_tiles;
};

template <int DT, bool ROWS, bool COLS, bool SCALED>
__global__ void __launch_bounds__(QTHREADS) mx_quant_kernel(const QuantArgs a) {
  using E = Elem<DT>;
  using Raw = typename E::Raw;
  // a few-token product may follow as this kernel's programmatic dependent
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  extern __shared__ __align__(16) uint8_t smem[];
  Raw* tile = reinterpret_cast<Raw*>(smem);                                      // COLS: [128][128]
  uint8_t* stage = smem + (COLS ? TILE * TILE * sizeof(Raw) : 0);                // COLS: [128][64]
  __shared__ __align__(16) uint8_t s_row[512], s_col[512];
  __shared__ float s_scale[TILE];
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int64_t tr = blockIdx.x / a.col_tiles, tc = blockIdx.x % a.col_tiles;
  const int64_t r0 = tr * TILE, c0 = tc * TILE;
  const int lc = 8 * (lane & 15);          // this lane's first column in the tile
  const bool col_ok = c0 + lc < a.cols;    // cols % 8 == 0: all 8 or none
  const Raw* x = static_cast<const Raw*>(a.x);

  float gam[8];
  if (SCALED) {
#pragma unroll
    for (int j = 0; j < 8; ++j) gam[j] = 1.0f;
    if (a.gamma && col_ok) {
      const uint16_t* gp = a.gamma + c0 + lc;
#pragma unroll
      for (int j = 0; j < 8; ++j) gam[j] = Elem<NVFP4B200_BF16>::get(gp + j);
    }
    if (tid < TILE) s_scale[tid] = r0 + tid < a.rows && a.row_scale ? __ldg(a.row_scale + r0 + tid) : 1.0f;
    __syncthreads();
  }

  typename E::Vec8 v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = r0 + wid * 16 + 2 * i + (lane >> 4);
    v[i] = E::zero();
    if (col_ok && r < a.rows) v[i] = E::load(x + r * a.ldx + c0 + lc);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int rl = wid * 16 + 2 * i + (lane >> 4);
    if (COLS) E::store(tile + rl * TILE + lc, v[i]);
    if (ROWS) {
      float f[8];
      E::unpack(v[i], f);
      if (SCALED) {
        const float rs = s_scale[rl];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = __fmul_rn(__fmul_rn(f[j], rs), gam[j]);
      }
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) m = max(m, absbits(f[j]));
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
      const uint32_t code = block_code(m);
      if ((lane & 3) == 0) s_row[atom_offset(rl, (lane & 15) >> 2)] = (uint8_t)code;
      const uint32_t nib = encode8(f, code_inverse(code));
      const int64_t r = r0 + rl;
      if (col_ok && r < a.rows) *reinterpret_cast<uint32_t*>(a.q + r * (a.cols >> 1) + ((c0 + lc) >> 1)) = nib;
    }
  }
  __syncthreads();
  if (COLS) {
    const int rb = wid >> 1, cp = ((wid & 1) << 5) + lane;   // 32-row block, column pair
    const Raw* t0 = tile + rb * 32 * TILE + 2 * cp;
    float g0 = 1.0f, g1 = 1.0f;
    if (SCALED && a.gamma && c0 + 2 * cp < a.cols) {
      g0 = Elem<NVFP4B200_BF16>::get(a.gamma + c0 + 2 * cp);
      g1 = Elem<NVFP4B200_BF16>::get(a.gamma + c0 + 2 * cp + 1);
    }
    auto at = [&](int r, float& f0, float& f1) {
      f0 = E::value(t0[r * TILE]);
      f1 = E::value(t0[r * TILE + 1]);
      if (SCALED) {
        const float rs = s_scale[rb * 32 + r];
        f0 = __fmul_rn(__fmul_rn(f0, rs), g0);
        f1 = __fmul_rn(__fmul_rn(f1, rs), g1);
      }
    };
    uint32_t m0 = 0, m1 = 0;
#pragma unroll
    for (int r = 0; r < 32; ++r) {
      float f0, f1;
      at(r, f0, f1);
      m0 = max(m0, absbits(f0));
      m1 = max(m1, absbits(f1));
    }
    const uint32_t code0 = block_code(m0), code1 = block_code(m1);
    s_col[atom_offset(2 * cp, rb)] = (uint8_t)code0;
    s_col[atom_offset(2 * cp + 1, rb)] = (uint8_t)code1;
    const float inv0 = code_inverse(code0), inv1 = code_inverse(code1);
    uint32_t n0[4], n1[4];
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      float f0[8], f1[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) at(8 * h + j, f0[j], f1[j]);
      n0[h] = encode8(f0, inv0);
      n1[h] = encode8(f1, inv1);
    }
    *reinterpret_cast<uint4*>(stage + (2 * cp) * 64 + rb * 16) = make_uint4(n0[0], n0[1], n0[2], n0[3]);
    *reinterpret_cast<uint4*>(stage + (2 * cp + 1) * 64 + rb * 16) = make_uint4(n1[0], n1[1], n1[2], n1[3]);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = i * 64 + (tid >> 2), piece = tid & 3;
      if (c0 + c < a.cols && r0 + 32 * piece < a.prows)
        *reinterpret_cast<uint4*>(a.qt + (c0 + c) * (a.prows >> 1) + ((r0 + 32 * piece) >> 1)) =
            *reinterpret_cast<const uint4*>(stage + c * 64 + piece * 16);
    }
  }
  if (ROWS && tid < 32)
    reinterpret_cast<uint4*>(a.s + (tr * a.col_tiles + tc) * 512)[tid] = reinterpret_cast<const uint4*>(s_row)[tid];
  if (COLS && tid >= 32 && tid < 64)
    reinterpret_cast<uint4*>(a.st + (tc * a.row_tiles + tr) * 512)[tid - 32] =
        reinterpret_cast<const uint4*>(s_col)[tid - 32];
}

template <int DT, bool ROWS, bool COLS, bool SCALED>
static int launch_quant(const QuantArgs& a, cudaStream_t st) {
  const int smem = COLS ? TILE * TILE * (int)sizeof(typename Elem<DT>::Raw) + TILE * 64 : 0;
  auto* fn = mx_quant_kernel<DT, ROWS, COLS, SCALED>;
  if (smem > 32 * 1024 &&   // with the static arrays, past the default limit
      cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return NVFP4B200_ERR_CUDA;
  fn<<<(unsigned)(a.row_tiles * a.col_tiles), QTHREADS, smem, st>>>(a);
  return launch_status();
}

template <int DT>
static int launch_quant_dt(const QuantArgs& a, cudaStream_t st) {
  const bool rows = a.q != nullptr, cols = a.qt != nullptr, scaled = a.row_scale || a.gamma;
  if (rows && cols) return scaled ? launch_quant<DT, true, true, true>(a, st) : launch_quant<DT, true, true, false>(a, st);
  if (rows) return scaled ? launch_quant<DT, true, false, true>(a, st) : launch_quant<DT, true, false, false>(a, st);
  return scaled ? launch_quant<DT, false, true, true>(a, st) : launch_quant<DT, false, true, false>(a, st);
}

// ---------------------------------------------------------------------------
// the way back
// ---------------------------------------------------------------------------

// Two nibbles of a byte -> two floats (low nibble first), exactly.
__device__ __forceinline__ float2 decode2(uint32_t byte) {
  uint32_t h;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b0;\n\t}"
      : "=r"(h)
      : "r"(byte));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// 8 elements per thread and step: 4 bytes of nibbles in, one 8-element vector
// out.  16 neighbouring lanes share one 4-byte word of four block scales.
template <int DT>
__global__ void __launch_bounds__(256) mx_dequant_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ s,
                                                         typename Elem<DT>::Raw* __restrict__ y, int64_t rows,
                                                         int64_t k, int64_t atoms) {
  const int64_t per_row = k >> 3;
  const int64_t n = rows * per_row;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / per_row, v = i - r * per_row;
    const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(q + r * (k >> 1)) + v);
    const int64_t blk = v >> 2;
    const uint32_t code = __ldg(s + ((r >> 7) * atoms + (blk >> 2)) * 512 + atom_offset((int)(r & 127), (int)(blk & 3)));
    const float sc = code_scale(code);
    float f[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 t = decode2((w >> (8 * j)) & 0xFFu);
      f[2 * j] = t.x * sc;
      f[2 * j + 1] = t.y * sc;
    }
    Elem<DT>::store(y + r * k + 8 * v, Elem<DT>::pack(f));
  }
}

}  // namespace mx

// Checked rows quantizer of bf16 x for the few-token product.
int mx_quant_rows_async(const void* x, void* q, void* s, int64_t rows, int64_t cols, int64_t ldx, cudaStream_t st) {
  return nvfp4b200_mx_quant(x, NVFP4B200_BF16, nullptr, nullptr, q, s, nullptr, nullptr, rows, cols, ldx, (void*)st);
}

}  // namespace nvfp4b200

using namespace nvfp4b200;

extern "C" {

int nvfp4b200_mx_quant(const void* x, int x_dtype, const float* row_scale, const void* gamma, void* q, void* s,
                       void* qt, void* st, int64_t rows, int64_t cols, int64_t ldx, void* stream) {
  if (!x || (!q && !qt) || (q == nullptr) != (s == nullptr) || (qt == nullptr) != (st == nullptr) ||
      !valid_dtype(x_dtype))
    return NVFP4B200_ERR_INVALID_ARG;
  if (rows < 0 || cols <= 0 || cols % 8 || (q && cols % 32) || ldx < cols || ldx % 8 || rows > (1ll << 30) ||
      cols > (1ll << 30))
    return NVFP4B200_ERR_BAD_SHAPE;
  if (!aligned(x, 16) || (q && !aligned(q, 16)) || (s && !aligned(s, 16)) || (qt && !aligned(qt, 16)) ||
      (st && !aligned(st, 16)) || (row_scale && !aligned(row_scale, 4)) || (gamma && !aligned(gamma, 16)))
    return NVFP4B200_ERR_MISALIGNED;
  mx::QuantArgs a;
  a.row_tiles = ceil_div(rows, mx::TILE);
  a.col_tiles = ceil_div(cols, mx::TILE);
  if (a.row_tiles * a.col_tiles > 0x7FFFFFFFll) return NVFP4B200_ERR_BAD_SHAPE;
  int rc = check_device();
  if (rc) return rc;
  if (rows == 0) return NVFP4B200_OK;
  a.x = x;
  a.row_scale = row_scale;
  a.gamma = static_cast<const uint16_t*>(gamma);
  a.q = static_cast<uint8_t*>(q);
  a.s = static_cast<uint8_t*>(s);
  a.qt = static_cast<uint8_t*>(qt);
  a.st = static_cast<uint8_t*>(st);
  a.rows = rows;
  a.cols = cols;
  a.ldx = ldx;
  a.prows = round_up(rows, 32);
  cudaStream_t cs = (cudaStream_t)stream;
  if (x_dtype == NVFP4B200_BF16) return mx::launch_quant_dt<NVFP4B200_BF16>(a, cs);
  if (x_dtype == NVFP4B200_F16) return mx::launch_quant_dt<NVFP4B200_F16>(a, cs);
  return mx::launch_quant_dt<NVFP4B200_F32>(a, cs);
}

int nvfp4b200_mx_dequant(const void* q, const void* s, void* y, int y_dtype, int64_t rows, int64_t k, void* stream) {
  if (!q || !s || !y || (y_dtype != NVFP4B200_BF16 && y_dtype != NVFP4B200_F32)) return NVFP4B200_ERR_INVALID_ARG;
  if (rows < 0 || k <= 0 || k % 32 || rows > (1ll << 30) || k > (1ll << 30)) return NVFP4B200_ERR_BAD_SHAPE;
  if (!aligned(q, 16) || !aligned(s, 16) || !aligned(y, 16)) return NVFP4B200_ERR_MISALIGNED;
  int rc = check_device();
  if (rc) return rc;
  if (rows == 0) return NVFP4B200_OK;
  const int64_t atoms = ceil_div(k, 128);
  const unsigned grid =
      (unsigned)std::min<int64_t>(ceil_div(rows * (k >> 3), 256), (int64_t)sm_count_current() * 16);
  cudaStream_t cs = (cudaStream_t)stream;
  const uint8_t *Q = static_cast<const uint8_t*>(q), *S = static_cast<const uint8_t*>(s);
  if (y_dtype == NVFP4B200_BF16)
    mx::mx_dequant_kernel<NVFP4B200_BF16><<<grid, 256, 0, cs>>>(Q, S, static_cast<uint16_t*>(y), rows, k, atoms);
  else
    mx::mx_dequant_kernel<NVFP4B200_F32><<<grid, 256, 0, cs>>>(Q, S, static_cast<float*>(y), rows, k, atoms);
  return launch_status();
}

}  // extern "C"
