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
// Traffic: 2 bytes read and 17/32 written per bf16 element and orientation.  The
// quantizer along rows and the way back are bound by HBM (92% of the copy rate
// and more), columns and both orientations at once by instructions too (84, 79%).
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

// max(|a|, |b|, |c|), NaN if any of them is.
__device__ __forceinline__ float absmax3(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

__device__ __forceinline__ float absmax2(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));   // both are magnitudes
  return d;
}
// ---------------------------------------------------------------------------
// quantizer: one CTA per 128 x 128 tile, which is one 512-byte scale atom of
// either orientation (128 rows x 4 blocks of 32 columns, 128 columns x 4
// blocks of 32 rows)
// ---------------------------------------------------------------------------
// Rows: 8 lanes read a row of the tile (16 elements each), a block is 2 lanes.
// Columns: the tile is kept in shared memory; a thread owns two neighbouring
// columns of half a 32-row block (16 rows, held in registers between the
// maximum and the encoding), neighbouring lanes the two halves.  Rows 16-31 of
// a block are shifted by half a bank cycle, so the two halves' reads do not
// meet in a bank.  The columns' nibbles are staged in shared memory (72 bytes
// a column, for the same reason) and written as 64-byte segments.
// Products are of packed pairs, and maxima take three operands: with both orientations the kernel is bound by its instructions,
// not by HBM.  112 us with one value at a time and the tile read twice, 80 us
// so (32768 x 4096 bf16, both orientations; 63 us of traffic).
constexpr int TILE = 128;
constexpr int QTHREADS = 256;
constexpr int STAGE_LD = 72;    // bytes per staged column

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

// First element of a row of the tile in shared memory: every 16 rows are
// shifted by 64 bytes, 16 of the 32 banks.
template <int DT>
__device__ __forceinline__ int tile_row(int r) {
  return r * TILE + (r >> 4) * (64 / (int)sizeof(typename Elem<DT>::Raw));
}
template <int DT>
constexpr int tile_bytes() { return TILE * TILE * (int)sizeof(typename Elem<DT>::Raw) + TILE / 16 * 64; }

// Two neighbouring elements as stored.
template <int DT>
struct Pair {   // 16-bit types: one word
  using T = uint32_t;
  static __device__ __forceinline__ uint64_t f2(T w) {
    if (DT == NVFP4B200_BF16) return bf16x2_to_f2(w);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    return f2pack(f.x, f.y);
  }
};
template <>
struct Pair<NVFP4B200_F32> {
  using T = uint64_t;
  static __device__ __forceinline__ uint64_t f2(T w) { return w; }
};

// 8 values given as pairs -> 8 nibbles, each value times inv.
__device__ __forceinline__ uint32_t encode_pairs(const uint64_t* v, float inv) {
  const uint64_t i2 = f2pack(inv, inv);
  float f[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint64_t p = f2mul(v[j], i2);
    f[2 * j] = f2lo(p);
    f[2 * j + 1] = f2hi(p);
  }
  return encode8(f);
}

template <int DT, bool ROWS, bool COLS, bool SCALED>
__global__ void __launch_bounds__(QTHREADS, DT == NVFP4B200_F32 && (COLS || SCALED) ? 2 : DT == NVFP4B200_F32 || (SCALED && ROWS) ? 3 : 4)
    mx_quant_kernel(const QuantArgs a) {
  using E = Elem<DT>;
  using Raw = typename E::Raw;
  using P = Pair<DT>;
  constexpr bool HALF = DT != NVFP4B200_F32;    // 16-bit elements
  constexpr int VL = 2;                         // 8-element vectors per lane and pass
  constexpr int LPR = TILE / (8 * VL);          // lanes per row
  constexpr int PASSES = 4;                     // a warp's 16 rows, 4 at a time
  // a few-token product may follow as this kernel's programmatic dependent
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  extern __shared__ __align__(16) uint8_t smem[];
  Raw* tile = reinterpret_cast<Raw*>(smem);                 // COLS: the tile, then the staged columns
  uint8_t* stage = smem + (COLS ? tile_bytes<DT>() : 0);
  __shared__ __align__(16) uint8_t s_row[512], s_col[512];
  __shared__ __align__(16) float2 s_scale[TILE];   // each row's scale twice, as a packed pair
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int tr = (int)(blockIdx.x / (unsigned)a.col_tiles), tc = (int)(blockIdx.x - tr * (unsigned)a.col_tiles);
  const int64_t r0 = (int64_t)tr * TILE, c0 = (int64_t)tc * TILE;
  const int lc = 8 * VL * (lane % LPR);    // this lane's first column in the tile
  const int row0 = wid * 16 + lane / LPR;  // its first row; a pass is 4 rows of the warp's 16
  const Raw* x = static_cast<const Raw*>(a.x) + (r0 + row0) * a.ldx + c0 + lc;
  const int rows_here = (int)imin64(TILE, a.rows - r0);
  bool ok[VL];                             // cols % 8 == 0: each vector of 8 whole or not at all
#pragma unroll
  for (int h = 0; h < VL; ++h) ok[h] = c0 + lc + 8 * h < a.cols;

  typename E::Vec8 v[PASSES][VL];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
#pragma unroll
    for (int h = 0; h < VL; ++h) {
      v[i][h] = E::zero();
      if (ok[h] && row0 + 4 * i < rows_here) v[i][h] = E::load(x + 8 * h);
    }
    x += 4 * a.ldx;
  }
  uint64_t gam[4 * VL];
  if (SCALED) {
#pragma unroll
    for (int j = 0; j < 4 * VL; ++j) gam[j] = f2pack(1.0f, 1.0f);
    if (ROWS && a.gamma && ok[0]) {   // rows: cols % 32 == 0, all of a lane's columns or none
#pragma unroll
      for (int h = 0; h < VL; ++h) {
        const uint4 g = __ldg(reinterpret_cast<const uint4*>(a.gamma + c0 + lc) + h);
        gam[4 * h] = bf16x2_to_f2(g.x); gam[4 * h + 1] = bf16x2_to_f2(g.y);
        gam[4 * h + 2] = bf16x2_to_f2(g.z); gam[4 * h + 3] = bf16x2_to_f2(g.w);
      }
    }
    if (tid < TILE) {
      const float v = tid < rows_here && a.row_scale ? __ldg(a.row_scale + r0 + tid) : 1.0f;
      s_scale[tid] = make_float2(v, v);
    }
    __syncthreads();
  }
  uint8_t* q = ROWS ? a.q + (r0 + row0) * (a.cols >> 1) + ((c0 + lc) >> 1) : nullptr;
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int rl = row0 + 4 * i;
    if (COLS) {
      Raw* t = tile + tile_row<DT>(rl) + lc;
      // lanes 4-7 of eight store their second vector first: no two of a quarter warp meet in a bank
      const bool swap = (lane & 4) != 0;
      E::store(t + (swap ? 8 : 0), swap ? v[i][1] : v[i][0]);
      E::store(t + (swap ? 0 : 8), swap ? v[i][0] : v[i][1]);
    }
    if (ROWS) {
      uint64_t f[4 * VL];
#pragma unroll
      for (int h = 0; h < VL; ++h) {
        if constexpr (HALF) {
          f[4 * h] = P::f2(v[i][h].a.x); f[4 * h + 1] = P::f2(v[i][h].a.y);
          f[4 * h + 2] = P::f2(v[i][h].a.z); f[4 * h + 3] = P::f2(v[i][h].a.w);
        } else {
          f[4 * h] = f2pack(v[i][h].a.x, v[i][h].a.y); f[4 * h + 1] = f2pack(v[i][h].a.z, v[i][h].a.w);
          f[4 * h + 2] = f2pack(v[i][h].b.x, v[i][h].b.y); f[4 * h + 3] = f2pack(v[i][h].b.z, v[i][h].b.w);
        }
      }
      if (SCALED) {
        const uint64_t rs = *reinterpret_cast<const uint64_t*>(s_scale + rl);
#pragma unroll
        for (int j = 0; j < 4 * VL; ++j) f[j] = f2mul(f2mul(f[j], rs), gam[j]);
      }
      float m = absmax3(f2lo(f[0]), f2hi(f[0]), f2lo(f[1]));
#pragma unroll
      for (int j = 1; j < 4 * VL - 1; ++j) m = absmax3(m, f2hi(f[j]), f2lo(f[j + 1]));
      m = absmax3(m, f2hi(f[4 * VL - 1]), f2hi(f[4 * VL - 1]));
      m = absmax2(m, __shfl_xor_sync(0xffffffffu, m, 1));
      const bool here = ok[0] && rl < rows_here;
      uint32_t code;
      float inv;
      block_scale(m, code, inv);
      // a block's two lanes write the one byte together; padding is 0
      s_row[atom_offset(rl, (lane % LPR) >> 1)] = (uint8_t)(here ? code : 0u);
      const uint2 nib = make_uint2(encode_pairs(f, inv), encode_pairs(f + 4, inv));
      if (here) *reinterpret_cast<uint2*>(q) = nib;
      q += 2 * a.cols;   // four rows of cols / 2 bytes
    }
  }
  __syncthreads();
  if (COLS) {
    const int half = lane & 1;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int task = wid + 8 * h;                       // 16 tasks: 4 row blocks x 4 runs of 16 column pairs
      const int rb = task >> 2, cp = ((task & 3) << 4) + (lane >> 1);
      const Raw* t0 = tile + tile_row<DT>(32 * rb + 16 * half) + 2 * cp;
      uint64_t g2 = f2pack(1.0f, 1.0f);
      if (SCALED && a.gamma && c0 + 2 * cp < a.cols)
        g2 = bf16x2_to_f2(__ldg(reinterpret_cast<const uint32_t*>(a.gamma + c0 + 2 * cp)));
      typename P::T w[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) w[r] = *reinterpret_cast<const typename P::T*>(t0 + r * TILE);
      uint64_t f[SCALED ? 16 : 1];
      float m0 = 0.0f, m1 = 0.0f;
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        uint64_t p = P::f2(w[r]), n = P::f2(w[r + 1]);
        if (SCALED) {
          const ulonglong2 rs = *reinterpret_cast<const ulonglong2*>(s_scale + 32 * rb + 16 * half + r);
          f[SCALED ? r : 0] = p = f2mul(f2mul(p, rs.x), g2);
          f[SCALED ? r + 1 : 0] = n = f2mul(f2mul(n, rs.y), g2);
        }
        m0 = absmax3(m0, f2lo(p), f2lo(n));
        m1 = absmax3(m1, f2hi(p), f2hi(n));
      }
      m0 = absmax2(m0, __shfl_xor_sync(0xffffffffu, m0, 1));
      m1 = absmax2(m1, __shfl_xor_sync(0xffffffffu, m1, 1));
      const bool block_ok = c0 + 2 * cp < a.cols && 32 * rb < rows_here;   // cols % 8 == 0: both columns or none
      uint32_t code0, code1;
      float inv0, inv1;
      block_scale(m0, code0, inv0);
      block_scale(m1, code1, inv1);
      // lane pairs: the even lane writes the even column's code, the odd lane the odd one's
      s_col[atom_offset(2 * cp + half, rb)] = (uint8_t)(!block_ok ? 0u : half ? code1 : code0);
      const uint64_t inv = f2pack(inv0, inv1);
      uint32_t n0[2], n1[2];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        float a0[8], a1[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint64_t p = f2mul(SCALED ? f[SCALED ? 8 * g + j : 0] : P::f2(w[8 * g + j]), inv);
          a0[j] = f2lo(p);
          a1[j] = f2hi(p);
        }
        n0[g] = encode8(a0);
        n1[g] = encode8(a1);
      }
      uint8_t* dst = stage + (2 * cp) * STAGE_LD + rb * 16 + half * 8;
      *reinterpret_cast<uint2*>(dst) = make_uint2(n0[0], n0[1]);
      *reinterpret_cast<uint2*>(dst + STAGE_LD) = make_uint2(n1[0], n1[1]);
    }
    __syncthreads();
    uint8_t* qt = a.qt + c0 * (a.prows >> 1) + (r0 >> 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = i * 32 + (tid >> 3), piece = tid & 7;   // 16 rows' nibbles
      if (c0 + c < a.cols && r0 + 16 * piece < a.prows)
        *reinterpret_cast<uint2*>(qt + c * (a.prows >> 1) + 8 * piece) =
            *reinterpret_cast<const uint2*>(stage + c * STAGE_LD + 8 * piece);
    }
  }
  if (ROWS && tid < 32)
    reinterpret_cast<uint4*>(a.s + ((int64_t)tr * a.col_tiles + tc) * 512)[tid] = reinterpret_cast<const uint4*>(s_row)[tid];
  if (COLS && tid >= 32 && tid < 64)
    reinterpret_cast<uint4*>(a.st + ((int64_t)tc * a.row_tiles + tr) * 512)[tid - 32] =
        reinterpret_cast<const uint4*>(s_col)[tid - 32];
}

template <int DT, bool ROWS, bool COLS, bool SCALED>
static int launch_quant(const QuantArgs& a, cudaStream_t st) {
  constexpr int SMEM = COLS ? tile_bytes<DT>() + TILE * STAGE_LD : 0;
  auto* fn = mx_quant_kernel<DT, ROWS, COLS, SCALED>;
  if (SMEM > 32 * 1024 && !allow_smem(fn, SMEM)) return NVFP4B200_ERR_CUDA;   // with the static arrays, past the default limit
  fn<<<(unsigned)(a.row_tiles * a.col_tiles), QTHREADS, SMEM, st>>>(a);
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

// A warp takes 2048 columns of a row: 8 elements per lane and step (4 bytes of
// nibbles in, one or two 16-byte vectors out), all its reads issued first.
// Neighbouring warps take neighbouring rows, which share scale atoms in L1.
constexpr int DQ_WARPS = 8, DQ_STEPS = 8, DQ_COLS = 256 * DQ_STEPS;

template <int DT>
__global__ void __launch_bounds__(32 * DQ_WARPS) mx_dequant_kernel(const uint8_t* __restrict__ q,
                                                                  const uint8_t* __restrict__ s,
                                                                  typename Elem<DT>::Raw* __restrict__ y, int64_t rows,
                                                                  int64_t k, int64_t atoms, int chunks) {
  const int lane = threadIdx.x & 31;
  const int64_t r = (int64_t)(blockIdx.x / (unsigned)chunks) * DQ_WARPS + (threadIdx.x >> 5);
  const int64_t c0 = (int64_t)(blockIdx.x % (unsigned)chunks) * DQ_COLS + 8 * lane;
  if (r >= rows) return;
  const uint8_t* qr = q + r * (k >> 1);
  const uint8_t* sr = s + (r >> 7) * atoms * 512 + atom_offset((int)(r & 127), 0);
  uint32_t w[DQ_STEPS], code[DQ_STEPS];
#pragma unroll
  for (int i = 0; i < DQ_STEPS; ++i) {
    const int64_t c = c0 + 256 * i;   // k % 32 == 0: all 8 or none
    w[i] = code[i] = 0;
    if (c < k) {
      w[i] = __ldg(reinterpret_cast<const uint32_t*>(qr + (c >> 1)));
      code[i] = __ldg(sr + (c >> 7) * 512 + ((c >> 5) & 3));
    }
  }
#pragma unroll
  for (int i = 0; i < DQ_STEPS; ++i) {
    const int64_t c = c0 + 256 * i;
    if (c >= k) return;
    const float sc = code_scale(code[i]);
    float f[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 t = decode2((w[i] >> (8 * j)) & 0xFFu);
      f[2 * j] = t.x * sc;
      f[2 * j + 1] = t.y * sc;
    }
    Elem<DT>::store(y + r * k + c, Elem<DT>::pack(f));
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
  const int64_t atoms = ceil_div(k, 128), chunks = ceil_div(k, mx::DQ_COLS);
  const int64_t grid = ceil_div(rows, mx::DQ_WARPS) * chunks;
  if (grid > 0x7FFFFFFFll) return NVFP4B200_ERR_BAD_SHAPE;
  cudaStream_t cs = (cudaStream_t)stream;
  const uint8_t *Q = static_cast<const uint8_t*>(q), *S = static_cast<const uint8_t*>(s);
  if (y_dtype == NVFP4B200_BF16)
    mx::mx_dequant_kernel<NVFP4B200_BF16>
        <<<(unsigned)grid, 32 * mx::DQ_WARPS, 0, cs>>>(Q, S, static_cast<uint16_t*>(y), rows, k, atoms, (int)chunks);
  else
    mx::mx_dequant_kernel<NVFP4B200_F32>
        <<<(unsigned)grid, 32 * mx::DQ_WARPS, 0, cs>>>(Q, S, static_cast<float*>(y), rows, k, atoms, (int)chunks);
  return launch_status();
}

}  // extern "C"
