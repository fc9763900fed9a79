// The RMSNorms after and before a block, fused with the block's gate and the
// residual's scale (B200, sm_100a).
//
//     y = alpha * x + s * gate[g] * (b * inv_b * gamma_post),   inv_b = rsqrt(mean(b^2) + eps)
//     n = y * inv_y * gamma_pre,                                inv_y = rsqrt(mean(y^2) + eps)
//
// b is the block's output, x the residual stream, gate [G, D] belongs to G
// equal runs of rows (G = 1: a channel gate, G = sequences: a gate of their
// own), n the next block's input.  n and inv_y come from y before y is rounded
// to its type: each output is rounded once, from fp32 (n of the rounded y has
// 1.4 times the error in bf16).
//
// Backward, given dy (the gradient that reaches y from behind) and dn:
//     yh = y * inv_y;  v = dn * gamma_pre
//     t  = dy + inv_y * (v - yh * mean(v * yh))
//     dx = alpha * t
//     bh = b * inv_b;  u = s * t * gate * gamma_post
//     db = inv_b * (u - bh * mean(u * bh))
//     S_g = sum over the rows of g of s * t * bh
//     dgate[g] = gamma_post * S_g;  dgamma_post = sum_g gate[g] * S_g
//     dgamma_pre = sum over rows of dn * yh
// so one column sum per group carries both the gate's and the norm weight's
// gradient.  All statistics and sums are fp32; column sums are added up in a
// fixed order (rows in a CTA, CTAs in a second kernel), never by atomics.
//
// Bound: HBM, one read of each input and one write of each output.
#include "bulk.cuh"
#include "row_stop.h"
#include "vec.cuh"

#include <algorithm>
#include <type_traits>

namespace nvfp4b200 {
namespace norm {

constexpr int VPT = 2;            // 8-element vectors per thread and row
constexpr int CPT = 8 * VPT;      // columns per thread
constexpr int MAX_D = 1024 * CPT;
constexpr int MAX_SMEM = 225 * 1024;   // dynamic, of one CTA: 227 KB less the static arrays; every kernel's limit
// what n CTAs of an SM can each have: its 228 KB less 1 KB per CTA that the system takes and 1 KB of static arrays
constexpr int smem_share(int n) { return n <= 1 ? MAX_SMEM : 228 * 1024 / n - 2048; }

// Threads of a CTA of the forward: rows of TPR threads each, 256 threads or a little more.
constexpr int threads_of(int tpr) { return (tpr < 256 ? (255 + tpr) / tpr : 1) * tpr; }

template <int DT>
constexpr int dtype_size() { return DT == NVFP4B200_F32 ? 4 : 2; }

// Column of a thread's element j: vectors of 8 (VEC), or strided single
// elements for widths and strides that no 16-byte vector fits.
template <bool VEC, int TPR>
__device__ __forceinline__ int column(int t, int j) {
  return VEC ? (j >> 3) * (TPR * 8) + 8 * t + (j & 7) : j * TPR + t;
}

// One row's elements of a tensor as raw vectors (VEC) or floats.
template <int DT, bool VEC, int TPR, int V = VPT>
struct Row {
  typename Elem<DT>::Vec8 v[VEC ? V : 1];
  float f[VEC ? 1 : 8 * V];

  __device__ __forceinline__ void load(const typename Elem<DT>::Raw* p, int t, int d) {
    if (VEC) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int c = column<true, TPR>(t, 8 * i);
        v[i] = Elem<DT>::zero();
        if (c < d) v[i] = Elem<DT>::load(p + c);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8 * V; ++j) {
        const int c = column<false, TPR>(t, j);
        f[j] = c < d ? Elem<DT>::get(p + c) : 0.0f;
      }
    }
  }
  __device__ __forceinline__ void values(float (&o)[8 * V]) const {
    if (VEC) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float t[8];
        Elem<DT>::unpack(v[i], t);
#pragma unroll
        for (int j = 0; j < 8; ++j) o[8 * i + j] = t[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8 * V; ++j) o[j] = f[j];
    }
  }
};

// Rounds the values to the stored type and writes them.
template <int DT, bool VEC, int TPR, int V = VPT>
__device__ __forceinline__ void store_row(typename Elem<DT>::Raw* p, int t, int d, const float (&o)[8 * V]) {
  if (VEC) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = column<true, TPR>(t, 8 * i);
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = o[8 * i + j];
      if (c < d) Elem<DT>::store(p + c, Elem<DT>::pack(f));
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8 * V; ++j) {
      const int c = column<false, TPR>(t, j);
      if (c < d) p[c] = Elem<DT>::bits(o[j]);
    }
  }
}

// Sum over the TPR threads of a row; the same bits in every thread.
template <int TPR>
__device__ __forceinline__ float row_sum(float s, float* red, int group) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (TPR == 32) return s;
  constexpr int W = TPR / 32;
  const int w = (threadIdx.x % TPR) >> 5;
  if ((threadIdx.x & 31) == 0) red[group * W + w] = s;
  if (TPR == 1024 || TPR == (int)blockDim.x) __syncthreads();
  else asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(TPR) : "memory");
  s = 0.0f;
#pragma unroll
  for (int i = 0; i < W; ++i) s += red[group * W + i];
  return s;
}

template <int DT>
struct Pairs;   // 8 stored elements -> 4 packed pairs
template <>
struct Pairs<NVFP4B200_BF16> {
  static __device__ __forceinline__ void get(const uint4* p, int stride, uint64_t (&o)[4]) {
    const uint4 v = *p;
    o[0] = bf16x2_to_f2(v.x); o[1] = bf16x2_to_f2(v.y); o[2] = bf16x2_to_f2(v.z); o[3] = bf16x2_to_f2(v.w);
  }
};
template <>
struct Pairs<NVFP4B200_F16> {
  static __device__ __forceinline__ void get(const uint4* p, int stride, uint64_t (&o)[4]) {
    const uint4 v = *p;
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      o[i] = f2pack(f.x, f.y);
    }
  }
};
template <>
struct Pairs<NVFP4B200_F32> {
  static __device__ __forceinline__ void get(const uint4* p, int stride, uint64_t (&o)[4]) {
    const uint4 a = p[0], b = p[stride];
    o[0] = ((uint64_t)a.y << 32) | a.x; o[1] = ((uint64_t)a.w << 32) | a.z;
    o[2] = ((uint64_t)b.y << 32) | b.x; o[3] = ((uint64_t)b.w << 32) | b.z;
  }
};

__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src)
               : "memory");
}
__device__ __forceinline__ uint64_t f2two(float v) { return f2pack(v, v); }
__device__ __forceinline__ float f2sum(uint64_t v) { return f2lo(v) + f2hi(v); }

constexpr int STAGES = 3;

// Set when a bounded wait for a copy gave up.
__device__ int g_norm_error = 0;

struct FwdArgs {
  const void *b, *x, *gamma_post, *gate, *gamma_pre;
  void *y, *n;
  float *inv_b, *inv_y;
  int64_t rows, ldb, ldx, rows_per_gate;
  int d;
  float alpha, s, eps;
  int pre;
  int stages;               // unaligned rows: rows of the ring
  int64_t safe_rows;        // those whose 16-byte windows lie inside both tensors
  int64_t rows_per_cta;
};

template <int DT, bool VEC, int TPR>
__global__ void __launch_bounds__(threads_of(TPR)) sandwich_fwd_kernel(const FwdArgs a) {
  using Raw = typename Elem<DT>::Raw;
  constexpr int GROUPS = threads_of(TPR) / TPR;
  __shared__ float red[4][GROUPS * (TPR / 32)];
  const int group = threadIdx.x / TPR, t = threadIdx.x % TPR;
  const Raw *B = static_cast<const Raw*>(a.b), *X = static_cast<const Raw*>(a.x);
  const float inv_d = 1.0f / (float)a.d;
  int buf = 0;
  for (int64_t r = (int64_t)blockIdx.x * GROUPS + group; r < a.rows; r += (int64_t)gridDim.x * GROUPS) {
    Row<DT, VEC, TPR> rb, rx, rw;
    float b[CPT], o[CPT], w[CPT];
    rb.load(B + r * a.ldb, t, a.d);
    rx.load(X + r * a.ldx, t, a.d);
    rb.values(b);
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < CPT; ++j) ss = fmaf(b[j], b[j], ss);
    const float inv_b = rsqrtf(row_sum<TPR>(ss, red[buf], group) * inv_d + a.eps);
#pragma unroll
    for (int j = 0; j < CPT; ++j) b[j] *= inv_b;
    if (a.gamma_post) {
      rw.load(static_cast<const Raw*>(a.gamma_post), t, a.d);
      rw.values(w);
#pragma unroll
      for (int j = 0; j < CPT; ++j) b[j] *= w[j];
    }
    if (a.gate) {
      rw.load(static_cast<const Raw*>(a.gate) + (r / a.rows_per_gate) * a.d, t, a.d);
      rw.values(w);
#pragma unroll
      for (int j = 0; j < CPT; ++j) b[j] *= w[j];
    }
    rx.values(o);
#pragma unroll
    for (int j = 0; j < CPT; ++j) o[j] = fmaf(a.s, b[j], a.alpha * o[j]);
    store_row<DT, VEC, TPR>(static_cast<Raw*>(a.y) + r * a.d, t, a.d, o);
    if (t == 0) a.inv_b[r] = inv_b;
    if (a.pre) {
      ss = 0.0f;
#pragma unroll
      for (int j = 0; j < CPT; ++j) ss = fmaf(o[j], o[j], ss);
      const float inv_y = rsqrtf(row_sum<TPR>(ss, red[buf + 1], group) * inv_d + a.eps);
#pragma unroll
      for (int j = 0; j < CPT; ++j) o[j] *= inv_y;
      if (a.gamma_pre) {
        rw.load(static_cast<const Raw*>(a.gamma_pre), t, a.d);
        rw.values(w);
#pragma unroll
        for (int j = 0; j < CPT; ++j) o[j] *= w[j];
      }
      store_row<DT, VEC, TPR>(static_cast<Raw*>(a.n) + r * a.d, t, a.d, o);
      if (t == 0) a.inv_y[r] = inv_y;
    }
    buf ^= 2;   // a row's two sums use two slots; a slot is written again two rows later, past two barriers
  }
}

// The same forward with the rows staged ahead in shared memory: every thread
// copies its own columns of b and x (cp.async, 16 bytes each) into a ring of
// STAGES rows and reads back only what it copied, so the ring needs no
// barrier and the loads of the next rows run while a row waits for its two
// reductions.  (The second sum is not folded into the first exchange: y's
// square sum from those of its parts cancels where y is small.)
template <int DT, int TPR, int V>
__global__ void __launch_bounds__(threads_of(TPR), 1024 / threads_of(TPR))
    sandwich_fwd_staged_kernel(const FwdArgs a) {
  using E = Elem<DT>;
  using Raw = typename E::Raw;
  constexpr int Q = (int)sizeof(Raw) * 8 / 16;
  constexpr int NP = 4 * V;
  constexpr int THREADS = threads_of(TPR), GROUPS = THREADS / TPR;
  extern __shared__ __align__(16) uint4 ring[];   // [STAGES][2][V * Q][THREADS]
  __shared__ float red[4][GROUPS * (TPR / 32)];
  const int group = threadIdx.x / TPR, t = threadIdx.x % TPR;
  const float inv_d = 1.0f / (float)a.d;
  const int64_t step = (int64_t)gridDim.x * GROUPS;
  auto slot = [&](int stage, int tensor, int piece) {
    return ring + ((stage * 2 + tensor) * (V * Q) + piece) * THREADS + threadIdx.x;
  };
  // first column of a 16-byte piece: neighbouring lanes' pieces are neighbours (fp32 8192 x 4096:
  // 146 us with a thread's two pieces side by side, half a sector each, 88 so)
  auto at = [&](int i, int q) { return ((i * Q + q) * TPR + t) * (8 / Q); };
  auto fetch = [&](int64_t r, int stage) {
    if (r < a.rows) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const Raw* row = k ? static_cast<const Raw*>(a.x) + r * a.ldx : static_cast<const Raw*>(a.b) + r * a.ldb;
#pragma unroll
        for (int i = 0; i < V; ++i) {
#pragma unroll
          for (int q = 0; q < Q; ++q)
            if (at(i, q) < a.d) cp_async16(slot(stage, k, i * Q + q), row + at(i, q));
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < V; ++i)   // columns past the end stay zero in every stage
    for (int q = 0; q < Q; ++q)
      if (at(i, q) >= a.d)
        for (int k = 0; k < STAGES * 2; ++k) *slot(k >> 1, k & 1, i * Q + q) = make_uint4(0, 0, 0, 0);
  int64_t r = (int64_t)blockIdx.x * GROUPS + group;
#pragma unroll
  for (int st = 0; st < STAGES - 1; ++st) fetch(r + st * step, st);

  // a weight vector's pairs times v, or v where there is none
  auto weigh = [&](const typename E::Vec8 (&w)[V], uint64_t (&v)[NP]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float f[8];
      E::unpack(w[i], f);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[4 * i + j] = f2mul(v[4 * i + j], f2pack(f[2 * j], f[2 * j + 1]));
    }
  };
  auto load_w = [&](const void* p, int64_t off, typename E::Vec8 (&w)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      w[i] = E::zero();
      const Raw* row = static_cast<const Raw*>(p) + off;
      if constexpr (Q == 1) {
        if (at(i, 0) < a.d) w[i] = E::load(row + at(i, 0));
      } else {
        if (at(i, 0) < a.d) w[i].a = *reinterpret_cast<const float4*>(row + at(i, 0));
        if (at(i, 1) < a.d) w[i].b = *reinterpret_cast<const float4*>(row + at(i, 1));
      }
    }
  };
  auto put = [&](void* base, int64_t r, const uint64_t (&v)[NP]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float f[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f[2 * j] = f2lo(v[4 * i + j]);
        f[2 * j + 1] = f2hi(v[4 * i + j]);
      }
      Raw* row = static_cast<Raw*>(base) + r * a.d;
      if constexpr (Q == 1) {
        if (at(i, 0) < a.d) E::store(row + at(i, 0), E::pack(f));
      } else {
        const auto v8 = E::pack(f);
        if (at(i, 0) < a.d) *reinterpret_cast<float4*>(row + at(i, 0)) = v8.a;
        if (at(i, 1) < a.d) *reinterpret_cast<float4*>(row + at(i, 1)) = v8.b;
      }
    }
  };
  int stage = 0, buf = 0;
  for (; r < a.rows; r += step) {
    typename E::Vec8 wp[V], wg[V], wn[V];   // read (from L1 after the first row) ahead of the reductions
    if (a.gamma_post) load_w(a.gamma_post, 0, wp);
    if (a.gate) load_w(a.gate, (r / a.rows_per_gate) * a.d, wg);
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    uint64_t v[NP], ss = 0ull;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      uint64_t p[4];
      Pairs<DT>::get(slot(stage, 0, i * Q), THREADS, p);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[4 * i + j] = p[j];
        ss = f2fma(p[j], p[j], ss);
      }
    }
    fetch(r + (STAGES - 1) * step, stage == 0 ? STAGES - 1 : stage - 1);
    const float inv_b = rsqrtf(row_sum<TPR>(f2sum(ss), red[buf], group) * inv_d + a.eps);
#pragma unroll
    for (int j = 0; j < NP; ++j) v[j] = f2mul(v[j], f2two(inv_b));
    if (a.gamma_post) weigh(wp, v);
    if (a.gate) weigh(wg, v);
    if (a.gamma_pre) load_w(a.gamma_pre, 0, wn);
    ss = 0ull;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      uint64_t x[4];
      Pairs<DT>::get(slot(stage, 1, i * Q), THREADS, x);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint64_t& y = v[4 * i + j];
        y = f2fma(f2two(a.s), y, f2mul(f2two(a.alpha), x[j]));
        ss = f2fma(y, y, ss);
      }
    }
    put(a.y, r, v);
    if (t == 0) a.inv_b[r] = inv_b;
    if (a.pre) {
      const float inv_y = rsqrtf(row_sum<TPR>(f2sum(ss), red[buf + 1], group) * inv_d + a.eps);
#pragma unroll
      for (int j = 0; j < NP; ++j) v[j] = f2mul(v[j], f2two(inv_y));
      if (a.gamma_pre) weigh(wn, v);
      put(a.n, r, v);
      if (t == 0) a.inv_y[r] = inv_y;
    }
    buf ^= 2;
    stage = stage == STAGES - 1 ? 0 : stage + 1;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// The forward for rows that do not start on 16-byte boundaries: one thread
// copies each row's window of whole 16-byte pieces of b and x into a ring, as
// in the backward below; a thread's eight columns are TPR apart and are read
// and written one by one.  The last rows, whose windows could reach past the
// tensors, are read straight from global memory.
template <int DT, int TPR>
__global__ void __launch_bounds__(TPR, 1024 / TPR) sandwich_fwd_odd_kernel(const FwdArgs a) {
  using E = Elem<DT>;
  using Raw = typename E::Raw;
  extern __shared__ __align__(16) uint8_t odd_ring[];   // [stages][2][slot]
  __shared__ float red[4][TPR / 32];
  __shared__ __align__(8) uint64_t full[STAGES];
  __shared__ int stop;   // row_stop.h: set where a wait ran out
  const int t = threadIdx.x;
  const float inv_d = 1.0f / (float)a.d;
  const int row_bytes = a.d * (int)sizeof(Raw), slot = ((row_bytes + 15) & ~15) + 16;
  auto skew = [&](int64_t r, int64_t ld) { return (int)((uint64_t)(r * ld) * sizeof(Raw) & 15); };
  const int64_t r0 = (int64_t)blockIdx.x * a.rows_per_cta, end = imin64(a.rows, r0 + a.rows_per_cta);
  const int64_t safe = imin64(end, a.safe_rows);
  auto fetch = [&](int64_t r, int stage) {   // one thread
    if (r >= safe) return;
    uint8_t* dst = odd_ring + (size_t)stage * 2 * slot;
    const int ob = skew(r, a.ldb), ox = skew(r, a.ldx);
    const uint32_t nb = (uint32_t)((ob + row_bytes + 15) & ~15), nx = (uint32_t)((ox + row_bytes + 15) & ~15);
    bulk::expect(&full[stage], nb + nx);
    bulk::copy(dst, static_cast<const uint8_t*>(a.b) + r * a.ldb * (int64_t)sizeof(Raw) - ob, nb, &full[stage]);
    bulk::copy(dst + slot, static_cast<const uint8_t*>(a.x) + r * a.ldx * (int64_t)sizeof(Raw) - ox, nx, &full[stage]);
  };
  if (t == 0) {
    stop = row_stop::NEVER;
    bulk::init(full, STAGES);
  }
  __syncthreads();
  if (t == 0)
    for (int st = 0; st < a.stages; ++st) fetch(r0 + st, st);
  // the weights stay in registers: s * gamma_post * gate of the rows' group, gamma_pre
  float w[8], wn[8];
  int64_t group = -1;
  auto times = [&](const void* p, int64_t off, float (&f)[8]) {   // past the row's end its last element
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] *= E::get(static_cast<const Raw*>(p) + off + min(t + j * TPR, a.d - 1));
  };
#pragma unroll
  for (int j = 0; j < 8; ++j) wn[j] = 1.0f;
  if (a.gamma_pre) times(a.gamma_pre, 0, wn);
  int stage = 0, buf = 0;
  uint32_t parity = 0;
  for (int64_t r = r0; r < end; ++r) {
    if (r / a.rows_per_gate != group) {
      group = r / a.rows_per_gate;
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = a.s;
      if (a.gamma_post) times(a.gamma_post, 0, w);
      if (a.gate) times(a.gate, group * a.d, w);
    }
    const bool staged = r < safe;
    if (staged && !bulk::wait(&full[stage], parity)) atomicMin(&stop, row_stop::before_barrier((int)(r - r0)));
    const uint8_t* src = odd_ring + (size_t)stage * 2 * slot;
    const Raw* rb = staged ? reinterpret_cast<const Raw*>(src + skew(r, a.ldb)) : static_cast<const Raw*>(a.b) + r * a.ldb;
    const Raw* rx = staged ? reinterpret_cast<const Raw*>(src + slot + skew(r, a.ldx)) : static_cast<const Raw*>(a.x) + r * a.ldx;
    auto put = [&](void* out, const float (&f)[8]) {
      Raw* o = static_cast<Raw*>(out) + r * a.d + t;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (t + j * TPR < a.d) o[j * TPR] = E::bits(f[j]);
    };
    float v[8], x[8], ss = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = min(t + j * TPR, a.d - 1);
      v[j] = E::value(rb[c]);
      x[j] = E::value(rx[c]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = t + j * TPR < a.d ? fmaf(v[j], v[j], ss) : ss;
    const float inv_b = rsqrtf(row_sum<TPR>(ss, red[buf], 0) * inv_d + a.eps);
    // past the sum's barrier every thread has read the row: its place is refilled,
    // where its copies arrived (a barrier whose phase is open takes no second ones)
    if (row_stop::leaves(stop, (int)(r - r0))) break;
    if (t == 0) fetch(r + a.stages, stage);
    ss = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[j] = fmaf(v[j] * inv_b, w[j], a.alpha * x[j]);
      ss = t + j * TPR < a.d ? fmaf(v[j], v[j], ss) : ss;
    }
    put(a.y, v);
    if (t == 0) a.inv_b[r] = inv_b;
    if (a.pre) {
      const float inv_y = rsqrtf(row_sum<TPR>(ss, red[buf + 1], 0) * inv_d + a.eps);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= inv_y * wn[j];
      put(a.n, v);
      if (t == 0) a.inv_y[r] = inv_y;
    }
    buf ^= 2;
    if (++stage == a.stages) {
      stage = 0;
      parity ^= 1u;
    }
  }
  if (stop != row_stop::NEVER && t == 0) {
    // a copy did not arrive in time: report it, and leave no copy in flight behind
    atomicExch(&g_norm_error, NVFP4B200_ERR_TIMEOUT);
    for (int st = 0; st < a.stages; ++st) bulk::wait(&full[st], parity ^ (st < stage ? 1u : 0u));
  }
}

struct BwdArgs {
  const void *dy, *dn, *b, *y, *gamma_post, *gate, *gamma_pre;
  const float *inv_b, *inv_y;
  void *dx, *db;
  float* part;              // [2][ctas][d]: gate-weighted S (dgamma_post), dgamma_pre
  float* part_gate;         // [G * parts][d]: S of a part of a group's rows (parts > 1)
  float* dgate;             // [G][d], written here when a CTA holds whole groups; or null
  int64_t rows, ldb, ld_dy, ld_dn, ldy, rows_per_gate, rows_per_cta;
  int d;
  float alpha, s;
  int stages;               // staged kernel: rows of the ring
  int64_t safe_rows;        // staged kernel, unaligned rows: those whose 16-byte windows lie inside every tensor
  int ws16;                 // part and part_gate are 16-byte aligned
};

// A CTA walks rows_per_cta consecutive rows, one at a time.  rows_per_cta
// divides rows_per_gate or is a multiple of it, so a CTA's rows lie in one
// group or are whole groups.  (Groups of rows that end early are handled by
// the host: parts of a group are cut at its end.)
// For tensors that start off a 16-byte boundary: single elements, straight from global memory.
template <int DT, int TPR, int V>
__global__ void __launch_bounds__(TPR) sandwich_bwd_kernel(const BwdArgs a, int64_t parts_per_group) {
  using Raw = typename Elem<DT>::Raw;
  constexpr int C = 8 * V;   // columns per thread
  __shared__ float red[4][TPR / 32];
  const int t = threadIdx.x;
  const float inv_d = 1.0f / (float)a.d;
  // the CTA's rows: part p of group g, or a run of whole groups
  int64_t r, end;
  if (parts_per_group > 1) {
    const int64_t g = blockIdx.x / parts_per_group, p = blockIdx.x % parts_per_group;
    r = g * a.rows_per_gate + p * a.rows_per_cta;
    end = imin64(r + a.rows_per_cta, (g + 1) * a.rows_per_gate);
  } else {
    r = (int64_t)blockIdx.x * a.rows_per_cta;
    end = imin64(r + a.rows_per_cta, a.rows);
  }
  float S[C], post[C], pre[C];
#pragma unroll
  for (int j = 0; j < C; ++j) S[j] = post[j] = pre[j] = 0.0f;
  int buf = 0;
  for (; r < end; ++r) {
    Row<DT, false, TPR, V> row, rb, rw;
    float tt[C], z[C], w[C], v[C];
    if (a.dy) row.load(static_cast<const Raw*>(a.dy) + r * a.ld_dy, t, a.d);
    rb.load(static_cast<const Raw*>(a.b) + r * a.ldb, t, a.d);
    if (a.dy) {
      row.values(tt);
    } else {
#pragma unroll
      for (int j = 0; j < C; ++j) tt[j] = 0.0f;
    }
    if (a.dn) {
      Row<DT, false, TPR, V> rn, ry;
      rn.load(static_cast<const Raw*>(a.dn) + r * a.ld_dn, t, a.d);
      ry.load(static_cast<const Raw*>(a.y) + r * a.ldy, t, a.d);
      rn.values(v);
      ry.values(z);
      const float inv = __ldg(a.inv_y + r);
#pragma unroll
      for (int j = 0; j < C; ++j) {
        z[j] *= inv;
        pre[j] = fmaf(v[j], z[j], pre[j]);
      }
      if (a.gamma_pre) {
        rw.load(static_cast<const Raw*>(a.gamma_pre), t, a.d);
        rw.values(w);
#pragma unroll
        for (int j = 0; j < C; ++j) v[j] *= w[j];
      }
      float dot = 0.0f;
#pragma unroll
      for (int j = 0; j < C; ++j) dot = fmaf(v[j], z[j], dot);
      const float mean = row_sum<TPR>(dot, red[buf], 0) * inv_d;
#pragma unroll
      for (int j = 0; j < C; ++j) tt[j] = fmaf(inv, fmaf(-mean, z[j], v[j]), tt[j]);
    }
    const float inv = __ldg(a.inv_b + r);
    rb.values(z);
#pragma unroll
    for (int j = 0; j < C; ++j) {
      z[j] *= inv;
      v[j] = a.s * tt[j];
      S[j] = fmaf(v[j], z[j], S[j]);
    }
    if (a.gamma_post) {
      rw.load(static_cast<const Raw*>(a.gamma_post), t, a.d);
      rw.values(w);
#pragma unroll
      for (int j = 0; j < C; ++j) v[j] *= w[j];
    }
    if (a.gate) {
      rw.load(static_cast<const Raw*>(a.gate) + (r / a.rows_per_gate) * a.d, t, a.d);
      rw.values(w);
#pragma unroll
      for (int j = 0; j < C; ++j) v[j] *= w[j];
    }
    float dot = 0.0f;
#pragma unroll
    for (int j = 0; j < C; ++j) dot = fmaf(v[j], z[j], dot);
    const float mean = row_sum<TPR>(dot, red[buf + 1], 0) * inv_d;
#pragma unroll
    for (int j = 0; j < C; ++j) z[j] = inv * fmaf(-mean, z[j], v[j]);
    store_row<DT, false, TPR, V>(static_cast<Raw*>(a.db) + r * a.d, t, a.d, z);
#pragma unroll
    for (int j = 0; j < C; ++j) tt[j] *= a.alpha;
    store_row<DT, false, TPR, V>(static_cast<Raw*>(a.dx) + r * a.d, t, a.d, tt);
    buf ^= 2;
    // the last row of a group (or of this CTA's part of it): hand S over
    if (a.gate && (r + 1 == end || (r + 1) % a.rows_per_gate == 0)) {
      const int64_t g = r / a.rows_per_gate;
      rw.load(static_cast<const Raw*>(a.gate) + g * a.d, t, a.d);
      rw.values(w);
#pragma unroll
      for (int j = 0; j < C; ++j) post[j] = fmaf(w[j], S[j], post[j]);
      float* out = parts_per_group > 1 ? a.part_gate + (int64_t)blockIdx.x * a.d : a.dgate ? a.dgate + g * a.d : nullptr;
      if (parts_per_group == 1 && a.gamma_post) {
        rw.load(static_cast<const Raw*>(a.gamma_post), t, a.d);
        rw.values(w);
#pragma unroll
        for (int j = 0; j < C; ++j) S[j] *= w[j];
      }
#pragma unroll
      for (int j = 0; j < C; ++j) {
        const int c = column<false, TPR>(t, j);
        if (out && c < a.d) out[c] = S[j];
        S[j] = 0.0f;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < C; ++j) {
    const int c = column<false, TPR>(t, j);
    if (c < a.d) {
      a.part[(int64_t)blockIdx.x * a.d + c] = a.gate ? post[j] : S[j];
      a.part[((int64_t)gridDim.x + blockIdx.x) * a.d + c] = pre[j];
    }
  }
}

// The same backward with the rows staged ahead in shared memory: one thread
// copies whole rows of dy, dn, b and y into a ring of STAGES rows (bulk
// copies on one barrier per row) and refills a row's place right after the
// barrier of the row's reduction, by when every thread has read it.  The
// row's two means come from that one exchange of three sums: with
// W = s * gate * gamma_post and t0 = dy + inv_y * v,
//     A = sum v yh,  B = sum W bh t0,  C = sum W bh yh
//     m1 = A / d,    m2 = (B - inv_y * m1 * C) / d
//     t = t0 - inv_y * m1 * yh,    db = inv_b * (W t - m2 bh).
// Arithmetic is on packed pairs of floats.  A CTA's rows lie in one group (W
// stays in registers) but in the MULTI form, so dgamma_post's part is gate * S
// at the end.  The column sums S leave out s; it is multiplied in at the end.
// The column sums live in shared memory, each thread's own words, so that a
// thread fits 64 registers and 32 warps share an SM: with the sums in registers
// 16 warps did, and waited for one another's barriers (147 us against 134 at 16000 x 4096).

constexpr int BWD_STAGES = 3;   // rows of the ring, at most
constexpr long long SETTLE_CYCLES = 1000000;   // about 0.5 ms: far longer than a store between two CTAs takes

// Eight elements per thread: TPR threads cover d <= 8 * TPR columns.  In fp32
// they are two pieces of four, a half of the row apart, so that neighbouring
// lanes' 16 bytes are neighbours (8192 x 4096: 186 us with the pieces side by side, 170
// so; 4096 x 8192 190 and 144).
// ODD: rows that do not start on 16-byte boundaries (widths that are no
// multiple of 8, say).  The bulk copies take each row's window of whole
// 16-byte pieces, a thread's eight columns are TPR apart and are read and
// written one by one; the last rows, whose windows could reach past the tensor,
// are read straight from global memory.
// MULTI: a CTA's rows are whole groups (few rows each, one at the least: a gate
// per token).  W is set up anew at a group's start, the next group's gate having
// been brought to L2, and S is handed over at its end; the sum of gate * S is
// kept beside the other column sums.  (With gate, gamma_post and that sum in
// registers 16 warps share an SM: 316 us at 16000 x 4096 with a gate per row, 246 so.)
// SPLIT: rows of more than 8192 columns, which no SM's shared memory holds
// together with their column sums.  The two CTAs of a cluster take half the
// columns each; every warp sends its parts of the row's sums to the other CTA,
// on a barrier that counts their bytes.  (With the cluster's own barrier in
// every row 250 us at 4096 x 16384 bf16 with the next
// norm, 229 so; 1016 with rows read straight from global memory.)
template <int DT, int TPR, bool PRE, bool ODD, bool MULTI, bool SPLIT>
__global__ void __launch_bounds__(TPR, DT == NVFP4B200_F32 && TPR >= 512 ? 1 : 1024 / TPR)
    sandwich_bwd_staged_kernel(const BwdArgs a, int64_t parts_per_group) {
  using E = Elem<DT>;
  using Raw = typename E::Raw;
  constexpr int NT = PRE ? 4 : 2;                 // tensors: dy, b [, dn, y]
  constexpr int NP = 4;                           // packed pairs per thread
  const int ST = a.stages;
  constexpr int W4 = (TPR / 32 + 3) / 4 * (SPLIT ? 2 : 1);   // 16-byte words of one sum's warp parts
  extern __shared__ __align__(16) uint8_t row_ring[];   // [ST][NT][d], then the column sums
  __shared__ __align__(16) float red[2][3][4 * W4];
  __shared__ __align__(8) uint64_t full[BWD_STAGES], theirs[SPLIT ? 2 : 1];
  __shared__ int stop;   // row_stop.h: set where a wait ran out
  const int t = threadIdx.x;
  const float inv_d = 1.0f / (float)a.d;
  // this CTA's columns: [c0, c0 + d) of the row
  const int rank = SPLIT ? (int)blockIdx.x & 1 : 0, half = SPLIT ? ((a.d + 1) / 2 + 7) & ~7 : a.d;
  const int c0 = rank * half, d = SPLIT ? min(half, a.d - c0) : a.d;
  const int64_t unit = SPLIT ? blockIdx.x >> 1 : blockIdx.x, units = SPLIT ? gridDim.x >> 1 : gridDim.x;
  auto pair_barrier = []() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  };
  const int row_bytes = d * (int)sizeof(Raw);
  const int slot = ODD ? ((row_bytes + 15) & ~15) + 16 : row_bytes;   // of one tensor's row in the ring
  const int64_t g = unit / parts_per_group, p = unit % parts_per_group;
  const int64_t r0 = MULTI ? unit * a.rows_per_cta : g * a.rows_per_gate + p * a.rows_per_cta;
  const int rows = (int)(imin64(r0 + a.rows_per_cta, MULTI ? a.rows : (g + 1) * a.rows_per_gate) - r0);

  const int staged = (int)imin64(rows, ODD ? (a.safe_rows > r0 ? a.safe_rows - r0 : 0) : rows);
  auto skew = [&](int64_t r, int64_t ld) { return ODD ? (int)((uint64_t)(r * ld) * sizeof(Raw) & 15) : 0; };

  auto fetch = [&](int i, int stage) {   // one thread: row r0 + i into a stage
    if (i >= staged) return;
    uint8_t* dst = row_ring + (size_t)stage * NT * slot;
    const int64_t r = r0 + i;
    const void* base[4] = {a.dy, a.b, a.dn, a.y};
    const int64_t ld[4] = {a.ld_dy, a.ldb, a.ld_dn, a.ldy};
    uint32_t total = 0;
#pragma unroll
    for (int q = 0; q < NT; ++q)
      if (base[q]) total += (uint32_t)(ODD ? (skew(r, ld[q]) + row_bytes + 15) & ~15 : row_bytes);
    bulk::expect(&full[stage], total);
#pragma unroll
    for (int q = 0; q < NT; ++q)
      if (base[q]) {
        const int off = skew(r, ld[q]);
        bulk::copy(dst + q * slot, static_cast<const uint8_t*>(base[q]) + (r * ld[q] + c0) * (int64_t)sizeof(Raw) - off,
                   (uint32_t)(ODD ? (off + row_bytes + 15) & ~15 : row_bytes), &full[stage]);
      }
  };
  if (t < 3 * 4 * W4 * 2) (&red[0][0][0])[t] = 0.0f;   // warp parts past the last stay zero
  if (t == 0) {
    stop = row_stop::NEVER;
    bulk::init(full, ST);
    if (SPLIT) bulk::init(theirs, 2);
  }
  if (SPLIT) pair_barrier();
  else __syncthreads();
  if (t == 0)
    for (int st = 0; st < ST; ++st) fetch(st, st);

  // column sums, each thread's own: S (2 float4), dgamma_pre's (2 more), gate * S over the groups (2 more)
  ulonglong2* sums_at = reinterpret_cast<ulonglong2*>(row_ring + (size_t)ST * NT * slot) + t;
#pragma unroll
  for (int j = 0; j < NT + (MULTI ? 2 : 0); ++j) sums_at[j * TPR] = make_ulonglong2(0ull, 0ull);
  // the thread's first column; the others follow, or are TPR apart (ODD), or half h of them starts at col(h)
  constexpr bool WIDE = !ODD && DT == NVFP4B200_F32;
  const int c = ODD ? t : WIDE ? 4 * t : 8 * t;
  const bool in = c < d;
  auto col = [&](int h) { return WIDE ? 4 * (h * TPR + t) : c + 4 * h; };
  auto weights = [&](const void* p, int64_t off, uint64_t (&w)[NP]) {
    float f[8];
    if (ODD) {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = c + j * TPR < d ? E::get(static_cast<const Raw*>(p) + off + c0 + c + j * TPR) : 0.0f;
    } else if constexpr (WIDE) {
      auto v = E::zero();
      if (col(0) < d) v.a = __ldg(reinterpret_cast<const float4*>(static_cast<const Raw*>(p) + off + c0 + col(0)));
      if (col(1) < d) v.b = __ldg(reinterpret_cast<const float4*>(static_cast<const Raw*>(p) + off + c0 + col(1)));
      E::unpack(v, f);
    } else {
      E::unpack(in ? E::load(static_cast<const Raw*>(p) + off + c0 + c) : E::zero(), f);
    }
#pragma unroll
    for (int j = 0; j < NP; ++j) w[j] = f2mul(w[j], f2pack(f[2 * j], f[2 * j + 1]));
  };
  uint64_t W[NP], gpre[PRE ? NP : 1];
#pragma unroll
  for (int j = 0; j < NP; ++j) W[j] = f2two(a.s);
  if (a.gamma_post) weights(a.gamma_post, 0, W);
  if (!MULTI && a.gate) weights(a.gate, g * a.d, W);
  int64_t group = MULTI ? r0 / a.rows_per_gate - 1 : 0, left = 0;
  if constexpr (PRE) {
#pragma unroll
    for (int j = 0; j < NP; ++j) gpre[j] = f2two(1.0f);
    if (a.gamma_pre) weights(a.gamma_pre, 0, gpre);
  }

  auto put = [&](float* row, bool wide, int h, uint64_t lo, uint64_t hi) {   // the thread's columns 4 h .. 4 h + 3
    if (ODD) {
      const float f[4] = {f2lo(lo), f2hi(lo), f2lo(hi), f2hi(hi)};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + (4 * h + j) * TPR < d) row[c0 + c + (4 * h + j) * TPR] = f[j];
      return;
    }
    if (WIDE && col(h) >= d) return;
    float* out = row + c0 + col(h);   // d % 8 == 0: 16-byte aligned where the first row is
    if (wide) {
      *reinterpret_cast<ulonglong2*>(out) = make_ulonglong2(lo, hi);
    } else {
      out[0] = f2lo(lo); out[1] = f2hi(lo); out[2] = f2lo(hi); out[3] = f2hi(hi);
    }
  };
  const bool aligned_dgate = MULTI && (reinterpret_cast<uintptr_t>(a.dgate) & 15) == 0;

  Raw *dx = static_cast<Raw*>(a.dx) + r0 * a.d + c0, *db = static_cast<Raw*>(a.db) + r0 * a.d + c0;
  const float *ib = a.inv_b + r0, *iy = PRE ? a.inv_y + r0 : nullptr;
  float next_b = __ldg(ib), next_y = PRE ? __ldg(iy) : 0.0f;
  int stage = 0, buf = 0;
  uint32_t parity = 0;
  for (int i = 0; i < rows; ++i) {
    const float inv_b = next_b, inv_y = next_y;
    if (i + 1 < rows) {   // a row ahead, so that its latency is not exposed once per row
      next_b = __ldg(ib + i + 1);
      if (PRE) next_y = __ldg(iy + i + 1);
    }
    if constexpr (MULTI) {
      if (left == 0) {   // a group begins
        left = a.rows_per_gate;
        ++group;
#pragma unroll
        for (int j = 0; j < NP; ++j) W[j] = f2two(a.s);
        if (a.gamma_post) weights(a.gamma_post, 0, W);
        weights(a.gate, group * a.d, W);
        if (i + left < rows && in && t % (128 / (ODD ? (int)sizeof(Raw) : 16)) == 0)
          for (int j = 0; j < (ODD ? 8 : WIDE ? 2 : 1); ++j)
            if (ODD ? c + j * TPR < d : col(j) < d)
              asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const Raw*>(a.gate) + (group + 1) * a.d + c0 + (ODD ? c + j * TPR : col(j))));
      }
      --left;
    }
    if (i < staged && !bulk::wait(&full[stage], parity)) atomicMin(&stop, row_stop::before_barrier(i));
    const uint8_t* src = row_ring + (size_t)stage * NT * slot;
    auto get = [&](int tensor, int c, uint64_t (&o)[4]) {
      if (!ODD) {
        const uint4* at = reinterpret_cast<const uint4*>(src + tensor * slot + c * (int)sizeof(Raw));
        Pairs<DT>::get(at, !WIDE || col(1) < d ? (WIDE ? TPR : 1) : 0, o);
        if (WIDE && col(1) >= d) o[2] = o[3] = 0ull;
        return;
      }
      const void* base = tensor == 0 ? a.dy : tensor == 1 ? a.b : tensor == 2 ? a.dn : a.y;
      const int64_t at = (r0 + i) * (tensor == 0 ? a.ld_dy : tensor == 1 ? a.ldb : tensor == 2 ? a.ld_dn : a.ldy);
      const Raw* row = i < staged ? reinterpret_cast<const Raw*>(src + tensor * slot + (int)((uint64_t)at * sizeof(Raw) & 15))
                                  : static_cast<const Raw*>(base) + at + c0;
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = c + j * TPR < d ? E::value(row[c + j * TPR]) : 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = f2pack(f[2 * j], f[2 * j + 1]);
    };
    uint64_t t0[NP], yh[PRE ? NP : 1], bh[NP];
    uint64_t A = 0ull, B = 0ull, C = 0ull;
    {
      uint64_t z[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
      for (int j = 0; j < NP; ++j) t0[j] = 0ull;
      if (in) {
        if (a.dy) get(0, c, t0);
        get(1, c, z);
      }
#pragma unroll
      for (int j = 0; j < NP; ++j) bh[j] = f2mul(z[j], f2two(inv_b));
      if constexpr (PRE) {
        uint64_t x[4] = {0ull, 0ull, 0ull, 0ull};
        if (in) {
          get(2, c, x);
          get(3, c, z);
        }
        const ulonglong2 p0 = sums_at[2 * TPR], p1 = sums_at[3 * TPR];
        uint64_t pre[NP] = {p0.x, p0.y, p1.x, p1.y};
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          yh[j] = f2mul(z[j], f2two(inv_y));
          pre[j] = f2fma(x[j], yh[j], pre[j]);
          const uint64_t v = f2mul(x[j], gpre[j]);
          A = f2fma(v, yh[j], A);
          t0[j] = f2fma(v, f2two(inv_y), t0[j]);
        }
        sums_at[2 * TPR] = make_ulonglong2(pre[0], pre[1]);
        sums_at[3 * TPR] = make_ulonglong2(pre[2], pre[3]);
      }
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const uint64_t wb = f2mul(W[j], bh[j]);
        B = f2fma(wb, t0[j], B);
        if (PRE) C = f2fma(wb, yh[j], C);
      }
    }
    float sums[3] = {f2sum(B), PRE ? f2sum(A) : 0.0f, PRE ? f2sum(C) : 0.0f};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int k = 0; k < (PRE ? 3 : 1); ++k) sums[k] += __shfl_xor_sync(0xffffffffu, sums[k], o);
    if (SPLIT) {   // three lanes, a sum each
      if ((t & 31) < (PRE ? 3 : 1)) {
        const int k = t & 31;
        const float v = k == 0 ? sums[0] : k == 1 ? sums[1] : sums[2];
        float* at = &red[buf][k][rank * (TPR / 32) + (t >> 5)];
        *at = v;
        asm volatile(
            "{\n\t.reg .b32 a, b;\n\tmapa.shared::cluster.u32 a, %0, %2;\n\tmapa.shared::cluster.u32 b, %1, %2;\n\t"
            "st.async.shared::cluster.mbarrier::complete_tx::bytes.b32 [a], %3, [b];\n\t}" ::"r"(bulk::addr(at)),
            "r"(bulk::addr(&theirs[buf])), "r"(rank ^ 1), "r"(__float_as_uint(v))
            : "memory");
      }
      if (t == 0) bulk::expect(&theirs[buf], (PRE ? 3 : 1) * (TPR / 32) * 4);
    } else if ((t & 31) == 0) {
#pragma unroll
      for (int k = 0; k < (PRE ? 3 : 1); ++k) red[buf][k][t >> 5] = sums[k];
    }
    __syncthreads();
    if (row_stop::leaves(stop, i)) break;   // the same in every thread
    if (SPLIT && !bulk::wait<true>(&theirs[buf], (uint32_t)(i >> 1) & 1u)) atomicMin(&stop, row_stop::after_barrier(i));
    // refilled only where the row's own copies arrived: a barrier whose phase is open takes no second one
    if (t == 0) fetch(i + ST, stage);
    if (TPR > 32) {
#pragma unroll
      for (int k = 0; k < (PRE ? 3 : 1); ++k) {
        float u = 0.0f;
#pragma unroll
        for (int w = 0; w < W4; ++w) {
          const float4 q = reinterpret_cast<const float4*>(red[buf][k])[w];
          u += (q.x + q.y) + (q.z + q.w);
        }
        sums[k] = u;
      }
    }
    buf ^= 1;
    const float m1 = PRE ? sums[1] * inv_d : 0.0f;
    const float m2 = (PRE ? fmaf(-inv_y * m1, sums[2], sums[0]) : sums[0]) * inv_d;
    const ulonglong2 s0 = sums_at[0], s1 = sums_at[TPR];
    uint64_t S[NP] = {s0.x, s0.y, s1.x, s1.y};
    float dxv[8], dbv[8];
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const uint64_t tt = PRE ? f2fma(yh[j], f2two(-inv_y * m1), t0[j]) : t0[j];
      S[j] = f2fma(tt, bh[j], S[j]);
      const uint64_t e_b = f2mul(f2fma(bh[j], f2two(-m2), f2mul(W[j], tt)), f2two(inv_b));
      const uint64_t e = f2mul(tt, f2two(a.alpha));
      dxv[2 * j] = f2lo(e); dxv[2 * j + 1] = f2hi(e);
      dbv[2 * j] = f2lo(e_b); dbv[2 * j + 1] = f2hi(e_b);
    }
    if constexpr (MULTI) {
      if (left == 0) {   // and ends
        const uint64_t one = f2two(1.0f);
        uint64_t dg[NP], gs[NP];
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          dg[j] = gs[j] = f2mul(S[j], f2two(a.s));
          S[j] = 0ull;
        }
        weights(a.gate, group * a.d, gs);
        if (a.gamma_post) weights(a.gamma_post, 0, dg);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const ulonglong2 v = sums_at[(NT + h) * TPR];
          sums_at[(NT + h) * TPR] = make_ulonglong2(f2fma(gs[2 * h], one, v.x), f2fma(gs[2 * h + 1], one, v.y));
        }
        if (a.dgate && in) {
          float* out = a.dgate + group * a.d;
          put(out, aligned_dgate, 0, dg[0], dg[1]);
          put(out, aligned_dgate, 1, dg[2], dg[3]);
        }
      }
    }
    sums_at[0] = make_ulonglong2(S[0], S[1]);
    sums_at[TPR] = make_ulonglong2(S[2], S[3]);
    if (ODD) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j * TPR < d) {
          dx[c + j * TPR] = E::bits(dxv[j]);
          db[c + j * TPR] = E::bits(dbv[j]);
        }
    } else if constexpr (WIDE) {
      const auto px = E::pack(dxv), pb = E::pack(dbv);
      if (col(0) < d) {
        *reinterpret_cast<float4*>(dx + col(0)) = px.a;
        *reinterpret_cast<float4*>(db + col(0)) = pb.a;
      }
      if (col(1) < d) {
        *reinterpret_cast<float4*>(dx + col(1)) = px.b;
        *reinterpret_cast<float4*>(db + col(1)) = pb.b;
      }
    } else if (in) {
      E::store(dx + c, E::pack(dxv));
      E::store(db + c, E::pack(dbv));
    }
    dx += a.d;
    db += a.d;
    if (++stage == ST) {
      stage = 0;
      parity ^= 1u;
    }
  }
  if (SPLIT) pair_barrier();   // no CTA leaves while the other may still send to it
  if (stop != row_stop::NEVER && t == 0) {
    // a copy, or the other CTA's sums, did not arrive in time: report it, and leave
    // nothing in flight behind.  Nothing tells when the other CTA's last sums have landed.
    atomicExch(&g_norm_error, NVFP4B200_ERR_TIMEOUT);
    for (int st = 0; st < ST; ++st) bulk::wait(&full[st], parity ^ (st < stage ? 1u : 0u));
    if (SPLIT)
      for (const long long t0 = clock64(); clock64() - t0 < SETTLE_CYCLES;) {
      }
  }

  // partial column sums: s * S, gate * s * S and dgamma_pre
  if (!in) return;
  uint64_t gate[NP];
#pragma unroll
  for (int j = 0; j < NP; ++j) gate[j] = f2two(1.0f);
  if (!MULTI && a.gate) weights(a.gate, g * a.d, gate);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if constexpr (MULTI) {
      const ulonglong2 v = sums_at[(NT + h) * TPR];
      put(a.part + unit * a.d, a.ws16, h, v.x, v.y);
    } else {
      const ulonglong2 sv = sums_at[h * TPR];
      const uint64_t lo = f2mul(sv.x, f2two(a.s)), hi = f2mul(sv.y, f2two(a.s));
      if (a.gate) put(a.part_gate + unit * a.d, a.ws16, h, lo, hi);
      put(a.part + unit * a.d, a.ws16, h, f2mul(lo, gate[2 * h]), f2mul(hi, gate[2 * h + 1]));
    }
    if (PRE) {
      const ulonglong2 pv = sums_at[(2 + h) * TPR];
      put(a.part + (units + unit) * a.d, a.ws16, h, pv.x, pv.y);
    }
  }
}

// Column sums of the partials, in CTA order.  Job 0 is dgamma_post, 1
// dgamma_pre, 2 + g dgate of group g.  A CTA takes 32 * V columns of a job;
// its 16 warps share the partials, each a contiguous run of them, and the
// runs' sums are added in order.  V = 4 where rows of partials are 16-byte
// aligned: wide loads and a quarter of the CTAs.
struct FinishArgs {
  const float *part, *part_gate;
  const void* gamma_post;
  float *dgamma_post, *dgamma_pre, *dgate;
  int64_t ctas, parts_per_group;
  int d;
};
constexpr int FINISH_WARPS = 16;

template <int DT, int V>
__global__ void __launch_bounds__(32 * FINISH_WARPS) sandwich_bwd_finish_kernel(const FinishArgs a) {
  __shared__ float red[FINISH_WARPS][32 * V];
  const int lane = threadIdx.x & 31, seg = threadIdx.x >> 5;
  const int blocks = (a.d + 32 * V - 1) / (32 * V);
  const int c0 = (int)(blockIdx.x % blocks) * 32 * V, c = c0 + lane * V;
  const int64_t job = blockIdx.x / blocks;
  const float* p;
  float* out;
  int64_t n;
  if (job == 0) { p = a.part; out = a.dgamma_post; n = a.ctas; }
  else if (job == 1) { p = a.part + a.ctas * a.d; out = a.dgamma_pre; n = a.ctas; }
  else { p = a.part_gate + (job - 2) * a.parts_per_group * a.d; out = a.dgate + (job - 2) * a.d; n = a.parts_per_group; }
  if ((job == 0 && !a.dgamma_post) || (job == 1 && !a.dgamma_pre)) return;
  const int64_t per = (n + FINISH_WARPS - 1) / FINISH_WARPS, lo = per * seg, hi = imin64(n, lo + per);
  float s[V];
#pragma unroll
  for (int j = 0; j < V; ++j) s[j] = 0.0f;
  if (c < a.d) {   // V = 4: d % 4 == 0
#pragma unroll 8
    for (int64_t i = lo; i < hi; ++i) {
      if (V == 4) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(p + i * a.d + c));
        s[0] += v.x; s[V > 1 ? 1 : 0] += v.y; s[V > 2 ? 2 : 0] += v.z; s[V > 3 ? 3 : 0] += v.w;
      } else {
        s[0] += __ldg(p + i * a.d + c);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) red[seg][lane * V + j] = s[j];
  __syncthreads();
  for (int k = threadIdx.x; k < 32 * V && c0 + k < a.d; k += 32 * FINISH_WARPS) {
    float u = red[0][k];
#pragma unroll
    for (int i = 1; i < FINISH_WARPS; ++i) u += red[i][k];
    if (job >= 2 && a.gamma_post) u *= Elem<DT>::get(static_cast<const typename Elem<DT>::Raw*>(a.gamma_post) + c0 + k);
    out[c0 + k] = u;
  }
}

// Threads per row, 16 columns each: the least of a few numbers of warps.  (With
// powers of two alone 13107 x 5120 bf16 took 119 us in the forward and 240 in the
// backward, 88 and 163 so; 43690 x 1536 129 and 166, 92 and 155; 26214 x 2560 125 and 198,
// 122 and 154.)
constexpr int WIDTHS[] = {32, 64, 96, 128, 160, 256, 320, 384, 512, 1024};

template <int I = 0, typename F>
static int by_width(int d, F f) {
  if constexpr (I + 1 < (int)(sizeof(WIDTHS) / sizeof(int))) {
    if (d > WIDTHS[I] * CPT) return by_width<I + 1>(d, f);
  }
  return f(std::integral_constant<int, WIDTHS[I]>());
}

template <typename F>
static int by_type(int dt, bool vec, F f) {
#define NORM_DT(D)                                                                         \
  return vec ? f(std::integral_constant<int, D>(), std::true_type())                       \
             : f(std::integral_constant<int, D>(), std::false_type())
  if (dt == NVFP4B200_BF16) { NORM_DT(NVFP4B200_BF16); }
  if (dt == NVFP4B200_F16) { NORM_DT(NVFP4B200_F16); }
  NORM_DT(NVFP4B200_F32);
#undef NORM_DT
}

// How the backward splits its rows over CTAs.  A function of the sizes alone.
struct Split {
  int64_t rows_per_cta, parts_per_group, ctas;
};

constexpr int START_ROWS = 4;

static Split split_rows(int64_t rows, int64_t groups, int64_t d, int sms) {
  // CTAs that run at a time: 1024 threads per SM, 8 columns each; narrow rows in
  // more, smaller CTAs
  int64_t tpr = 0;
  by_width((int)d, [&](auto t) { tpr = t; return 0; });
  // rows of more than 8192 columns take two SMs
  const int64_t per = rows / groups, target = tpr > 512 ? std::max(1, sms / 2) : 1024 / (2 * tpr) * sms;
  // A CTA takes a part of a group's rows, or whole groups.  The cost is counted in
  // rows: waves of CTAs times the rows of one and some more for its start.  (As many
  // whole groups, or parts of one, as fill one wave: 16000 x 4096 with 160 gates 242
  // us against 170 so, 100 gates 195 / 167, 320 gates 244 / 185.)
  Split s{0, 1, 0};
  int64_t best = INT64_MAX;
  for (int64_t waves = 1; waves <= 4; ++waves) {
    const int64_t fit = waves * target / groups;      // parts of a group
    const int64_t whole = ceil_div(groups, waves * target);
    for (const int64_t rows_per : {fit > 1 && per > 1 ? ceil_div(per, fit) : int64_t(0), whole * per}) {
      if (rows_per == 0) continue;
      const int64_t parts = rows_per < per ? ceil_div(per, rows_per) : 1;
      const int64_t ctas = rows_per < per ? groups * parts : ceil_div(groups, rows_per / per);
      const int64_t cost = ceil_div(ctas, target) * (rows_per + START_ROWS);
      if (cost < best) {
        best = cost;
        s = {rows_per, parts, ctas};
      }
    }
  }
  return s;
}

}  // namespace norm

int take_norm_device_error() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, norm::g_norm_error, sizeof(int)) != cudaSuccess) return NVFP4B200_ERR_CUDA;
  if (v && cudaMemcpyToSymbol(norm::g_norm_error, &zero, sizeof(int)) != cudaSuccess) return NVFP4B200_ERR_CUDA;
  return v;
}

}  // namespace nvfp4b200

using namespace nvfp4b200;

static bool vec_ok(const void* p, int64_t ld, int bytes) { return !p || (aligned(p, 16) && (ld * bytes) % 16 == 0); }

extern "C" {

int nvfp4b200_sandwich_norm(const void* b, const void* x, const void* gamma_post, const void* gate,
                            const void* gamma_pre, void* y, void* n, float* inv_b, float* inv_y, int dtype,
                            int64_t rows, int64_t d, int64_t groups, int64_t ldb, int64_t ldx, float residual_scale,
                            float branch_scale, float eps, void* stream) {
  if (!b || !x || !y || !inv_b || (n == nullptr) != (inv_y == nullptr) || (gamma_pre && !n) || !valid_dtype(dtype))
    return NVFP4B200_ERR_INVALID_ARG;
  if (rows < 0 || d <= 0 || d > norm::MAX_D || ldb < d || ldx < d || groups < 0 || (gate == nullptr) != (groups == 0) ||
      (groups && rows % groups))
    return NVFP4B200_ERR_BAD_SHAPE;
  const int bytes = dtype_bytes(dtype);
  for (const void* p : {b, x, gamma_post, gate, gamma_pre, (const void*)y, (const void*)n})
    if (p && !aligned(p, bytes)) return NVFP4B200_ERR_MISALIGNED;
  if (!aligned(inv_b, 4) || (inv_y && !aligned(inv_y, 4))) return NVFP4B200_ERR_MISALIGNED;
  int rc = check_device();
  if (rc) return rc;
  if (rows == 0) return NVFP4B200_OK;
  norm::FwdArgs a{b, x, gamma_post, gate, gamma_pre, y, n, inv_b, inv_y, rows, ldb, ldx, groups ? rows / groups : rows,
                  (int)d, residual_scale, branch_scale, eps, n != nullptr, 0, 0, 0};
  const bool vec = (d * bytes) % 16 == 0 && d % 8 == 0 && vec_ok(b, ldb, bytes) && vec_ok(x, ldx, bytes) &&
                   vec_ok(gamma_post, d, bytes) && vec_ok(gate, d, bytes) && vec_ok(gamma_pre, d, bytes) &&
                   vec_ok(y, d, bytes) && vec_ok(n, d, bytes);
  cudaStream_t st = (cudaStream_t)stream;
  return norm::by_type(dtype, vec, [&](auto dt, auto v) {
    return norm::by_width((int)d, [&](auto tpr) {
      constexpr int T = decltype(tpr)::value, THREADS = norm::threads_of(T), GROUPS = THREADS / T;
      constexpr int DT = decltype(dt)::value;
      constexpr bool VEC = decltype(v)::value;
      // the staged kernel where its ring fits (all but fp32 rows of more than 8192 columns): 195 us without,
      // 168 to 187 by the GPU with it, at 16384 x 8192 bf16 with the next norm.  fp32: 8 columns a thread,
      // so that 32 warps share an SM (8192 x 4096: 88 us, 141 with 16 columns; bf16 at 16384 x 4096 93 with
      // 16 columns, 109 with 8)
      constexpr int V = DT == NVFP4B200_F32 && T <= 512 ? 1 : norm::VPT, TV = T * norm::VPT / V;
      constexpr int THREADS_V = norm::threads_of(TV);
      constexpr int smem = norm::STAGES * 2 * THREADS_V * 8 * V * norm::dtype_size<DT>();
      if constexpr (VEC && smem <= norm::MAX_SMEM) {
        auto* fn = norm::sandwich_fwd_staged_kernel<DT, TV, V>;
        if (smem > 32 * 1024 && !allow_smem(fn, norm::MAX_SMEM))   // with the static arrays, past the default limit
          return (int)NVFP4B200_ERR_CUDA;
        const int per_sm = std::max(1, std::min(228 * 1024 / (smem + 2048), 1024 / THREADS_V));
        fn<<<(unsigned)std::min<int64_t>(ceil_div(rows, THREADS_V / TV), (int64_t)sm_count_current() * per_sm), THREADS_V, smem, st>>>(a);
        return launch_status();
      } else {
        if constexpr (!VEC && T >= 64 && T <= 512) {
          // unaligned rows of more than 512 columns, 8 columns a thread: 114 -> 82 us at 8000 x
          // 4095 bf16 with the next norm (20000 x 301: 24 us without, 28 with)
          constexpr int T2 = 2 * T;
          const int row = 2 * ((int)round_up(d * bytes, 16) + 16), share = norm::smem_share(1024 / T2);
          if (aligned(b, 16) && aligned(x, 16) && row <= share) {
            a.stages = std::min(norm::STAGES, share / row);
            a.safe_rows = std::max<int64_t>(0, rows - 1 - 15 / (std::min(ldb, ldx) * bytes));
            auto* odd = norm::sandwich_fwd_odd_kernel<DT, T2>;
            const int size = a.stages * row;
            if (size > 32 * 1024 && !allow_smem(odd, norm::MAX_SMEM)) return (int)NVFP4B200_ERR_CUDA;
            a.rows_per_cta = ceil_div(rows, (int64_t)sm_count_current() * (1024 / T2));
            odd<<<(unsigned)ceil_div(rows, a.rows_per_cta), T2, size, st>>>(a);
            return launch_status();
          }
        }
        const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(rows, GROUPS), (int64_t)sm_count_current() * (2048 / THREADS));
        norm::sandwich_fwd_kernel<DT, VEC, T><<<grid, THREADS, 0, st>>>(a);
        return launch_status();
      }
    });
  });
}

int nvfp4b200_sandwich_norm_bwd_ws(int64_t rows, int64_t d, int64_t groups, int64_t* floats) {
  if (!floats) return NVFP4B200_ERR_INVALID_ARG;
  if (rows < 0 || d <= 0 || d > norm::MAX_D || groups < 0 || (groups && rows % groups)) return NVFP4B200_ERR_BAD_SHAPE;
  *floats = 0;
  if (rows == 0) return NVFP4B200_OK;
  const norm::Split s = norm::split_rows(rows, groups ? groups : 1, d, sm_count_current());
  *floats = (2 * s.ctas + (groups && s.parts_per_group > 1 ? s.ctas : 0)) * d;
  return NVFP4B200_OK;
}

int nvfp4b200_sandwich_norm_bwd(const void* dy, const void* dn, const void* b, const void* y, const float* inv_b,
                                const float* inv_y, const void* gamma_post, const void* gate, const void* gamma_pre,
                                void* dx, void* db, float* dgamma_post, float* dgate, float* dgamma_pre, float* ws,
                                int64_t ws_floats, int dtype, int64_t rows, int64_t d, int64_t groups, int64_t ld_dy,
                                int64_t ld_dn, int64_t ldb, int64_t ldy, float residual_scale, float branch_scale,
                                void* stream) {
  if ((!dy && !dn) || !b || !inv_b || !dx || !db || !ws || (dn == nullptr) != (y == nullptr) ||
      (dn == nullptr) != (inv_y == nullptr) || (gamma_pre && !dn) || (dgamma_pre && !dn) || (dgate && !gate) ||
      !valid_dtype(dtype))
    return NVFP4B200_ERR_INVALID_ARG;
  if (rows < 0 || d <= 0 || d > norm::MAX_D || (dy && ld_dy < d) || ldb < d || (dn && (ld_dn < d || ldy < d)) || groups < 0 ||
      (gate == nullptr) != (groups == 0) || (groups && rows % groups))
    return NVFP4B200_ERR_BAD_SHAPE;
  const int bytes = dtype_bytes(dtype);
  for (const void* p : {dy, dn, b, y, gamma_post, gate, gamma_pre, (const void*)dx, (const void*)db})
    if (p && !aligned(p, bytes)) return NVFP4B200_ERR_MISALIGNED;
  for (const void* p : {(const void*)inv_b, (const void*)inv_y, (const void*)dgamma_post, (const void*)dgate,
                        (const void*)dgamma_pre, (const void*)ws})
    if (p && !aligned(p, 4)) return NVFP4B200_ERR_MISALIGNED;
  int rc = check_device();
  if (rc) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  if (rows == 0) {
    for (float* p : {dgamma_post, dgamma_pre})
      if (p && cudaMemsetAsync(p, 0, d * sizeof(float), st) != cudaSuccess) return NVFP4B200_ERR_CUDA;
    if (dgate && cudaMemsetAsync(dgate, 0, groups * d * sizeof(float), st) != cudaSuccess) return NVFP4B200_ERR_CUDA;
    return NVFP4B200_OK;
  }
  const int64_t g = groups ? groups : 1;
  const norm::Split sp = norm::split_rows(rows, g, d, sm_count_current());
  int64_t need = 0;
  nvfp4b200_sandwich_norm_bwd_ws(rows, d, groups, &need);
  if (ws_floats < need) return NVFP4B200_ERR_BAD_SHAPE;
  norm::BwdArgs a{dy, dn, b, y, gamma_post, gate, gamma_pre, inv_b, inv_y, dx, db, ws, ws + 2 * sp.ctas * d, dgate, rows, ldb,
                  ld_dy, ld_dn, ldy, rows / g, sp.rows_per_cta, (int)d, residual_scale, branch_scale, 0, 0,
                  aligned(ws, 16)};
  const bool vec = (d * bytes) % 16 == 0 && d % 8 == 0 && vec_ok(dy, ld_dy, bytes) && vec_ok(dn, ld_dn, bytes) &&
                   vec_ok(b, ldb, bytes) && vec_ok(y, ldy, bytes) && vec_ok(gamma_post, d, bytes) &&
                   vec_ok(gate, d, bytes) && vec_ok(gamma_pre, d, bytes) && vec_ok(dx, d, bytes) && vec_ok(db, d, bytes);
  const norm::FinishArgs f{a.part, a.part_gate, gamma_post, dgamma_post, dgamma_pre, dgate, sp.ctas,
                           sp.parts_per_group, (int)d};
  return norm::by_type(dtype, vec, [&](auto dt, auto v) {
    const int r = norm::by_width((int)d, [&](auto tpr) {
      constexpr int T = decltype(tpr)::value, DT = decltype(dt)::value;
      constexpr bool ODD = !decltype(v)::value;
      // the staged kernel: at 16000 x 4096 bf16 with 8 gates and the next norm 346 us without, 149 to 165 by the
      // GPU with it; 611 and 246 with a gate per row
      auto staged = [&]() -> int {
        constexpr bool SPLIT = T > 512;
        constexpr int T2 = SPLIT ? T : 2 * T;
        // two CTAs' worth of threads share an SM (fewer where one is that large), and
        // so its memory: as many ring rows as fit, up to 3 (2 with the next norm's
        // tensors); one row at least, alone on the SM if need be
        const int width = (int)(SPLIT ? round_up(ceil_div(d, 2), 8) : d) * bytes, row = (dn ? 4 : 2) * (ODD ? (int)round_up(width, 16) + 16 : width);
        static_assert(4 * (8192 * norm::dtype_size<DT>() + 16) + (4 + 2) * 16 * T2 <= norm::MAX_SMEM, "one row and the column sums");
        const bool multi = gate && sp.parts_per_group == 1;   // a CTA's rows are whole groups
        const int sums = ((dn ? 4 : 2) + (multi ? 2 : 0)) * 16 * T2;
        const int share = norm::smem_share(1024 / T2);
        a.stages = std::max(std::min(dn ? 2 : norm::BWD_STAGES, (share - sums) / row), 1);
        const int smem = a.stages * row + sums;
        const int64_t ld_min = std::min(std::min(dy ? ld_dy : ldb, ldb), dn ? std::min(ld_dn, ldy) : ldb);
        a.safe_rows = std::max<int64_t>(0, rows - 1 - 15 / (ld_min * bytes));
        auto* fn = multi ? (dn ? norm::sandwich_bwd_staged_kernel<DT, T2, true, ODD, true, SPLIT>
                               : norm::sandwich_bwd_staged_kernel<DT, T2, false, ODD, true, SPLIT>)
                         : (dn ? norm::sandwich_bwd_staged_kernel<DT, T2, true, ODD, false, SPLIT>
                               : norm::sandwich_bwd_staged_kernel<DT, T2, false, ODD, false, SPLIT>);
        if (smem > 32 * 1024 && !allow_smem(fn, norm::MAX_SMEM)) return NVFP4B200_ERR_CUDA;
        if (!SPLIT) {
          fn<<<(unsigned)sp.ctas, T2, smem, st>>>(a, sp.parts_per_group);
          return launch_status();
        }
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(2 * sp.ctas), 1, 1);
        cfg.blockDim = dim3(T2, 1, 1);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = st;
        cudaLaunchAttribute pair;
        pair.id = cudaLaunchAttributeClusterDimension;
        pair.val.clusterDim.x = 2;
        pair.val.clusterDim.y = pair.val.clusterDim.z = 1;
        cfg.attrs = &pair;
        cfg.numAttrs = 1;
        if (cudaLaunchKernelEx(&cfg, fn, a, sp.parts_per_group) != cudaSuccess) {
          cudaGetLastError();
          return NVFP4B200_ERR_LAUNCH;
        }
        return launch_status();
      };
      if constexpr (!ODD) {
        return staged();
      } else {
        // the ring's copies start on 16-byte boundaries.  (Without the ring 16000 x 4096 bf16 takes 784 us, and
        // 4096 x 16384, 32 registers for 16 columns a thread, 2099 against 225: such tensors are better copied.)
        if (aligned(b, 16) && (!dy || aligned(dy, 16)) && (!dn || (aligned(dn, 16) && aligned(y, 16)))) return staged();
        // 8 columns a thread while 1024 threads cover the row: twice the warps of 16
        // columns (166 -> 123 us at 2013 x 4971 fp16)
        constexpr int T2 = T <= 512 ? 2 * T : T, V = T <= 512 ? 1 : norm::VPT;
        norm::sandwich_bwd_kernel<DT, T2, V><<<(unsigned)sp.ctas, T2, 0, st>>>(a, sp.parts_per_group);
        return launch_status();
      }
    });
    if (r) return r;
    if (!dgamma_post && !dgamma_pre && !dgate) return (int)NVFP4B200_OK;
    const int64_t jobs = dgate && sp.parts_per_group > 1 ? groups + 2 : 2;
    if (d % 4 == 0 && aligned(ws, 16))
      norm::sandwich_bwd_finish_kernel<decltype(dt)::value, 4>
          <<<(unsigned)(jobs * ceil_div(d, 128)), 32 * norm::FINISH_WARPS, 0, st>>>(f);
    else
      norm::sandwich_bwd_finish_kernel<decltype(dt)::value, 1>
          <<<(unsigned)(jobs * ceil_div(d, 32)), 32 * norm::FINISH_WARPS, 0, st>>>(f);
    return launch_status();
  });
}

}  // extern "C"
