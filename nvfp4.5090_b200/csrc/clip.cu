// Global gradient norm over many tensors, and clipping, for B200 (sm_100a).
//
//     norm   = grad_scale * sqrt(sum over all tensors of g^2)     (or max |g|)
//     coef   = min(1, max_norm / (norm + 1e-6))
//     out_i  = round(g_i * (grad_scale * coef))
//
// The tensors travel as a table in the kernel's parameters (no copy to the
// device, so a captured graph holds it), cut into chunks of one size; CTAs
// stride over the chunks and find a chunk's tensor by bisection.  The first
// kernel leaves one double per CTA in the workspace; whoever needs the norm
// adds those up in one fixed order, so the result does not depend on the
// order in which CTAs finish, nothing has to be zeroed before a call, and
// calls on other streams share nothing.
//
// Squares are summed in fp32 over 8 elements and in fp64 from there on: long
// sums keep their low bits.  A group whose fp32 sum leaves [1e-30, 1e38] is
// summed again in fp64, so neither |g| > 1e19 nor |g| < 1e-19 is lost.
//
// Bound: HBM.  The norm has to be known before the first write, so a
// gradient that does not fit L2 is read twice; the second pass walks the
// chunks backwards and finds the last ones still in L2.
#include "vec.cuh"

#include <algorithm>
#include <vector>

namespace nvfp4b200 {
namespace clip {

constexpr int MAX_TENSORS = 112;   // per launch: 32 bytes each, inside the 4 KB parameter space
constexpr int MAX_CTAS = 1024;     // partial sums per launch
constexpr int THREADS = 256;

struct Table {
  const void* src[MAX_TENSORS];
  void* dst[MAX_TENSORS];
  int64_t numel[MAX_TENSORS];
  int start[MAX_TENSORS];          // first chunk of each tensor
  uint8_t src_dt[MAX_TENSORS], dst_dt[MAX_TENSORS];
  int count, chunks, chunk;        // chunk: elements per chunk
};
static_assert(sizeof(Table) + 64 <= 4096, "kernel parameters");

__device__ __forceinline__ int find_tensor(const Table& t, int chunk) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.start[mid] <= chunk) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// sum of squares of 8 values
__device__ __forceinline__ double sumsq8(const float (&f)[8]) {
  float s = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) s = fmaf(f[j], f[j], s);
  if (s > 1e-30f && s < 1e38f) return (double)s;
  double d = 0.0;
#pragma unroll
  for (int j = 0; j < 8; ++j) d = fma((double)f[j], (double)f[j], d);
  return d;
}

// Largest |f|, a NaN winning: |f| as bits orders NaN above infinity.
__device__ __forceinline__ uint32_t absmax8(const float (&f)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(f[j]) & 0x7FFFFFFFu);
  return m;
}

// Elements before the first 16-byte boundary at or after p (at most n).
template <typename T>
__device__ __forceinline__ int head_of(const T* p, int n) {
  return min(n, (int)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / (int)sizeof(T));
}

template <int DT, bool INF>
__device__ __forceinline__ void reduce_chunk(const void* base, int64_t lo, int64_t hi, double& sum, uint32_t& top) {
  using E = Elem<DT>;
  const typename E::Raw* p = static_cast<const typename E::Raw*>(base) + lo;
  const int n = (int)(hi - lo), head = head_of(p, n), nv = (n - head) >> 3;
  float f[8];
#pragma unroll 4
  for (int i = threadIdx.x; i < nv; i += THREADS) {
    E::unpack(E::load(p + head + 8 * i), f);
    if (INF) top = max(top, absmax8(f)); else sum += sumsq8(f);
  }
  // up to 7 elements before the first vector and 7 after the last
  const int rest = n - 8 * nv, t = threadIdx.x;
  if (t < rest) {
#pragma unroll
    for (int j = 1; j < 8; ++j) f[j] = 0.0f;
    f[0] = E::get(p + (t < head ? t : 8 * nv + t));
    if (INF) top = max(top, absmax8(f)); else sum += sumsq8(f);
  }
}

template <bool INF>
__global__ void __launch_bounds__(THREADS) partials_kernel(const __grid_constant__ Table t, double* __restrict__ partials) {
  __shared__ double red[THREADS / 32];
  double sum = 0.0;
  uint32_t top = 0;
  for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
    const int i = find_tensor(t, c);
    const int64_t lo = (int64_t)(c - t.start[i]) * t.chunk, hi = imin64(t.numel[i], lo + t.chunk);
    if (t.src_dt[i] == NVFP4B200_BF16) reduce_chunk<NVFP4B200_BF16, INF>(t.src[i], lo, hi, sum, top);
    else if (t.src_dt[i] == NVFP4B200_F32) reduce_chunk<NVFP4B200_F32, INF>(t.src[i], lo, hi, sum, top);
    else reduce_chunk<NVFP4B200_F16, INF>(t.src[i], lo, hi, sum, top);
  }
  if (INF) sum = (double)__uint_as_float(__reduce_max_sync(0xffffffffu, top));
  else {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double s = red[0];
#pragma unroll
    for (int w = 1; w < THREADS / 32; ++w) s = INF ? (red[w] > s || red[w] != red[w] ? red[w] : s) : s + red[w];
    partials[blockIdx.x] = s;
  }
}

// The total of n partials in one fixed order, in every thread of the CTA.
template <bool INF>
__device__ __forceinline__ double total_of(const double* __restrict__ partials, int n) {
  __shared__ double red[THREADS / 32];
  auto join = [](double a, double b) { return INF ? (b > a || b != b ? b : a) : a + b; };
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += THREADS) s = join(s, partials[i]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const double other = __shfl_xor_sync(0xffffffffu, s, o);
    s = (threadIdx.x & o) ? join(other, s) : join(s, other);   // the same order in both lanes
  }
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  s = red[0];
#pragma unroll
  for (int w = 1; w < THREADS / 32; ++w) s = join(s, red[w]);
  return s;
}

struct Norm {
  const double* partials;
  int n, inf;
  float grad_scale, max_norm;
  float *norm, *coef;      // optional outputs
  double* total;           // optional: the bare total
};

// grad_scale * coef; thread `writer` also writes the norm and the coefficient.
// A NaN norm gives a NaN coefficient, an infinite one 0, whatever the limit (inf / inf is no factor).
__device__ __forceinline__ float clip_factor(const Norm& a, bool writer) {
  const double total = a.inf ? total_of<true>(a.partials, a.n) : total_of<false>(a.partials, a.n);
  const double norm = (a.inf ? total : sqrt(total)) * fabs((double)a.grad_scale);
  double c = (double)a.max_norm / (norm + 1e-6);
  if (c > 1.0) c = 1.0;
  if (norm == INFINITY) c = 0.0;
  if (writer) {
    if (a.norm) *a.norm = (float)norm;
    if (a.coef) *a.coef = (float)c;
    if (a.total) *a.total = total;
  }
  return a.grad_scale * (float)c;
}

__global__ void __launch_bounds__(THREADS) finish_kernel(const Norm a) { clip_factor(a, threadIdx.x == 0); }

// One chunk, read and written in 16-byte vectors whatever the two tensors'
// alignment (a bucket's views start anywhere): vectors of 8 elements are read
// on the source's boundaries, and where the destination's boundaries fall e
// elements later, each output vector takes its last e elements from the next
// lane's.  A few elements at the chunk's ends go one by one.
template <int SD, int DD>
__device__ __forceinline__ void scale_chunk(const void* src, void* dst, int64_t lo, int64_t hi, float k) {
  using S = Elem<SD>;
  using D = Elem<DD>;
  const typename S::Raw* p = static_cast<const typename S::Raw*>(src) + lo;
  typename D::Raw* o = static_cast<typename D::Raw*>(dst) + lo;
  const int n = (int)(hi - lo), head = head_of(p, n), e = head_of(o + head, n - head);
  // whole vectors of the source, and of the destination (an output vector between
  // the source's boundaries needs two whole ones)
  const int nv = (n - head) >> 3, ov = e == 0 ? nv : max(0, nv - 1);
  p += head;
  o += head + e;
  const int lane = threadIdx.x & 31;
  if (e == 0) {
#pragma unroll 4
    for (int i = threadIdx.x; i < nv; i += THREADS) {
      float f[8];
      S::unpack(S::load(p + 8 * i), f);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] *= k;
      D::store(o + 8 * i, D::pack(f));
    }
  } else {
#pragma unroll 1
    for (int i0 = threadIdx.x - lane; i0 < ov; i0 += THREADS) {   // a warp's 32 output vectors
      const int i = i0 + lane;
      float f[8], t[8];
      const auto own_src = i < nv ? S::load(p + 8 * i) : S::zero();
      const auto next_src = lane == 31 && i + 1 < nv ? S::load(p + 8 * i + 8) : S::zero();
      S::unpack(own_src, f);
      S::unpack(next_src, t);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] *= k;
      if constexpr (DD != NVFP4B200_F32) {
        // 16-bit results are shifted packed: two conditional word shifts, then a half-word
        const auto own = D::pack(f);
        uint32_t x[8] = {own.a.x, own.a.y, own.a.z, own.a.w, 0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 4; ++j) x[4 + j] = __shfl_down_sync(0xffffffffu, x[j], 1);
        if (lane == 31) {
#pragma unroll
          for (int j = 0; j < 8; ++j) t[j] *= k;
          const auto next = D::pack(t);
          x[4] = next.a.x; x[5] = next.a.y; x[6] = next.a.z; x[7] = next.a.w;
        }
#pragma unroll
        for (int j = 0; j < 6; ++j) x[j] = (e & 4) ? x[j + 2] : x[j];
#pragma unroll
        for (int j = 0; j < 5; ++j) x[j] = (e & 2) ? x[j + 1] : x[j];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = __funnelshift_r(x[j], x[j + 1], 16 * (e & 1));
        if (i < ov) *reinterpret_cast<uint4*>(o + 8 * i) = make_uint4(x[0], x[1], x[2], x[3]);
      } else {   // e < 4
        float x[11];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = f[j];
#pragma unroll
        for (int j = 0; j < 3; ++j) x[8 + j] = __shfl_down_sync(0xffffffffu, f[j], 1);
        if (lane == 31) {
#pragma unroll
          for (int j = 0; j < 3; ++j) x[8 + j] = t[j] * k;
        }
#pragma unroll
        for (int j = 0; j < 9; ++j) x[j] = (e & 2) ? x[j + 2] : x[j];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = (e & 1) ? x[j + 1] : x[j];
        if (i < ov) D::store(o + 8 * i, D::pack(f));
      }
    }
  }
  // the elements before and after the output vectors: at most 7 + 7 and 15
  const int before = head + e, rest = n - 8 * ov, t = threadIdx.x;
  if (t < rest) {
    const int j = t < before ? t - before : 8 * ov + t - before;   // relative to o
    o[j] = D::bits(S::get(p + e + j) * k);
  }
}

__global__ void __launch_bounds__(THREADS, 5) scale_kernel(const __grid_constant__ Table t, const Norm a, int first) {
  const float k = clip_factor(a, first && blockIdx.x == 0 && threadIdx.x == 0);
  for (int j = blockIdx.x; j < t.chunks; j += gridDim.x) {
    const int c = t.chunks - 1 - j;
    const int i = find_tensor(t, c);
    if (k == 1.0f && t.dst[i] == t.src[i]) continue;   // in place and nothing to change
    const int64_t lo = (int64_t)(c - t.start[i]) * t.chunk, hi = imin64(t.numel[i], lo + t.chunk);
    const int kind = t.src_dt[i] * 3 + t.dst_dt[i];
    switch (kind) {
      case 0: scale_chunk<0, 0>(t.src[i], t.dst[i], lo, hi, k); break;
      case 1: scale_chunk<0, 1>(t.src[i], t.dst[i], lo, hi, k); break;
      case 2: scale_chunk<0, 2>(t.src[i], t.dst[i], lo, hi, k); break;
      case 3: scale_chunk<1, 0>(t.src[i], t.dst[i], lo, hi, k); break;
      case 4: scale_chunk<1, 1>(t.src[i], t.dst[i], lo, hi, k); break;
      case 5: scale_chunk<1, 2>(t.src[i], t.dst[i], lo, hi, k); break;
      case 6: scale_chunk<2, 0>(t.src[i], t.dst[i], lo, hi, k); break;
      case 7: scale_chunk<2, 1>(t.src[i], t.dst[i], lo, hi, k); break;
      default: scale_chunk<2, 2>(t.src[i], t.dst[i], lo, hi, k); break;
    }
  }
}

// ---- host ----------------------------------------------------------------

// Checks a list of tensors; dst / dst_dt may be null (norm only).
static int check_list(const void* const* src, const int* src_dt, void* const* dst, const int* dst_dt,
                      const int64_t* numel, int count) {
  if (count < 0 || (count > 0 && (!src || !src_dt || !numel)) || (dst && !dst_dt)) return NVFP4B200_ERR_INVALID_ARG;
  for (int i = 0; i < count; ++i) {
    if (numel[i] < 0) return NVFP4B200_ERR_BAD_SHAPE;
    if (!valid_dtype(src_dt[i]) || (dst && !valid_dtype(dst_dt[i]))) return NVFP4B200_ERR_INVALID_ARG;
    if (numel[i] == 0) continue;
    if (!src[i] || (dst && !dst[i])) return NVFP4B200_ERR_INVALID_ARG;
    if (!aligned(src[i], dtype_bytes(src_dt[i])) || (dst && !aligned(dst[i], dtype_bytes(dst_dt[i]))))
      return NVFP4B200_ERR_MISALIGNED;
  }
  return NVFP4B200_OK;
}

// True when every output is apart from all other outputs and from every input
// but its own (which it may equal exactly): otherwise one chunk's writes
// could be another chunk's reads.  -1 when there is no host memory for the check.
static int disjoint(const void* const* src, const int* src_dt, void* const* dst, const int* dst_dt,
                    const int64_t* numel, int count) {
  struct Span {
    uintptr_t lo, hi;
    int i, out;
  };
  std::vector<Span> s;
  try {
    s.reserve(2 * (size_t)count);
  } catch (...) {
    return -1;
  }
  for (int i = 0; i < count; ++i) {
    if (numel[i] == 0) continue;
    const uintptr_t d = reinterpret_cast<uintptr_t>(dst[i]), r = reinterpret_cast<uintptr_t>(src[i]);
    s.push_back({d, d + (uintptr_t)numel[i] * dtype_bytes(dst_dt[i]), i, 1});
    if (r != d || src_dt[i] != dst_dt[i]) s.push_back({r, r + (uintptr_t)numel[i] * dtype_bytes(src_dt[i]), i, 0});
  }
  std::sort(s.begin(), s.end(), [](const Span& a, const Span& b) { return a.lo < b.lo; });
  uintptr_t out_end = 0, in_end = 0;   // furthest end of the outputs / inputs so far
  for (const Span& x : s) {
    if (x.lo < out_end || (x.out && x.lo < in_end)) return 0;
    if (x.out) out_end = std::max(out_end, x.hi); else in_end = std::max(in_end, x.hi);
  }
  return 1;
}

// Elements per chunk: 16384 once that gives every SM four chunks, 4096 below.
static int chunk_for(const int64_t* numel, int count) {
  int64_t total = 0;
  for (int i = 0; i < count; ++i) total += numel[i];
  return total >= (int64_t)4 * 148 * 16384 ? 16384 : 4096;
}

// Fills a table with tensors [i, ..); returns the index after the last one taken.
static int fill(Table& t, const void* const* src, const int* src_dt, void* const* dst, const int* dst_dt,
                const int64_t* numel, int count, int i, int chunk) {
  t.count = 0;
  t.chunk = chunk;
  int64_t chunks = 0;
  for (; i < count && t.count < MAX_TENSORS; ++i) {
    if (numel[i] == 0) continue;
    const int64_t c = ceil_div(numel[i], chunk);
    if (chunks + c > 0x7FFFFFFFll) break;
    const int k = t.count++;
    t.src[k] = src[i];
    t.dst[k] = dst ? dst[i] : nullptr;
    t.numel[k] = numel[i];
    t.start[k] = (int)chunks;
    t.src_dt[k] = (uint8_t)src_dt[i];
    t.dst_dt[k] = dst ? (uint8_t)dst_dt[i] : 0;
    chunks += c;
  }
  t.chunks = (int)chunks;
  return i;
}

static int run_partials(const void* const* src, const int* src_dt, const int64_t* numel, int count, int inf,
                        double* partials, int64_t cap, int64_t* n_out, cudaStream_t st) {
  const int chunk = chunk_for(numel, count);
  const int most = std::min(MAX_CTAS, sm_count_current() * 6);
  int64_t n = 0;
  Table t;
  for (int i = 0; i < count;) {
    i = fill(t, src, src_dt, nullptr, nullptr, numel, count, i, chunk);
    if (t.count == 0) {
      if (i < count) return NVFP4B200_ERR_BAD_SHAPE;
      break;
    }
    const int grid = std::min(t.chunks, most);
    if (n + grid > cap) return NVFP4B200_ERR_BAD_SHAPE;
    if (inf) partials_kernel<true><<<grid, THREADS, 0, st>>>(t, partials + n);
    else partials_kernel<false><<<grid, THREADS, 0, st>>>(t, partials + n);
    const int rc = launch_status();
    if (rc) return rc;
    n += grid;
  }
  *n_out = n;
  return NVFP4B200_OK;
}

}  // namespace clip
}  // namespace nvfp4b200

using namespace nvfp4b200;

extern "C" {

int nvfp4b200_grad_norm(const void* const* grads, const int* grad_dtypes, void* const* outs, const int* out_dtypes,
                        const int64_t* numels, int count, int norm_type, float grad_scale, float max_norm,
                        double* ws, int64_t ws_doubles, float* norm, float* coef, double* total, void* stream) {
  if ((norm_type != 0 && norm_type != 2) || !ws || (!outs && !norm && !coef && !total)) return NVFP4B200_ERR_INVALID_ARG;
  if (!(max_norm >= 0.0f) || !(grad_scale == grad_scale)) return NVFP4B200_ERR_INVALID_ARG;
  int rc = clip::check_list(grads, grad_dtypes, outs, out_dtypes, numels, count);
  if (rc) return rc;
  if (!aligned(ws, 8) || (norm && !aligned(norm, 4)) || (coef && !aligned(coef, 4)) || (total && !aligned(total, 8)))
    return NVFP4B200_ERR_MISALIGNED;
  if (outs) {
    const int apart = clip::disjoint(grads, grad_dtypes, outs, out_dtypes, numels, count);
    if (apart != 1) return apart ? NVFP4B200_ERR_CUDA : NVFP4B200_ERR_INVALID_ARG;
  }
  rc = check_device();
  if (rc) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  int64_t n = 0;
  rc = clip::run_partials(grads, grad_dtypes, numels, count, norm_type == 0, ws, ws_doubles, &n, st);
  if (rc) return rc;
  const clip::Norm a{ws, (int)n, norm_type == 0, grad_scale, max_norm, norm, coef, total};
  bool first = true;
  if (outs) {
    const int chunk = clip::chunk_for(numels, count);
    clip::Table t;
    for (int i = 0; i < count;) {
      i = clip::fill(t, grads, grad_dtypes, outs, out_dtypes, numels, count, i, chunk);
      if (t.count == 0) break;
      const int grid = std::min(t.chunks, sm_count_current() * 8);
      clip::scale_kernel<<<grid, clip::THREADS, 0, st>>>(t, a, first);
      rc = launch_status();
      if (rc) return rc;
      first = false;
    }
  }
  if (first) clip::finish_kernel<<<1, clip::THREADS, 0, st>>>(a);
  return launch_status();
}

int nvfp4b200_grad_norm_finish(const double* partials, int64_t n, int norm_type, float grad_scale, float max_norm,
                               float* norm, float* coef, void* stream) {
  if (!partials || (norm_type != 0 && norm_type != 2) || (!norm && !coef) || !(max_norm >= 0.0f) ||
      !(grad_scale == grad_scale))
    return NVFP4B200_ERR_INVALID_ARG;
  if (n < 0 || n > (1 << 20)) return NVFP4B200_ERR_BAD_SHAPE;
  if (!aligned(partials, 8) || (norm && !aligned(norm, 4)) || (coef && !aligned(coef, 4)))
    return NVFP4B200_ERR_MISALIGNED;
  int rc = check_device();
  if (rc) return rc;
  const clip::Norm a{partials, (int)n, norm_type == 0, grad_scale, max_norm, norm, coef, nullptr};
  clip::finish_kernel<<<1, clip::THREADS, 0, (cudaStream_t)stream>>>(a);
  return launch_status();
}

}  // extern "C"
