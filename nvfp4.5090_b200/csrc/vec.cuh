// Typed element access shared by the kernels that take bf16, fp16 and fp32
// tensors: 8 elements at a time as floats (16-byte vectors) or one by one.
#pragma once

#include "common.cuh"

#include <cuda_fp16.h>

namespace nvfp4b200 {

template <int DT>
struct Elem;

template <>
struct Elem<NVFP4B200_BF16> {
  using Raw = uint16_t;
  struct Vec8 {
    uint4 a;
  };
  static __device__ __forceinline__ Vec8 load(const Raw* p) { return Vec8{__ldg(reinterpret_cast<const uint4*>(p))}; }
  static __device__ __forceinline__ Vec8 zero() { return Vec8{make_uint4(0, 0, 0, 0)}; }
  static __device__ __forceinline__ void unpack(const Vec8& v, float (&f)[8]) {
    const uint32_t w[4] = {v.a.x, v.a.y, v.a.z, v.a.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[2 * j] = bf16lo(w[j]);
      f[2 * j + 1] = bf16hi(w[j]);
    }
  }
  static __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ Vec8 pack(const float (&f)[8]) {
    return Vec8{make_uint4(pack2(f[0], f[1]), pack2(f[2], f[3]), pack2(f[4], f[5]), pack2(f[6], f[7]))};
  }
  static __device__ __forceinline__ void store(Raw* p, const Vec8& v) { *reinterpret_cast<uint4*>(p) = v.a; }
  static __device__ __forceinline__ float get(const Raw* p) { return __uint_as_float((uint32_t)__ldg(p) << 16); }
  static __device__ __forceinline__ Raw bits(float f) { return __bfloat16_as_ushort(__float2bfloat16_rn(f)); }
  static __device__ __forceinline__ float value(Raw b) { return __uint_as_float((uint32_t)b << 16); }
};

template <>
struct Elem<NVFP4B200_F16> {
  using Raw = uint16_t;
  using Vec8 = Elem<NVFP4B200_BF16>::Vec8;
  static __device__ __forceinline__ Vec8 load(const Raw* p) { return Vec8{__ldg(reinterpret_cast<const uint4*>(p))}; }
  static __device__ __forceinline__ Vec8 zero() { return Vec8{make_uint4(0, 0, 0, 0)}; }
  static __device__ __forceinline__ void unpack(const Vec8& v, float (&f)[8]) {
    const uint32_t w[4] = {v.a.x, v.a.y, v.a.z, v.a.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
      f[2 * j] = t.x;
      f[2 * j + 1] = t.y;
    }
  }
  static __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ Vec8 pack(const float (&f)[8]) {
    return Vec8{make_uint4(pack2(f[0], f[1]), pack2(f[2], f[3]), pack2(f[4], f[5]), pack2(f[6], f[7]))};
  }
  static __device__ __forceinline__ void store(Raw* p, const Vec8& v) { *reinterpret_cast<uint4*>(p) = v.a; }
  static __device__ __forceinline__ float get(const Raw* p) { return __half2float(__ushort_as_half(__ldg(p))); }
  static __device__ __forceinline__ Raw bits(float f) { return __half_as_ushort(__float2half_rn(f)); }
  static __device__ __forceinline__ float value(Raw b) { return __half2float(__ushort_as_half(b)); }
};

template <>
struct Elem<NVFP4B200_F32> {
  using Raw = float;
  struct Vec8 {
    float4 a, b;
  };
  static __device__ __forceinline__ Vec8 load(const Raw* p) {
    return Vec8{__ldg(reinterpret_cast<const float4*>(p)), __ldg(reinterpret_cast<const float4*>(p) + 1)};
  }
  static __device__ __forceinline__ Vec8 zero() {
    return Vec8{make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
  }
  static __device__ __forceinline__ void unpack(const Vec8& v, float (&f)[8]) {
    f[0] = v.a.x; f[1] = v.a.y; f[2] = v.a.z; f[3] = v.a.w;
    f[4] = v.b.x; f[5] = v.b.y; f[6] = v.b.z; f[7] = v.b.w;
  }
  static __device__ __forceinline__ Vec8 pack(const float (&f)[8]) {
    return Vec8{make_float4(f[0], f[1], f[2], f[3]), make_float4(f[4], f[5], f[6], f[7])};
  }
  static __device__ __forceinline__ void store(Raw* p, const Vec8& v) {
    reinterpret_cast<float4*>(p)[0] = v.a;
    reinterpret_cast<float4*>(p)[1] = v.b;
  }
  static __device__ __forceinline__ float get(const Raw* p) { return __ldg(p); }
  static __device__ __forceinline__ Raw bits(float f) { return f; }
  static __device__ __forceinline__ float value(Raw b) { return b; }
};

inline bool valid_dtype(int dt) { return dt == NVFP4B200_BF16 || dt == NVFP4B200_F32 || dt == NVFP4B200_F16; }
inline int dtype_bytes(int dt) { return dt == NVFP4B200_F32 ? 4 : 2; }

}  // namespace nvfp4b200
