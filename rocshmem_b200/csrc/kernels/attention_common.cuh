// Pieces that the attention operators share: rows spread over groups of lanes, conversions between element types.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "attention_kernels.hpp"
#include "attention_plan.hpp"
#include "launch.cuh"

namespace rocshmem {
namespace kernels {
namespace attn {

struct e4m3 {
  uint8_t v;
};

// Eight consecutive elements of a row in 32 bits. 16-bit and fp32 rows move 16 bytes an access, e4m3 rows eight.
template <typename T>
struct Raw8;
template <>
struct Raw8<float> {
  float4 a, b;
};
template <>
struct Raw8<__nv_bfloat16> {
  uint4 a;
};
template <>
struct Raw8<__half> {
  uint4 a;
};
template <>
struct Raw8<e4m3> {
  uint2 a;
};

// Elements [8 at, 8 at + 8) of the row at `p`.
template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T *p, int at = 0) {
  return *reinterpret_cast<const Raw8<T> *>(p + 8 * at);
}

__device__ __forceinline__ void unpack8(const Raw8<float> &r, float (&x)[8]) {
  x[0] = r.a.x, x[1] = r.a.y, x[2] = r.a.z, x[3] = r.a.w, x[4] = r.b.x, x[5] = r.b.y, x[6] = r.b.z, x[7] = r.b.w;
}
__device__ __forceinline__ void unpack8(const Raw8<__nv_bfloat16> &r, float (&x)[8]) {
  const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack8(const Raw8<__half> &r, float (&x)[8]) {
  const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
    x[2 * i] = f.x, x[2 * i + 1] = f.y;
  }
}
// Four e4m3 codes as two pairs of fp16 values (exact).
__device__ __forceinline__ void e4m3_pairs(uint32_t w, uint32_t &lo, uint32_t &hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi) : "r"(w));
}
__device__ __forceinline__ void unpack8(const Raw8<e4m3> &r, float (&x)[8]) {
  uint32_t w[4];
  e4m3_pairs(r.a.x, w[0], w[1]);
  e4m3_pairs(r.a.y, w[2], w[3]);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
    x[2 * i] = f.x, x[2 * i + 1] = f.y;
  }
}

// Four consecutive elements in 32 bits.
template <typename T>
struct Raw4 {
  uint2 a;
};
template <>
struct Raw4<float> {
  float4 a;
};
template <typename T>
__device__ __forceinline__ Raw4<T> load4(const T *p) {
  return *reinterpret_cast<const Raw4<T> *>(p);
}
__device__ __forceinline__ void unpack4(const Raw4<float> &r, float2 *x) {
  x[0] = make_float2(r.a.x, r.a.y), x[1] = make_float2(r.a.z, r.a.w);
}
__device__ __forceinline__ void unpack4(const Raw4<__nv_bfloat16> &r, float2 *x) {
  x[0] = make_float2(__uint_as_float(r.a.x << 16), __uint_as_float(r.a.x & 0xffff0000u));
  x[1] = make_float2(__uint_as_float(r.a.y << 16), __uint_as_float(r.a.y & 0xffff0000u));
}
__device__ __forceinline__ void unpack4(const Raw4<__half> &r, float2 *x) {
  x[0] = __half22float2(*reinterpret_cast<const __half2 *>(&r.a.x));
  x[1] = __half22float2(*reinterpret_cast<const __half2 *>(&r.a.y));
}
__device__ __forceinline__ void store4(float *p, const float2 *x) {
  *reinterpret_cast<float4 *>(p) = make_float4(x[0].x, x[0].y, x[1].x, x[1].y);
}
__device__ __forceinline__ void store4(__nv_bfloat16 *p, const float2 *x) {
  const __nv_bfloat162 lo = __floats2bfloat162_rn(x[0].x, x[0].y), hi = __floats2bfloat162_rn(x[1].x, x[1].y);
  *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const uint32_t *>(&lo),
      *reinterpret_cast<const uint32_t *>(&hi));
}
__device__ __forceinline__ void store4(__half *p, const float2 *x) {
  const __half2 lo = __floats2half2_rn(x[0].x, x[0].y), hi = __floats2half2_rn(x[1].x, x[1].y);
  *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const uint32_t *>(&lo),
      *reinterpret_cast<const uint32_t *>(&hi));
}

// One rounding to the nearest value of the type, ties to even.
__device__ __forceinline__ void store8(float *p, const float (&x)[8]) {
  float4 *v = reinterpret_cast<float4 *>(p);
  v[0] = make_float4(x[0], x[1], x[2], x[3]);
  v[1] = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16 *p, const float (&x)[8]) {
  uint4 o;
  uint32_t *w = reinterpret_cast<uint32_t *>(&o);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t *>(&h);
  }
  *reinterpret_cast<uint4 *>(p) = o;
}
__device__ __forceinline__ void store8(__half *p, const float (&x)[8]) {
  uint4 o;
  uint32_t *w = reinterpret_cast<uint32_t *>(&o);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t *>(&h);
  }
  *reinterpret_cast<uint4 *>(p) = o;
}

__device__ __forceinline__ void store1(float *p, float x) { *p = x; }
__device__ __forceinline__ void store1(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ void store1(__half *p, float x) { *p = __float2half_rn(x); }

// Two fp32 operations in one instruction.
__device__ __forceinline__ unsigned long long bits2(float2 a) { return *reinterpret_cast<unsigned long long *>(&a); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)), "l"(bits2(c)));
  return *reinterpret_cast<float2 *>(&r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)));
  return *reinterpret_cast<float2 *>(&r);
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// Sum over the `LANES` neighbouring lanes (a power of two) that hold one row.
template <int LANES>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The largest magnitude among the row's elements, of which the lane holds eight: that of the bits, so that a NaN or
// infinity is it. 16-bit types compare two elements in one instruction.
template <int LANES>
__device__ __forceinline__ float group_top(const Raw8<float> &r) {
  const float v[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
#pragma unroll
  for (int o = LANES / 2; o; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  return __uint_as_float(top);
}
template <int LANES>
__device__ __forceinline__ uint32_t group_top16(const uint4 &r) {
  uint32_t top = __vmaxu2(__vmaxu2(r.x & 0x7fff7fffu, r.y & 0x7fff7fffu),
      __vmaxu2(r.z & 0x7fff7fffu, r.w & 0x7fff7fffu));
#pragma unroll
  for (int o = LANES / 2; o; o >>= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, o));
  return max(top & 0xffffu, top >> 16);
}
template <int LANES>
__device__ __forceinline__ float group_top(const Raw8<__nv_bfloat16> &r) {
  return __uint_as_float(group_top16<LANES>(r.a) << 16);
}
template <int LANES>
__device__ __forceinline__ float group_top(const Raw8<__half> &r) {
  return __half2float(__ushort_as_half(static_cast<unsigned short>(group_top16<LANES>(r.a))));
}

template <int V>
struct Int {
  static constexpr int value = V;
};

// Launches a kernel that may be set up while the one before it on the stream is running; it has to wait for that one's
// end (griddepcontrol.wait) before it reads.
template <typename... KArgs>
cudaError_t launch_after(void (*kernel)(KArgs...), dim3 grid, unsigned threads, cudaStream_t s,
                         typename same_as_kernel<KArgs>::type... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Lanes that hold a row of `dim` elements, eight each: 8, 16 or 32 (those past the row's end hold zeros).
inline int row_lanes(int dim) { return dim <= 64 ? 8 : dim <= 128 ? 16 : 32; }

}  // namespace attn
}  // namespace kernels
}  // namespace rocshmem
