// Rows of float32 / bfloat16 / e4m3 values in registers, and the arithmetic that the token-sequence kernels share.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace cssm {

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef short s16x2_t __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));

struct Bf16 { uint16_t u; };   // storage type of a bfloat16 tensor

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const f32x2_t v = {lo, hi};
  const bf16x2_t b = __builtin_convertvector(v, bf16x2_t);   // to nearest, ties to even
  return __builtin_bit_cast(uint32_t, b);
}

// V consecutive values of a row as loaded
template <typename T, int V>
struct Raw;
template <>
struct Raw<float, 4> {
  float4 q;
  __device__ __forceinline__ float get(int i) const { return i == 0 ? q.x : i == 1 ? q.y : i == 2 ? q.z : q.w; }
};
template <>
struct Raw<float, 2> {
  float2 q;
  __device__ __forceinline__ float get(int i) const { return i ? q.y : q.x; }
};
template <>
struct Raw<float, 1> {
  float q;
  __device__ __forceinline__ float get(int) const { return q; }
};
template <>
struct Raw<Bf16, 8> {
  uint4 q;
  __device__ __forceinline__ float get(int i) const {
    const uint32_t w = i < 2 ? q.x : i < 4 ? q.y : i < 6 ? q.z : q.w;
    return __uint_as_float((i & 1) ? (w & 0xffff0000u) : (w << 16));
  }
};
template <>
struct Raw<Bf16, 4> {
  uint2 q;
  __device__ __forceinline__ float get(int i) const {
    const uint32_t w = i < 2 ? q.x : q.y;
    return __uint_as_float((i & 1) ? (w & 0xffff0000u) : (w << 16));
  }
};
template <>
struct Raw<Bf16, 1> {
  uint16_t q;
  __device__ __forceinline__ float get(int) const { return __uint_as_float(uint32_t(q) << 16); }
};

template <typename T, int V>
__device__ __forceinline__ Raw<T, V> load_raw(const T* p) {
  return *reinterpret_cast<const Raw<T, V>*>(p);
}

// V values to a row of T, each rounded once to nearest even
template <int V>
__device__ __forceinline__ void store_row(float* p, const float* v) {
  if constexpr (V == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  else if constexpr (V == 2) *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
  else p[0] = v[0];
}
template <int V>
__device__ __forceinline__ void store_row(Bf16* p, const float* v) {
  if constexpr (V == 8)
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
  else if constexpr (V == 4) *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
  else p->u = uint16_t(pack_bf16(v[0], 0.0f) & 0xffffu);
}

// exp(x) on the hardware's exp2: within an ulp or two, and |x| half steps for the rounding of x log2(e)
__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }
__device__ __forceinline__ float sigmoidf(float z) { return __builtin_amdgcn_rcpf(1.0f + fast_exp(-z)); }

// Biased exponent byte of the least power of two 2^e, e >= -126, with top <= 448 2^e, 448 = 1.75 * 2^8 the largest
// e4m3 value: 1..247; 127 (2^0) for a block of zeros.  top finite and >= 0.
__device__ __forceinline__ int e4m3_scale_byte(float top) {
  const uint32_t u = __float_as_uint(top);
  if (u == 0) return 127;
  const int e = int(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < 1 ? 1 : e;
}
__device__ __forceinline__ float pow2_of(int byte) { return __uint_as_float(uint32_t(byte) << 23); }
__device__ __forceinline__ float pow2_inv(int byte) { return pow2_of(254 - byte); }   // byte 1..247

// four e4m3 values of v[i] * inv, to nearest even; a NaN or an infinite value is stored as NaN
__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true));
}
__device__ __forceinline__ uint32_t pack_e4m3x2(float a, float b) {
  return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false)) & 0xffffu;
}

}  // namespace cssm
