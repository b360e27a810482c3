// Matrix product of 8-bit rows and an 8-bit weight (gfx950):
//   out[m][n] = act(sum over 128-blocks b of 2^(sa[m][b] + sw[n / 128][b]) sum_{k in b} a[m][k] w[n][k] + bias[n])
// a (M, K), w (N, K) e4m3.  Two forms, by the output's type:
//   bfloat16  the 8-bit matrix instruction.  The scales are powers of two, which the scaled form
//             (v_mfma_scale_f32_16x16x128) applies exactly in its float32 accumulation, one instruction for a whole
//             128-block.  Its own scales are one for each 32 of k; the four of a block get the same byte, so the order
//             of k within a block does not matter as long as both sides agree.  The instruction adds the products of
//             neighbouring k with what lies about 13 bits below the largest of them dropped: 1.4e-5 of a result of
//             normal values, 1 / 100 of the output's own rounding.
//   float32   the values as bfloat16, which holds each exactly, on the bfloat16 instruction, whose sums are off by a
//             float32 rounding (1e-8 .. 1e-7 measured), each block's sum scaled as it joins the others.
// The weight is the instruction's first operand: a lane then holds four consecutive n of one m.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "launch.h"
#include "token_util.h"

namespace cssm {

namespace {

typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

// 8 e4m3 values as bfloat16 (exact)
__device__ __forceinline__ bf16x8_t widen(int lo, int hi) {
  const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
  const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
  return bf16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// 32 bytes of a row at k, zeros behind K (a multiple of 16)
__device__ __forceinline__ i32x8_t load32(const uint8_t* row, int k, int K) {
  uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
  if (k < K) lo = *reinterpret_cast<const uint4*>(row + k);
  if (k + 16 < K) hi = *reinterpret_cast<const uint4*>(row + k + 16);
  return i32x8_t{int(lo.x), int(lo.y), int(lo.z), int(lo.w), int(hi.x), int(hi.y), int(hi.z), int(hi.w)};
}

__device__ __forceinline__ float activate(float v, int act) {
  if (act == 1) {   // gelu, tanh form: v sigmoid(2 t)
    const float t = 0.7978845608028654f * fmaf(0.044715f * v * v, v, v);
    return v * sigmoidf(2.0f * t);
  }
  return act == 2 ? v * sigmoidf(v) : v;
}

template <typename O>
__device__ __forceinline__ void store4(O* out, size_t at, int n, int N, bool wide, const float* v) {
  if (wide && n + 4 <= N) {
    store_row<4>(out + at, v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < N) store_row<1>(out + at + i, v + i);
  }
}

// 128 x 128 of the output a workgroup, 64 x 64 a wave, operands straight from global memory
template <typename O, bool WIDE>
__global__ void __launch_bounds__(256) product_tile(Product8 p) {
  const int nmt = (p.M + 127) / 128;
  const int mt = int(blockIdx.x) % nmt, nt = int(blockIdx.x) / nmt;
  const int wave = threadIdx.x / 64, l = threadIdx.x % 64, r = l % 16, kq = l / 16;
  const int m0 = mt * 128 + (wave % 2) * 64, n0 = nt * 128 + (wave / 2) * 64;
  const int nkb = (p.K + 127) / 128;
  const uint8_t *wr[4], *ar[4], *as[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = min(n0 + i * 16 + r, p.N - 1), m = min(m0 + i * 16 + r, p.M - 1);
    wr[i] = p.w + size_t(n) * p.K;
    ar[i] = p.a + size_t(m) * p.K;
    as[i] = p.sa + size_t(m) * nkb;
  }
  const uint8_t* ws = p.sw + size_t(nt) * nkb;
  f32x4_t acc[4][4] = {};
  for (int b = 0; b < nkb; ++b) {
    i32x8_t fw[4], fa[4];
    int sa[4];
    const int sw = ws[b];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      fw[i] = load32(wr[i], b * 128 + kq * 32, p.K);
      fa[i] = load32(ar[i], b * 128 + kq * 32, p.K);
      sa[i] = as[i][b];
    }
    if constexpr (WIDE) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f32x4_t part = {};
#pragma unroll
          for (int s = 0; s < 4; ++s)
            part = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(fw[i][2 * s], fw[i][2 * s + 1]),
                                                           widen(fa[j][2 * s], fa[j][2 * s + 1]), part, 0, 0, 0);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] += __builtin_amdgcn_ldexpf(part[e], sw + sa[j] - 254);
        }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fw[i], fa[j], acc[i][j], 0, 0, 0, sw, 0, sa[j]);
    }
  }
  const bool wide = p.N % 4 == 0 && reinterpret_cast<uintptr_t>(p.out) % (4 * sizeof(O)) == 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = n0 + i * 16 + kq * 4;
    float bias[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) bias[e] = p.bias && n + e < p.N ? p.bias[n + e] : 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + j * 16 + r;
      if (m >= p.M) continue;
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = activate(acc[i][j][e] + bias[e], p.act);
      store4(static_cast<O*>(p.out), size_t(m) * p.N + n, n, p.N, wide, v);
    }
  }
}

}  // namespace

hipError_t launch_product8(const Product8& p, int out_dtype, hipStream_t s) {
  const unsigned g = unsigned((p.M + 127) / 128) * unsigned((p.N + 127) / 128);
  if (out_dtype == 0) product_tile<float, true><<<g, 256, 0, s>>>(p);
  else product_tile<Bf16, false><<<g, 256, 0, s>>>(p);
  return hipGetLastError();
}

}  // namespace cssm
