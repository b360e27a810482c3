// Root-mean-square norm of rows, with the residual's addition before it and an 8-bit output with scales (gfx950):
//   s = round(x + residual) (the sum the next layer reads, so the norm is of its rounded values),
//   n = s rstd, rstd = 1 / sqrt(mean(s^2) + eps), y = n w;  8 bits: y = 2^e q, one e for each 128 of a row
// and its adjoint ds = rstd (w dy - n mean(w dy n)) + dstream, dw = sum over rows of dy n.
// Both are bound by HBM: a row is read once into registers (64 or 256 threads a row, 16 bytes a load), reduced by
// lane exchanges and written once.  Sums are float32 in a row and float64 over the rows' partial sums.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "launch.h"
#include "token_util.h"

namespace cssm {

namespace {

constexpr int kNormBlocks = 1024;   // workgroups whose rows' sums of dw are added up afterwards, at most

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int l = 32; l > 0; l /= 2) v += __shfl_xor(v, l);
  return v;
}
// sum over the TPR threads of a row; scratch: 4 floats (TPR = 256)
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* scratch) {
  v = wave_sum(v);
  if constexpr (TPR == 256) {
    __syncthreads();
    if (threadIdx.x % 64 == 0) scratch[threadIdx.x / 64] = v;
    __syncthreads();
    v = (scratch[0] + scratch[1]) + (scratch[2] + scratch[3]);
  }
  return v;
}
__device__ __forceinline__ float rstd_of(float sum, int C, float eps) {
  return float(1.0 / sqrt(double(sum) / double(C) + double(eps)));
}

__device__ __forceinline__ float round_to(float v, float) { return v; }
__device__ __forceinline__ float round_to(float v, Bf16) { return __uint_as_float(pack_bf16(0.0f, v) & 0xffff0000u); }
__device__ __forceinline__ float load_one(const float* p) { return *p; }
__device__ __forceinline__ float load_one(const Bf16* p) { return __uint_as_float(uint32_t(p->u) << 16); }

// the largest finite magnitude of lanes l ^ 1, l ^ 2, .. l ^ (LANES - 1)
template <int LANES>
__device__ __forceinline__ float top_of(float top) {
#pragma unroll
  for (int l = 1; l < LANES; l *= 2) top = fmaxf(top, __shfl_xor(top, l));
  return top;
}

// C % V == 0, 16-byte aligned rows, C <= V NV TPR.  Bound by HBM: 16384 x 4096 bf16 with a residual, to 8 bits, 85 us,
// 5.5 TB/s; to bf16 98 us, 5.5 TB/s
template <typename T, int V, int NV, int TPR, bool E4M3>
__global__ void __launch_bounds__(256) rms_norm_fwd(const T* __restrict__ x, const T* __restrict__ res, long long M,
                                                    int C, const float* __restrict__ w, float eps, T* __restrict__ s,
                                                    void* __restrict__ y, uint8_t* __restrict__ scales) {
  __shared__ float scratch[4];
  const int l = threadIdx.x % TPR;
  const long long row = (long long)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
  const bool on = row < M;
  const size_t at = size_t(on ? row : 0) * C;
  float f[NV][V], sum = 0.0f;
  Raw<T, V> a[NV], r[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * TPR + l) * V;
    if (on && c < C) {
      a[j] = load_raw<T, V>(x + at + c);
      if (res) r[j] = load_raw<T, V>(res + at + c);
    }
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * TPR + l) * V;
#pragma unroll
    for (int v = 0; v < V; ++v) f[j][v] = 0.0f;
    if (on && c < C) {
#pragma unroll
      for (int v = 0; v < V; ++v) f[j][v] = res ? round_to(a[j].get(v) + r[j].get(v), T()) : a[j].get(v);
      if (res) store_row<V>(s + at + c, f[j]);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) sum = fmaf(f[j][v], f[j][v], sum);
  }
  const float rstd = rstd_of(row_sum<TPR>(sum, scratch), C, eps);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * TPR + l) * V;
    float top = 0.0f;
    if (c < C) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        f[j][v] = (f[j][v] * rstd) * w[c + v];
        const float m = fabsf(f[j][v]);
        if (E4M3) top = fmaxf(top, m < INFINITY ? m : 0.0f);
      }
    }
    if constexpr (E4M3) {
      top = top_of<128 / V>(top);
      if (!on || c >= C) continue;
      const int byte = e4m3_scale_byte(top);
      const float inv = pow2_inv(byte);
      uint32_t q[V / 4];
#pragma unroll
      for (int v = 0; v < V; v += 4)
        q[v / 4] = pack_e4m3x4(f[j][v] * inv, f[j][v + 1] * inv, f[j][v + 2] * inv, f[j][v + 3] * inv);
      uint8_t* out = static_cast<uint8_t*>(y) + at + c;
      if constexpr (V == 8) *reinterpret_cast<uint2*>(out) = make_uint2(q[0], q[1]);
      else *reinterpret_cast<uint32_t*>(out) = q[0];
      if (c % 128 == 0) scales[size_t(row) * ((C + 127) / 128) + c / 128] = uint8_t(byte);
    } else {
      if (on && c < C) store_row<V>(static_cast<T*>(y) + at + c, f[j]);
    }
  }
}

// any C and alignment: a workgroup a row, a wave for each 128 columns, the rounded sum read again for the output.
// Element loads: 16384 x 4095 bf16 takes 301 us where 4096 takes 98; 8192 x 8192 float32, past the registers' widths, 317
template <typename T, bool E4M3>
__global__ void __launch_bounds__(256) rms_norm_any(const T* __restrict__ x, const T* __restrict__ res, int C,
                                                    const float* __restrict__ w, float eps, T* __restrict__ s,
                                                    void* __restrict__ y, uint8_t* __restrict__ scales) {
  __shared__ float scratch[4];
  const size_t at = size_t(blockIdx.x) * C;
  const int wave = threadIdx.x / 64, l = threadIdx.x % 64;
  auto value = [&](int c) {
    const float v = load_one(x + at + c);
    return res ? round_to(v + load_one(res + at + c), T()) : v;
  };
  float sum = 0.0f;
  for (int b = wave * 128; b < C; b += 512)
    for (int c = b + l; c < C && c < b + 128; c += 64) {
      float v = value(c);
      if (res) store_row<1>(s + at + c, &v);
      sum = fmaf(v, v, sum);
    }
  const float rstd = rstd_of(row_sum<256>(sum, scratch), C, eps);
  for (int b = wave * 128; b < C; b += 512) {
    float f[2], top = 0.0f;
    for (int k = 0; k < 2; ++k) {
      const int c = b + l + 64 * k;
      f[k] = c < C ? (value(c) * rstd) * w[c] : 0.0f;
      const float m = fabsf(f[k]);
      top = fmaxf(top, m < INFINITY ? m : 0.0f);
    }
    if (E4M3) {
      const int byte = e4m3_scale_byte(top_of<64>(top));
      const float inv = pow2_inv(byte);
      for (int k = 0; k < 2; ++k) {
        const int c = b + l + 64 * k;
        if (c < C) static_cast<uint8_t*>(y)[at + c] = uint8_t(pack_e4m3x2(f[k] * inv, 0.0f));
      }
      if (l == 0) scales[size_t(blockIdx.x) * ((C + 127) / 128) + b / 128] = uint8_t(byte);
    } else {
      for (int k = 0; k < 2; ++k) {
        const int c = b + l + 64 * k;
        if (c < C) store_row<1>(static_cast<T*>(y) + at + c, &f[k]);
      }
    }
  }
}

// the adjoint; each workgroup walks rows row0, row0 + grid, .. and keeps its columns' sums of dw in registers.  Bound by
// HBM: 32768 x 1024 bf16 with the stream's gradient, right behind the forward, 47 us, 5.7 TB/s, and 4 for the sums behind
// it; both 62 us on tensors that no cache holds
template <typename T, int V, int NV, int TPR>
__global__ void __launch_bounds__(256) rms_norm_bwd(const T* __restrict__ dy, const T* __restrict__ ds,
                                                    const T* __restrict__ s, long long M, int C,
                                                    const float* __restrict__ w, float eps, T* __restrict__ dx,
                                                    float* __restrict__ parts) {
  __shared__ float scratch[8];
  __shared__ float dws[TPR == 64 ? 4 * V * NV * 64 : 1];
  const int l = threadIdx.x % TPR, RPB = 256 / TPR;
  float ww[NV][V], dw[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (j * TPR + l) * V + v;
      ww[j][v] = c < C ? w[c] : 0.0f;
      dw[j][v] = 0.0f;
    }
  const long long step = (long long)gridDim.x * RPB;
  const long long trips = (M + step - 1) / step;
  for (long long i = 0; i < trips; ++i) {
    const long long row = i * step + (long long)blockIdx.x * RPB + threadIdx.x / TPR;
    const bool on = row < M;
    const size_t at = size_t(on ? row : 0) * C;
    Raw<T, V> g[NV], q[NV], e[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * TPR + l) * V;
      if (on && c < C) {
        q[j] = load_raw<T, V>(s + at + c);
        g[j] = load_raw<T, V>(dy + at + c);
        if (ds) e[j] = load_raw<T, V>(ds + at + c);
      }
    }
    float ss = 0.0f, sd = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (on && (j * TPR + l) * V < C)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float f = q[j].get(v);
          ss = fmaf(f, f, ss);
          sd = fmaf(f, ww[j][v] * g[j].get(v), sd);
        }
    ss = row_sum<TPR>(ss, scratch);
    sd = row_sum<TPR>(sd, scratch + 4);
    const float rstd = rstd_of(ss, C, eps), mean = sd * rstd / float(C);   // mean of w dy n
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * TPR + l) * V;
      if (on && c < C) {
        float o[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float n = q[j].get(v) * rstd, gg = g[j].get(v);
          dw[j][v] = fmaf(gg, n, dw[j][v]);
          o[v] = rstd * fmaf(-n, mean, ww[j][v] * gg);
          if (ds) o[v] += e[j].get(v);
        }
        store_row<V>(dx + at + c, o);
      }
    }
  }
  if constexpr (TPR == 64) {
    const int wave = threadIdx.x / 64;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) dws[(wave * NV + j) * 64 * V + l * V + v] = dw[j][v];
    __syncthreads();
    for (int c = threadIdx.x; c < C; c += 256)
      parts[size_t(blockIdx.x) * C + c] = (dws[c] + dws[NV * 64 * V + c]) + (dws[2 * NV * 64 * V + c] + dws[3 * NV * 64 * V + c]);
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int c = (j * TPR + l) * V + v;
        if (c < C) parts[size_t(blockIdx.x) * C + c] = dw[j][v];
      }
  }
}

// any C and alignment: ds and the rows' rstd, then dw's partial sums from both (16384 x 4095 bf16 310 us, 4096: 129)
template <typename T>
__global__ void __launch_bounds__(256) rms_norm_bwd_any(const T* __restrict__ dy, const T* __restrict__ ds,
                                                        const T* __restrict__ s, int C, const float* __restrict__ w,
                                                        float eps, T* __restrict__ dx, float* __restrict__ rstds) {
  __shared__ float scratch[8];
  const size_t at = size_t(blockIdx.x) * C;
  float ss = 0.0f, sd = 0.0f;
  for (int c = threadIdx.x; c < C; c += 256) {
    const float f = load_one(s + at + c);
    ss = fmaf(f, f, ss);
    sd = fmaf(f, w[c] * load_one(dy + at + c), sd);
  }
  ss = row_sum<256>(ss, scratch);
  sd = row_sum<256>(sd, scratch + 4);
  const float rstd = rstd_of(ss, C, eps), mean = sd * rstd / float(C);
  for (int c = threadIdx.x; c < C; c += 256) {
    const float n = load_one(s + at + c) * rstd;
    float o = rstd * fmaf(-n, mean, w[c] * load_one(dy + at + c));
    if (ds) o += load_one(ds + at + c);
    store_row<1>(dx + at + c, &o);
  }
  if (threadIdx.x == 0) rstds[blockIdx.x] = rstd;
}
template <typename T>
__global__ void __launch_bounds__(256) rms_norm_dw_any(const T* __restrict__ dy, const T* __restrict__ s, long long M,
                                                       int C, const float* __restrict__ rstds,
                                                       float* __restrict__ parts) {
  const int nct = (C + 255) / 256, c = int(blockIdx.x % unsigned(nct)) * 256 + threadIdx.x;
  const int slice = int(blockIdx.x / unsigned(nct)), slices = int(gridDim.x / unsigned(nct));
  if (c >= C) return;
  float sum = 0.0f;
  for (long long m = slice; m < M; m += slices)
    sum = fmaf(load_one(dy + size_t(m) * C + c), load_one(s + size_t(m) * C + c) * rstds[m], sum);
  parts[size_t(slice) * C + c] = sum;
}

__global__ void __launch_bounds__(1024) column_sums(const float* __restrict__ parts, int n, int C, float* __restrict__ out) {
  __shared__ double sum[64][16];
  const int l = threadIdx.x % 16, grp = threadIdx.x / 16, c = int(blockIdx.x) * 16 + l;
  double k = 0.0;
  if (c < C)
#pragma unroll 4
    for (int i = grp; i < n; i += 64) k += double(parts[size_t(i) * C + c]);
  sum[grp][l] = k;
  for (int m = 32; m > 0; m /= 2) {
    __syncthreads();
    if (grp < m) sum[grp][l] += sum[grp + m][l];
  }
  if (grp == 0 && c < C) out[c] = float(sum[0][l]);
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// f(T, V NV TPR of the register kernels) or false where none fits
template <typename T, int V, typename F>
bool by_width(int C, F&& f) {
  using std::integral_constant;
  if (C <= 64 * V) f(integral_constant<int, 1>(), integral_constant<int, 64>());
  else if (C <= 128 * V) f(integral_constant<int, 2>(), integral_constant<int, 64>());
  else if (C <= 256 * V) f(integral_constant<int, 4>(), integral_constant<int, 64>());
  else if (C <= 512 * V) f(integral_constant<int, 2>(), integral_constant<int, 256>());
  else if (C <= 1024 * V) f(integral_constant<int, 4>(), integral_constant<int, 256>());
  else return false;
  return true;
}

template <typename T, int V>
hipError_t norm_fwd(const RmsNorm& a, hipStream_t st) {
  const T* x = static_cast<const T*>(a.x);
  const T* r = static_cast<const T*>(a.res);
  T* s = static_cast<T*>(a.s);
  bool done = false;
  if (a.C % V == 0 && aligned16(x) && aligned16(r) && aligned16(s) && aligned16(a.y))
    done = by_width<T, V>(a.C, [&](auto nv, auto tpr) {
      constexpr int NV = decltype(nv)::value, TPR = decltype(tpr)::value;
      const unsigned g = unsigned((a.M + 256 / TPR - 1) / (256 / TPR));
      if (a.scales) rms_norm_fwd<T, V, NV, TPR, true><<<g, 256, 0, st>>>(x, r, a.M, a.C, a.w, a.eps, s, a.y, a.scales);
      else rms_norm_fwd<T, V, NV, TPR, false><<<g, 256, 0, st>>>(x, r, a.M, a.C, a.w, a.eps, s, a.y, nullptr);
    });
  if (!done) {
    if (a.scales) rms_norm_any<T, true><<<unsigned(a.M), 256, 0, st>>>(x, r, a.C, a.w, a.eps, s, a.y, a.scales);
    else rms_norm_any<T, false><<<unsigned(a.M), 256, 0, st>>>(x, r, a.C, a.w, a.eps, s, a.y, nullptr);
  }
  return hipGetLastError();
}

template <typename T, int V>
hipError_t norm_bwd(const RmsNorm& a, hipStream_t st) {
  const T* dy = static_cast<const T*>(a.dy);
  const T* ds = static_cast<const T*>(a.ds);
  const T* s = static_cast<const T*>(a.x);
  T* dx = static_cast<T*>(a.dx);
  int n = 0;
  const bool done = a.C % V == 0 && aligned16(dy) && aligned16(ds) && aligned16(s) && aligned16(dx) &&
                    by_width<T, V>(a.C, [&](auto nv, auto tpr) {
                      constexpr int NV = decltype(nv)::value, TPR = decltype(tpr)::value;
                      const long long g = (a.M + 256 / TPR - 1) / (256 / TPR);
                      n = int(g < kNormBlocks ? g : kNormBlocks);
                      rms_norm_bwd<T, V, NV, TPR><<<unsigned(n), 256, 0, st>>>(dy, ds, s, a.M, a.C, a.w, a.eps, dx, a.parts);
                    });
  if (!done) {
    n = int(a.M < 256 ? a.M : 256);
    rms_norm_bwd_any<T><<<unsigned(a.M), 256, 0, st>>>(dy, ds, s, a.C, a.w, a.eps, dx, a.rstds);
    rms_norm_dw_any<T><<<unsigned((a.C + 255) / 256) * unsigned(n), 256, 0, st>>>(dy, s, a.M, a.C, a.rstds, a.parts);
  }
  column_sums<<<unsigned((a.C + 15) / 16), 1024, 0, st>>>(a.parts, n, a.C, a.dw);
  return hipGetLastError();
}

// ---- 8-bit values of whole tensors: rows for the left side of a product, a weight for the right

// (M, K) -> e4m3 and the exponent of each 128 of a row.  Bound by HBM: 16 threads a block of 128, 8 values a thread in 16-
// or 32-byte loads, where the rows are aligned for it (K % 8 == 0): 16384 x 4096 bf16 41 us, 4.9 TB/s
template <typename T>
__global__ void __launch_bounds__(256) quantize_rows8(const T* __restrict__ x, long long M, int K,
                                                      uint8_t* __restrict__ q, uint8_t* __restrict__ scales) {
  constexpr int V = 16 / sizeof(T), N = 8 / V;
  const int nb = (K + 127) / 128, l = threadIdx.x % 16;
  const long long i = (long long)blockIdx.x * 16 + threadIdx.x / 16;
  if (i >= M * nb) return;   // (a block's 16 threads alike)
  const long long m = i / nb;
  const int c = int(i % nb) * 128 + l * 8;
  const size_t at = size_t(m) * K + c;
  float f[8], top = 0.0f;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    Raw<T, V> r = {};
    if (c < K) r = load_raw<T, V>(x + at + j * V);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      f[j * V + v] = r.get(v);
      const float w = fabsf(f[j * V + v]);
      top = fmaxf(top, w < INFINITY ? w : 0.0f);
    }
  }
  const int byte = e4m3_scale_byte(top_of<16>(top));
  const float inv = pow2_inv(byte);
  if (c < K)
    *reinterpret_cast<uint2*>(q + at) = make_uint2(pack_e4m3x4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv),
                                                   pack_e4m3x4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv));
  if (l == 0) scales[i] = uint8_t(byte);
}
// any K and alignment: a wave a block, 2 values a lane (16384 x 4090 bf16: 142 us)
template <typename T>
__global__ void __launch_bounds__(256) quantize_rows(const T* __restrict__ x, long long M, int K,
                                                     uint8_t* __restrict__ q, uint8_t* __restrict__ scales) {
  const int nb = (K + 127) / 128, l = threadIdx.x % 64;
  const long long i = (long long)blockIdx.x * 4 + threadIdx.x / 64;
  if (i >= M * nb) return;
  const long long m = i / nb;
  const int b = int(i % nb) * 128;
  float f[2], top = 0.0f;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int c = b + l * 2 + k;
    f[k] = c < K ? load_one(x + size_t(m) * K + c) : 0.0f;
    const float v = fabsf(f[k]);
    top = fmaxf(top, v < INFINITY ? v : 0.0f);
  }
  const int byte = e4m3_scale_byte(top_of<64>(top));
  const float inv = pow2_inv(byte);
  const uint32_t p = pack_e4m3x2(f[0] * inv, f[1] * inv);
  uint8_t* o = q + size_t(m) * K + b + l * 2;
  if (b + l * 2 < K) o[0] = uint8_t(p);
  if (b + l * 2 + 1 < K) o[1] = uint8_t(p >> 8);
  if (l == 0) scales[i] = uint8_t(byte);
}

// Dense kernel (K, N) float32 -> (N, K) e4m3 and the exponent of each 128 x 128: a workgroup a tile, in registers, turned
// in LDS.  Done once a weight: 4096 x 8192 49 us, 3.4 TB/s
__global__ void __launch_bounds__(256) quantize_weight(const float* __restrict__ w, int K, int N, uint8_t* __restrict__ q,
                                                       uint8_t* __restrict__ scales) {
  __shared__ float tops[4];
  __shared__ uint8_t tile[128][132];
  const int nkb = (K + 127) / 128, kb = int(blockIdx.x) % nkb, nb = int(blockIdx.x) / nkb;
  const int k0 = kb * 128, n0 = nb * 128, nl = threadIdx.x % 128, kl = threadIdx.x / 128;
  float f[64], top = 0.0f;
#pragma unroll
  for (int i = 0; i < 64; ++i) {
    const int k = k0 + 2 * i + kl, n = n0 + nl;
    f[i] = k < K && n < N ? w[size_t(k) * N + n] : 0.0f;
    const float v = fabsf(f[i]);
    top = fmaxf(top, v < INFINITY ? v : 0.0f);
  }
  top = top_of<64>(top);
  if (threadIdx.x % 64 == 0) tops[threadIdx.x / 64] = top;
  __syncthreads();
  const int byte = e4m3_scale_byte(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])));
  const float inv = pow2_inv(byte);
#pragma unroll
  for (int i = 0; i < 64; ++i) tile[nl][2 * i + kl] = uint8_t(pack_e4m3x2(f[i] * inv, 0.0f));
  __syncthreads();
  for (int i = threadIdx.x; i < 128 * 128; i += 256) {
    const int n = i / 128, k = i % 128;
    if (n0 + n < N && k0 + k < K) q[size_t(n0 + n) * K + k0 + k] = tile[n][k];
  }
  if (threadIdx.x == 0) scales[size_t(nb) * nkb + kb] = uint8_t(byte);
}

}  // namespace

size_t rms_norm_bwd_workspace(long long M, int C) {
  return (size_t(M < kNormBlocks ? M : kNormBlocks) * size_t(C) + size_t(M)) * 4;
}

hipError_t launch_rms_norm(const RmsNorm& a, int dtype, hipStream_t s) {
  return dtype == 0 ? norm_fwd<float, 4>(a, s) : norm_fwd<Bf16, 8>(a, s);
}
hipError_t launch_rms_norm_bwd(const RmsNorm& a, int dtype, hipStream_t s) {
  return dtype == 0 ? norm_bwd<float, 4>(a, s) : norm_bwd<Bf16, 8>(a, s);
}
template <typename T>
static void quantize(const T* x, long long M, int K, uint8_t* q, uint8_t* scales, hipStream_t s) {
  const long long blocks = M * ((K + 127) / 128);
  if (K % 8 == 0 && aligned16(x) && reinterpret_cast<uintptr_t>(q) % 8 == 0)
    quantize_rows8<T><<<unsigned((blocks + 15) / 16), 256, 0, s>>>(x, M, K, q, scales);
  else
    quantize_rows<T><<<unsigned((blocks + 3) / 4), 256, 0, s>>>(x, M, K, q, scales);
}
hipError_t launch_quantize_rows(const void* x, int dtype, long long M, int K, uint8_t* q, uint8_t* scales, hipStream_t s) {
  if (dtype == 0) quantize(static_cast<const float*>(x), M, K, q, scales, s);
  else quantize(static_cast<const Bf16*>(x), M, K, q, scales, s);
  return hipGetLastError();
}
hipError_t launch_quantize_weight(const float* w, int K, int N, uint8_t* q, uint8_t* scales, hipStream_t s) {
  quantize_weight<<<unsigned((K + 127) / 128) * unsigned((N + 127) / 128), 256, 0, s>>>(w, K, N, q, scales);
  return hipGetLastError();
}

}  // namespace cssm
