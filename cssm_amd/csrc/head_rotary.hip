// Norm of each head of queries and keys with the rotation by their positions in the same pass (gfx950):
//   n = x r w,  r = 1 / sqrt(mean(x^2) + eps) or 1 / sqrt(sum(x^2) + eps) or 1;  pair (n_a, n_b) turned by f_j p_{axis j}
// and its adjoint: g = dy turned back,  dx = r w g - x r^3 / count sum(w g x),  dw = sum over rows and heads of g x r.
// An angle is the product of a whole number and a float64, reduced to a part of a turn in float64, so that it is as exact
// for far positions as for near ones.  Cosines and sines are made once for a row and serve all of its heads.
// Bound by HBM: a lane holds 2 V values of a head, those that are turned together, in two vectors; 16384 rows of 16 + 16
// heads of 128 in bfloat16 move 537 MB with their outputs.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "launch.h"
#include "token_util.h"

namespace cssm {

namespace {

constexpr int kAxes = 4, kRotaryGroups = 1024;   // workgroups of the adjoint, at most

template <typename T, int V>
struct Lane {   // a lane's values of a head: a at o0 .. o0 + V - 1, b at o1 ..
  float a[V], b[V];
};

__device__ __forceinline__ const char* head_row(const RotaryHeads& x, long long m, int T, size_t size) {
  const long long b = m / T, t = m - b * T;
  return static_cast<const char*>(x.x.p) + (b * x.x.batch + t * x.x.row) * (long long)size;
}

// what a lane keeps for the rows it takes
template <int V, int NV, bool HALVES>
struct Pairs {
  double f[NV][V];       // turns a position
  int axis[NV][V], o0[NV], o1[NV];
  float c[NV][V], s[NV][V];
  bool on[NV];
  __device__ __forceinline__ void init(const Rotary& a, int l, int lanes) {
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int p = (l + lanes * n) * V;
      on[n] = 2 * p < a.D;
      const bool apart = HALVES && p < a.P;
      o0[n] = apart ? p : 2 * p;
      o1[n] = apart ? p + a.P : 2 * p + V;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const bool turned = p + v < a.P;
        f[n][v] = turned ? a.freq[p + v] * 0.15915494309189535 : 0.0;   // 1 / (2 pi)
        axis[n][v] = turned ? a.axis[p + v] : 0;
      }
    }
  }
  // cosines and sines of row m
  __device__ __forceinline__ void row(const Rotary& a, long long m) {
    int at[kAxes];
#pragma unroll
    for (int i = 0; i < kAxes; ++i) at[i] = i < a.axes ? a.positions[m * a.axes + i] : at[i ? i - 1 : 0];
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        int p = at[0];
#pragma unroll
        for (int i = 1; i < kAxes; ++i) p = axis[n][v] >= i ? at[i] : p;
        double t = double(p) * f[n][v];
        t -= rint(t);
        sincospif(2.0f * float(t), &s[n][v], &c[n][v]);
      }
  }
  // (a, b) turned, or with BACK turned back
  template <bool BACK>
  __device__ __forceinline__ void turn(float (&a)[V], float (&b)[V], int n) const {
    if constexpr (HALVES || V == 1) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float sn = BACK ? -s[n][v] : s[n][v], x = a[v], y = b[v];
        a[v] = x * c[n][v] - y * sn, b[v] = y * c[n][v] + x * sn;
      }
    } else {   // the lane's pairs are neighbours: half of them in a, half in b
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float* q = v < V / 2 ? a + 2 * v : b + 2 * v - V;
        const float sn = BACK ? -s[n][v] : s[n][v], x = q[0], y = q[1];
        q[0] = x * c[n][v] - y * sn, q[1] = y * c[n][v] + x * sn;
      }
    }
  }
};

template <typename T, int V>
__device__ __forceinline__ void load_values(const T* p, bool on, float (&v)[V]) {
  if (on) {
    const Raw<T, V> r = load_raw<T, V>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = r.get(i);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = 0.0f;
  }
}

__device__ __forceinline__ float lanes_sum(float v, int lanes) {
  for (int o = 1; o < lanes; o *= 2) v += __shfl_xor(v, o);
  return v;
}

__device__ __forceinline__ float scale_of(const Rotary& a, float squares) {
  if (a.norm == 2) return 1.0f;
  return 1.0f / sqrtf((a.norm == 0 ? squares / float(a.D) : squares) + a.eps);
}

// `lanes` lanes side by side take a head (a power of two), a wave 64 / lanes heads at once and `slices` waves a row's heads
template <typename T, int V, int NV, bool HALVES, bool BACK>
__global__ __launch_bounds__(256) void rotate_heads(Rotary a, int lanes, int slices, long long units) {
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, l = lane % lanes, group = lane / lanes, heads = 64 / lanes;
  extern __shared__ float s_dw[];   // BACK with weights: (4 waves, 2, D)
  Pairs<V, NV, HALVES> pairs;
  pairs.init(a, l, lanes);
  float w[2][NV][2][V], dw[2][NV][2][V];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float* from = a.of[i].w;
        w[i][n][0][v] = from && pairs.on[n] ? from[pairs.o0[n] + v] : 1.0f;
        w[i][n][1][v] = from && pairs.on[n] ? from[pairs.o1[n] + v] : 1.0f;
        if (BACK) dw[i][n][0][v] = dw[i][n][1][v] = 0.0f;
      }
  for (long long u = (long long)blockIdx.x * 4 + wave; u < units; u += (long long)gridDim.x * 4) {
    const long long m = slices == 1 ? u : u / slices;
    const int slice = slices == 1 ? 0 : int(u - m * slices);
    if (a.P) pairs.row(a, m);
    else {
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int v = 0; v < V; ++v) pairs.c[n][v] = 1.0f, pairs.s[n][v] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const RotaryHeads& r = a.of[i];
      const T* x = reinterpret_cast<const T*>(head_row(r, m, a.T, sizeof(T)));
      for (int h0 = slice * heads; h0 < r.H; h0 += slices * heads) {
        const int h = h0 + group;
        const bool on = h < r.H;
        float xa[NV][V], xb[NV][V], squares = 0.0f;
#pragma unroll
        for (int n = 0; n < NV; ++n) {
          load_values<T, V>(x + h * a.D + pairs.o0[n], on && pairs.on[n], xa[n]);
          load_values<T, V>(x + h * a.D + pairs.o1[n], on && pairs.on[n], xb[n]);
        }
        const size_t out = (size_t(m) * r.H + h) * a.D;
        float ga[NV][V], gb[NV][V];
        if constexpr (BACK) {
          const T* dy = static_cast<const T*>(r.dy.p) + (m / a.T) * r.dy.batch + (m % a.T) * r.dy.row + h * a.D;
#pragma unroll
          for (int n = 0; n < NV; ++n) {
            load_values<T, V>(dy + pairs.o0[n], on && pairs.on[n], ga[n]);
            load_values<T, V>(dy + pairs.o1[n], on && pairs.on[n], gb[n]);
          }
        }
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
          for (int v = 0; v < V; ++v) squares = fmaf(xa[n][v], xa[n][v], squares), squares = fmaf(xb[n][v], xb[n][v], squares);
        const float rs = scale_of(a, lanes_sum(squares, lanes));
        if constexpr (!BACK) {
#pragma unroll
          for (int n = 0; n < NV; ++n) {
#pragma unroll
            for (int v = 0; v < V; ++v) xa[n][v] = xa[n][v] * rs * w[i][n][0][v], xb[n][v] = xb[n][v] * rs * w[i][n][1][v];
            pairs.template turn<false>(xa[n], xb[n], n);
            if (on && pairs.on[n]) {
              store_row<V>(static_cast<T*>(r.y) + out + pairs.o0[n], xa[n]);
              store_row<V>(static_cast<T*>(r.y) + out + pairs.o1[n], xb[n]);
            }
          }
        } else {
          float dot = 0.0f;
#pragma unroll
          for (int n = 0; n < NV; ++n) {
            pairs.template turn<true>(ga[n], gb[n], n);
#pragma unroll
            for (int v = 0; v < V; ++v) {
              dw[i][n][0][v] = fmaf(ga[n][v], xa[n][v] * rs, dw[i][n][0][v]);
              dw[i][n][1][v] = fmaf(gb[n][v], xb[n][v] * rs, dw[i][n][1][v]);
              ga[n][v] *= w[i][n][0][v], gb[n][v] *= w[i][n][1][v];
              dot = fmaf(ga[n][v], xa[n][v], dot), dot = fmaf(gb[n][v], xb[n][v], dot);
            }
          }
          dot = lanes_sum(dot, lanes);
          // x's share: r^3 / count sum(w g x), in an order that a large or small r does not overflow
          const float share = a.norm == 2 ? 0.0f : rs * (rs * dot) * (a.norm == 0 ? rs / float(a.D) : rs);
#pragma unroll
          for (int n = 0; n < NV; ++n) {
#pragma unroll
            for (int v = 0; v < V; ++v) xa[n][v] = rs * ga[n][v] - share * xa[n][v], xb[n][v] = rs * gb[n][v] - share * xb[n][v];
            if (on && pairs.on[n]) {
              store_row<V>(static_cast<T*>(r.y) + out + pairs.o0[n], xa[n]);
              store_row<V>(static_cast<T*>(r.y) + out + pairs.o1[n], xb[n]);
            }
          }
        }
      }
    }
  }
  if constexpr (BACK) {
    if (!a.parts) return;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float x = dw[i][n][0][v], y = dw[i][n][1][v];
          for (int o = lanes; o < 64; o *= 2) x += __shfl_xor(x, o), y += __shfl_xor(y, o);
          if (group == 0 && pairs.on[n]) {
            s_dw[(wave * 2 + i) * a.D + pairs.o0[n] + v] = x;
            s_dw[(wave * 2 + i) * a.D + pairs.o1[n] + v] = y;
          }
        }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * a.D; c += 256)
      a.parts[size_t(blockIdx.x) * 2 * a.D + c] = (s_dw[c] + s_dw[2 * a.D + c]) + (s_dw[4 * a.D + c] + s_dw[6 * a.D + c]);
  }
}

// the workgroups' sums of dw added up: 16 columns and 16 threads down the rows each
__global__ __launch_bounds__(256) void rotary_dw(const float* parts, int groups, int D, float* dwq, float* dwk) {
  __shared__ double s[16][17];
  const int x = threadIdx.x % 16, y = threadIdx.x / 16, c = blockIdx.x * 16 + x;
  double sum = 0.0;
  if (c < 2 * D)
    for (int i = y; i < groups; i += 16) sum += parts[size_t(i) * 2 * D + c];
  s[y][x] = sum;
  __syncthreads();
  if (y || c >= 2 * D) return;
  for (int i = 1; i < 16; ++i) sum += s[i][x];
  float* out = c < D ? dwq : dwk;
  if (out) out[c < D ? c : c - D] = float(sum);
}

bool wide(const TokenRows& r, int D, size_t size) {
  return reinterpret_cast<uintptr_t>(r.p) % 16 == 0 && r.batch * (long long)size % 16 == 0 && r.row * (long long)size % 16 == 0 &&
         D * size % 16 == 0;
}

template <typename T, int V, int NV, bool BACK>
void launch(const Rotary& a, int lanes, hipStream_t s) {
  const int heads = 64 / lanes, most = a.of[0].H > a.of[1].H ? a.of[0].H : a.of[1].H;
  // few rows: a row's heads over several waves, each with the angles of its own (16 rows of 16 + 4 heads: one launch's time)
  int slices = (most + heads - 1) / heads;
  while (slices > 1 && a.M * slices > 4096) slices = (slices + 1) / 2;
  const long long units = a.M * slices, groups = (units + 3) / 4;
  const int grid = int(BACK ? (groups < kRotaryGroups ? groups : kRotaryGroups) : groups < 8192 ? groups : 8192);
  const size_t lds = BACK && a.parts ? size_t(8) * a.D * sizeof(float) : 0;
  if (a.halves) rotate_heads<T, V, NV, true, BACK><<<grid, 256, lds, s>>>(a, lanes, slices, units);
  else rotate_heads<T, V, NV, false, BACK><<<grid, 256, lds, s>>>(a, lanes, slices, units);
  if (BACK && a.parts) rotary_dw<<<(2 * a.D + 15) / 16, 256, 0, s>>>(a.parts, grid, a.D, a.of[0].dw, a.of[1].dw);
}

template <typename T, bool BACK>
void run(const Rotary& a, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
  bool vec = a.D % (2 * V) == 0 && a.P % V == 0;
  for (int i = 0; i < 2 && vec; ++i)
    if (a.of[i].H)
      vec = wide(a.of[i].x, a.D, sizeof(T)) && reinterpret_cast<uintptr_t>(a.of[i].y) % 16 == 0 && (!BACK || wide(a.of[i].dy, a.D, sizeof(T)));
  int lanes = 1;
  while (lanes * V * 2 < a.D) lanes *= 2;
  // vectors, two a lane; else single elements, a wave a head
  if (vec && lanes <= 64) launch<T, V, 1, BACK>(a, lanes, s);
  else launch<T, 1, 4, BACK>(a, 64, s);
}

}  // namespace

size_t rotate_heads_bwd_workspace(int D) { return size_t(kRotaryGroups) * 2 * D * sizeof(float); }

hipError_t launch_rotate_heads(const Rotary& a, int dtype, bool back, hipStream_t s) {
  if (dtype == 0) back ? run<float, true>(a, s) : run<float, false>(a, s);
  else back ? run<Bf16, true>(a, s) : run<Bf16, false>(a, s);
  return hipGetLastError();
}

}  // namespace cssm
