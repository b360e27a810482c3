// Norm of each head of queries and keys with the rotation by their positions in the same pass (gfx950):
//   n = x r w,  r = 1 / sqrt(mean(x^2) + eps) or 1 / sqrt(sum(x^2) + eps) or 1;  pair (n_a, n_b) turned by f_j p_{axis j}
// and its adjoint: g = dy turned back,  dx = r w g - x r^3 / count sum(w g x),  dw = sum over rows and heads of g x r.
// An angle is the product of a whole number and a float64, reduced to a part of a turn in float64, so that it is as exact
// for far positions as for near ones.  Cosines and sines are made once for a row and serve all of its heads.
// Bound by HBM: a lane holds 2 V values of a head, those that are turned together, in two vectors, and the next ones are on
// their way while they are computed.  16384 rows of 16 + 16 heads of 128 in bfloat16: 55 us, 4.9 TB/s (81 us without the
// loads ahead and a row's table for each wave); adjoint 108 us, 3.7 TB/s, where 207 registers leave two waves a SIMD.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "launch.h"
#include "token_util.h"

namespace cssm {

namespace {

constexpr int kAxes = 4, kRotaryGroups = 1024;   // workgroups of a launch, at most

__device__ __forceinline__ const char* head_row(const TokenRows& x, long long m, int T, size_t size) {
  const int b = int(m) / T, t = int(m) - b * T;   // M is at most 2^31 - 1
  return static_cast<const char*>(x.p) + ((long long)b * x.batch + (long long)t * x.row) * (long long)size;
}

// V values aligned to their elements, in loads of 16 bytes
template <typename E, int V>
__device__ __forceinline__ void load_some(const E* p, bool on, E none, E (&v)[V]) {
  constexpr int W = V * sizeof(E) < 16 ? V : 16 / sizeof(E);
  typedef E vec __attribute__((ext_vector_type(W), aligned(sizeof(E))));
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = none;
  if (!on) return;
#pragma unroll
  for (int i = 0; i < V; i += W) {
    if constexpr (W == 1) {
      v[i] = p[i];
    } else {
      const vec q = *reinterpret_cast<const vec*>(p + i);
#pragma unroll
      for (int j = 0; j < W; ++j) v[i + j] = q[j];
    }
  }
}

// what a lane keeps for the rows it takes
template <int V, int NV, bool HALVES>
struct Pairs {
  double f[NV][V];       // turns a position
  int axis[NV][V], o0[NV], o1[NV];
  float c[NV][V], s[NV][V];
  bool on[NV];
  __device__ __forceinline__ void place(const Rotary& a, int l, int lanes) {
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int p = (l + lanes * n) * V;
      on[n] = 2 * p < a.D;
      const bool apart = HALVES && p < a.P;
      o0[n] = apart ? p : 2 * p;
      o1[n] = apart ? p + a.P : 2 * p + V;
    }
  }
  __device__ __forceinline__ void init(const Rotary& a, int l, int lanes) {
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int p = (l + lanes * n) * V;   // P a multiple of V
      load_some<double, V>(a.freq + p, p < a.P, 0.0, f[n]);
      load_some<int, V>(a.axis + p, p < a.P, 0, axis[n]);
#pragma unroll
      for (int v = 0; v < V; ++v) f[n][v] *= 0.15915494309189535;   // 1 / (2 pi)
    }
  }
  // cosines and sines of row m
  __device__ __forceinline__ void row(const Rotary& a, long long m) {
    if (!a.P) {
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int v = 0; v < V; ++v) c[n][v] = 1.0f, s[n][v] = 0.0f;
      return;
    }
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
__device__ __forceinline__ void load_values(const T* p, bool on, Raw<T, V>& r) {
  r = Raw<T, V>{};
  if (on) r = load_raw<T, V>(p);
}
template <typename T, int V>
__device__ __forceinline__ void unpack(const Raw<T, V>& r, float (&v)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = r.get(i);
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
__global__ __launch_bounds__(256) void rotate_heads(Rotary a, int lanes, int slices, uint32_t units) {
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), l = lane % lanes, group = lane / lanes, heads = 64 / lanes;
  extern __shared__ float s_dw[];   // BACK with weights: (4 waves, 2, D)
  Pairs<V, NV, HALVES> pairs;
  pairs.place(a, l, lanes);
  float w[2][NV][2][V], dw[2][NV][2][V];
  // a row's turns: q's heads, then k's; while one is computed the next one's values are on their way
  const uint32_t step = gridDim.x * 4;
  uint32_t u = blockIdx.x * 4 + wave, m = slices == 1 ? u : u / uint32_t(slices);   // with step below 2^32
  int slice = int(u - m * slices), turn = 0;
  const auto turns_of = [&](int i) { return a.of[i].H <= slice * heads ? 0 : (a.of[i].H - slice * heads - 1) / (slices * heads) + 1; };
  Raw<T, V> xa[NV], xb[NV], ya[NV], yb[NV];
  const auto fetch = [&](int i, int t) {
    const RotaryHeads& r = a.of[i];
    const int h = (slice + t * slices) * heads + group;
    const bool on = h < r.H;
    const T* x = reinterpret_cast<const T*>(head_row(r.x, m, a.T, sizeof(T))) + h * a.D;
    const T* dy = BACK ? reinterpret_cast<const T*>(head_row(r.dy, m, a.T, sizeof(T))) + h * a.D : nullptr;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      load_values<T, V>(x + pairs.o0[n], on && pairs.on[n], xa[n]);
      load_values<T, V>(x + pairs.o1[n], on && pairs.on[n], xb[n]);
      if (BACK) {
        load_values<T, V>(dy + pairs.o0[n], on && pairs.on[n], ya[n]);
        load_values<T, V>(dy + pairs.o1[n], on && pairs.on[n], yb[n]);
      }
    }
  };
  const auto take = [&](auto which, int t, long long row, int part, const Raw<T, V> (&ra)[NV], const Raw<T, V> (&rb)[NV],
                        const Raw<T, V> (&qa)[NV], const Raw<T, V> (&qb)[NV]) {
    constexpr int i = decltype(which)::value;
    const RotaryHeads& r = a.of[i];
    const int h = (part + t * slices) * heads + group;
    const bool on = h < r.H;
    T* out = static_cast<T*>(r.y) + (size_t(row) * r.H + h) * a.D;
    float fa[NV][V], fb[NV][V], squares = 0.0f;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      unpack<T, V>(ra[n], fa[n]), unpack<T, V>(rb[n], fb[n]);
#pragma unroll
      for (int v = 0; v < V; ++v) squares = fmaf(fa[n][v], fa[n][v], squares), squares = fmaf(fb[n][v], fb[n][v], squares);
    }
    const float rs = scale_of(a, a.norm == 2 ? 0.0f : lanes_sum(squares, lanes));
    if constexpr (!BACK) {
#pragma unroll
      for (int n = 0; n < NV; ++n) {
#pragma unroll
        for (int v = 0; v < V; ++v) fa[n][v] = fa[n][v] * rs * w[i][n][0][v], fb[n][v] = fb[n][v] * rs * w[i][n][1][v];
        pairs.template turn<false>(fa[n], fb[n], n);
      }
    } else {
      float ga[NV][V], gb[NV][V], dot = 0.0f;
      const float rw = on ? rs : 0.0f;   // without a head and eps r has no value
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        unpack<T, V>(qa[n], ga[n]), unpack<T, V>(qb[n], gb[n]);
        pairs.template turn<true>(ga[n], gb[n], n);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          dw[i][n][0][v] = fmaf(ga[n][v], fa[n][v] * rw, dw[i][n][0][v]);
          dw[i][n][1][v] = fmaf(gb[n][v], fb[n][v] * rw, dw[i][n][1][v]);
          ga[n][v] *= w[i][n][0][v], gb[n][v] *= w[i][n][1][v];
          dot = fmaf(ga[n][v], fa[n][v], dot), dot = fmaf(gb[n][v], fb[n][v], dot);
        }
      }
      // x's share: r^3 / count sum(w g x), in an order that a large or small r does not overflow
      const float share = a.norm == 2 ? 0.0f : rs * (rs * lanes_sum(dot, lanes)) * (a.norm == 0 ? rs / float(a.D) : rs);
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int v = 0; v < V; ++v) fa[n][v] = rs * ga[n][v] - share * fa[n][v], fb[n][v] = rs * gb[n][v] - share * fb[n][v];
    }
#pragma unroll
    for (int n = 0; n < NV; ++n)
      if (on && pairs.on[n]) store_row<V>(out + pairs.o0[n], fa[n]), store_row<V>(out + pairs.o1[n], fb[n]);
  };
  int turns_q = turns_of(0), turns = turns_q + turns_of(1);
  const auto advance = [&]() {   // to the next turn of this row, or the next row that has one
    for (++turn; u < units && turn >= turns;) {
      u += step, m = slices == 1 ? u : u / uint32_t(slices), slice = int(u - m * slices), turn = 0;
      turns_q = turns_of(0), turns = turns_q + turns_of(1);
    }
  };
  turn = -1;
  advance();
  if (u < units) fetch(turn >= turns_q, turn >= turns_q ? turn - turns_q : turn);
  pairs.init(a, l, lanes);
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const float* from = a.of[i].w;
      load_some<float, V>(from + pairs.o0[n], from && pairs.on[n], 1.0f, w[i][n][0]);
      load_some<float, V>(from + pairs.o1[n], from && pairs.on[n], 1.0f, w[i][n][1]);
      if (BACK)
#pragma unroll
        for (int v = 0; v < V; ++v) dw[i][n][0][v] = dw[i][n][1][v] = 0.0f;
    }
  long long angles = -1;   // the row that the cosines are of
  while (u < units) {
    const long long row = m;
    const int part = slice, i = turn >= turns_q, t = i ? turn - turns_q : turn;
    Raw<T, V> ra[NV], rb[NV], qa[NV], qb[NV];
#pragma unroll
    for (int n = 0; n < NV; ++n) ra[n] = xa[n], rb[n] = xb[n], qa[n] = ya[n], qb[n] = yb[n];
    advance();
    if (u < units) fetch(turn >= turns_q, turn >= turns_q ? turn - turns_q : turn);
    if (row != angles) pairs.row(a, row), angles = row;
    if (i == 0) take(std::integral_constant<int, 0>(), t, row, part, ra, rb, qa, qb);
    else take(std::integral_constant<int, 1>(), t, row, part, ra, rb, qa, qb);
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

// the workgroups' sums of dw added up: 16 columns and 64 threads down the rows each
__global__ __launch_bounds__(1024) void rotary_dw(const float* parts, int groups, int D, float* dwq, float* dwk) {
  __shared__ double s[64][17];
  const int x = threadIdx.x % 16, y = threadIdx.x / 16, c = blockIdx.x * 16 + x;
  double sum = 0.0;
  if (c < 2 * D) {
#pragma unroll 8
    for (int i = y; i < groups; i += 64) sum += parts[size_t(i) * 2 * D + c];
  }
  s[y][x] = sum;
  __syncthreads();
  if (y || c >= 2 * D) return;
  for (int i = 1; i < 64; ++i) sum += s[i][x];
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
  const long long units = a.M * slices, groups = (units + 3) / 4;   // at most 2^31 - 1, or 4096
  const int grid = int(groups < kRotaryGroups ? groups : kRotaryGroups);
  const size_t lds = BACK && a.parts ? size_t(8) * a.D * sizeof(float) : 0;
  if (a.halves) rotate_heads<T, V, NV, true, BACK><<<grid, 256, lds, s>>>(a, lanes, slices, uint32_t(units));
  else rotate_heads<T, V, NV, false, BACK><<<grid, 256, lds, s>>>(a, lanes, slices, uint32_t(units));
  if (BACK && a.parts) rotary_dw<<<(2 * a.D + 15) / 16, 1024, 0, s>>>(a.parts, grid, a.D, a.of[0].dw, a.of[1].dw);
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
