// Adjoint of the gated delta rule over token sequences (gfx950).  In a chunk (csrc/delta_rule.hip has the forward's form and
// its L, P, D, gamma, d), with E the errors and S the states that the forward kept, U = beta E, and dS the state's gradient:
//   dU = P^T dY + d K dS',  X = dU - L^T beta dU,  dV = beta X,  dbeta = X.E (row by row)
//   dS <- gamma_31 dS' + scale Q^T gamma dY - K^T gamma beta X
//   Y_ij = scale D_ij dY_i.U_j (i >= j),  Z_ij = D_ij beta_i X_i.U_j (i > j)
//   dQ = Y K + scale gamma dY S^T,  read = -Z K - gamma beta X S^T,  write = Y^T Q - Z^T K + d U dS'^T,  dK = read + write
// A decay is a factor of whatever crosses it, from a writer before it or the chunk's first state to a reader from it on or the
// chunk's last state, and its gradient is the sum of just that:
//   ddecay_l = sum over i >= l > j of W_ij + sum over i >= l of r_i + sum over j < l of c_j + gamma_31 <S, dS'>
//   W_ij = P_ij dY_i.U_j - A_ij beta_i X_i.U_j,  r_i = q_i.(scale gamma_i S dY_i) - k_i.(gamma_i beta_i S X_i),  c_j = d_j k_j.(dS' U_j)
// Every term has the factor a_l: nothing cancels that is larger than it, and a_l = 0 gives 0.  What the rows from l on read
// less what they write, the shorter sum, is the same by cancellation: at a = exp(-8) nothing of it was right.
// delta_back_pairs (bfloat16; float32: delta_walk_back) carries dS from chunk to chunk, as the forward does S, and keeps it
// behind every 128th row; then delta_grads takes each 128 rows by themselves, forwards with S and backwards with dS, a wave 16
// of the keys' columns, so that the sums over dv lie within a wave.  The states between a segment's chunks go to the workspace
// on the way forwards and are read again by the same threads on the way back, where dS' is at hand, for <S, dS'>.
// Training 4 x 4096 x 16 heads of 128: delta_back_pairs 350 us (2.7 a chunk, a chain of products as the forward's; one kind of
// wave for all of it 410), delta_grads 700 us (2048 workgroups of 8 waves, two a SIMD), of which ddecay is some 130: the states
// between the chunks 75 (one of the two in LDS changed nothing, nor did loading them a barrier earlier), the sums of W 37, r and c
// 22.  32 columns a wave halve what is read from LDS, but leave one wave a SIMD (880 in place of 575, both without ddecay's).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "delta_rule.h"
#include "launch.h"
#include "token_util.h"

namespace cssm {

namespace {

constexpr int kBackColumns = 64;   // of a workgroup: 16 for each of its four waves
constexpr int kChunks = kSegment / kChunk;

template <int DKP>
struct BackLds {
  uint4 k[3 * DKP * 4], kt[3 * DKP * 4], qt[3 * DKP * 4], lp[kUnits];
  float gains[256];
};

// float32: one kind of wave for all of it, as the forward's
template <int DKP, bool WIDE>
__global__ __launch_bounds__(256, 1) void delta_walk_back(DeltaRule a) {
  using T = float;
  constexpr int N = 3, PLANE = DKP * 4, KS = DKP / 32, MT = DKP / 16, LP = kUnits / 256;
  __shared__ BackLds<DKP> lds;
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, g = lane / 16;
  const int x = blockIdx.x / a.Hv, h = blockIdx.x - x * a.Hv, hk = h / (a.Hv / a.Hk);
  const int seq = __builtin_amdgcn_readfirstlane(longest_first(a, x));
  const int b = a.offsets ? 0 : seq;
  const Span sp = span_of(a, seq);
  const int chunks = chunks_of(sp.rows);
  const int col = blockIdx.y * kBackColumns + wave * 16 + lane % 16;
  const bool mine = col < a.dv;
  const size_t state = (size_t(seq) * a.Hv + h) * a.dk * a.dv + col;
  const int v_row = a.Hv * a.dv;

  f32x4_t S[MT];   // the state's gradient
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 16 * m + 4 * g + i;
      S[m][i] = a.dh && mine && r < a.dk ? a.dh[state + size_t(r) * a.dv] : 0.0f;
    }

  const int p_tok = tid % 8 + tid / (8 * 2 * KS) * 8, p_at = tid / 8 % (2 * KS);
  const bool p_on = KS == 4 || tid < 64 * KS;
  const int p_col = p_at / 2 * 32 + p_at % 2 * 8;
  const int p_unit = ((p_at / 2 * 2 + p_tok / 16) * 4 + p_at % 2 * 2) * 16 + p_tok % 16;
  const int c_g = tid / (DKP / 2), c_col = tid % (DKP / 2) * 2;
  const bool c_on = DKP == 128 || tid < 2 * DKP;
  const int c_unit = (c_col / 16 * 4 + c_g) * 16 + c_col % 16;
  Piece<T, WIDE> pk;
  Columns<T, WIDE> ck, cq;
  u32x4_t lp[LP];
  float gain;
  uint32_t dy[8];
  const auto fetch = [&](int c) {
    const long long t = sp.row + (long long)c * kChunk;
    const int rows = sp.rows - c * kChunk;
    const Rows k(row_at<T>(a.k, b, t) + hk * a.dk, a.k.row, rows, a.dk), q(row_at<T>(a.q, b, t) + hk * a.dk, a.q.row, rows, a.dk);
    const Rows y(row_at<T>(a.dy, b, t) + h * a.dv, a.dy.row, rows, a.dv);
    const size_t head = size_t(sp.slot + c) * a.Hv + h;
    const u32x4_t* units = reinterpret_cast<const u32x4_t*>(a.units) + head * kUnits + tid;
#pragma unroll
    for (int i = 0; i < 8; ++i) dy[i] = load_element<T>(y, y.at<T, WIDE>(unit_row(4 * g, i), col, a.dv));
    if (p_on) pk.load(k, p_tok, p_col, a.dk);
    if (c_on) ck.load(k, 4 * c_g, c_col, a.dk), cq.load(q, 4 * c_g, c_col, a.dk);
#pragma unroll
    for (int i = 0; i < LP; ++i) lp[i] = units[256 * i];
    gain = a.gains[head * 96 + tid];   // past the 96: the next ones, or the room behind the last
  };
  const auto stash = [&] {
    if (p_on) pk.store(lds.k + p_unit, PLANE);
    if (c_on) ck.store(lds.kt + c_unit, PLANE), cq.store(lds.qt + c_unit, PLANE);
#pragma unroll
    for (int i = 0; i < LP; ++i) lds.lp[tid + 256 * i] = __builtin_bit_cast(uint4, lp[i]);
    lds.gains[tid] = gain;
  };

  if (chunks) {
    fetch(chunks - 1);
    stash();
  }
  for (int c = chunks - 1; c >= 0; --c) {
    __syncthreads();
    float dY[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) dY[i] = element<T>(dy[i]);
    if (c > 0) fetch(c - 1);

    if ((c % kChunks == kChunks - 1 || c == chunks - 1) && mine) {
      float* st = a.dstates + (size_t(sp.segment + c / kChunks) * a.Hv + h) * a.dk * a.dv + col;
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (16 * m + 4 * g + i < a.dk) st[size_t(16 * m + 4 * g + i) * a.dv] = S[m][i];
    }
    f32x4_t ks[2] = {};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const float x[8] = {S[2 * s][0], S[2 * s][1], S[2 * s][2], S[2 * s][3],
                          S[2 * s + 1][0], S[2 * s + 1][1], S[2 * s + 1][2], S[2 * s + 1][3]};
      Unit u[3];
      split<3>(x, u);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        Unit w[N];
        take(lds.k + (s * 2 + t) * 64 + lane, PLANE, w);
        ks[t] = product(w, u, ks[t]);
      }
    }
    float gm[8], dd[8], bt[8], x[8], dU[8], X[8];
    take_rows(lds.gains, g, gm), take_rows(lds.gains + 32, g, dd), take_rows(lds.gains + 64, g, bt);
    {
      Unit u[N];
      split<N>(dY, u);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        Unit w[3];
        take(lds.lp + 3 * 128 + t * 64 + lane, 128, w);
        const f32x4_t py = product(w, u, f32x4_t{});
#pragma unroll
        for (int i = 0; i < 4; ++i) dU[4 * t + i] = py[i] + dd[4 * t + i] * ks[t][i], x[4 * t + i] = bt[4 * t + i] * dU[4 * t + i];
      }
    }
    {
      Unit u[3];
      split<3>(x, u);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        Unit w[3];
        take(lds.lp + t * 64 + lane, 128, w);
        const f32x4_t le = product(w, u, f32x4_t{});
#pragma unroll
        for (int i = 0; i < 4; ++i) X[4 * t + i] = dU[4 * t + i] - le[i];
      }
    }
    {
      const int rows = sp.rows - c * kChunk;
      const size_t head = ((size_t(b) * a.T + sp.row + (long long)c * kChunk) * a.Hv + h) * a.dv;
      const Rows dv(static_cast<T*>(a.dv_out) + head, v_row, rows, a.dv), xx(a.duals + head, v_row, rows, a.dv);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        store_element<T>(dv, dv.at<T, true>(unit_row(4 * g, i), col, a.dv), bt[i] * X[i]);
        store_element<float>(xx, xx.at<float, true>(unit_row(4 * g, i), col, a.dv), X[i]);
      }
    }
    {
      float z[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = a.scale * gm[i] * dY[i], z[i] = -gm[i] * bt[i] * X[i];
      Unit u[3], v[3];
      split<3>(x, u), split<3>(z, v);
      const float all = lds.gains[31];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        Unit w[N];
        S[m] *= all;
        take(lds.qt + m * 64 + lane, PLANE, w);
        S[m] = product(w, u, S[m]);
        take(lds.kt + m * 64 + lane, PLANE, w);
        S[m] = product(w, v, S[m]);
      }
    }
    if (c > 0) {
      __syncthreads();
      stash();
    }
  }
  if (a.dh0 && mine)
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 16 * m + 4 * g + i;
        if (r < a.dk) a.dh0[state + size_t(r) * a.dv] = S[m][i];
      }
}

template <int DKP>
struct BackPairLds {
  static constexpr int kPlane = DKP * 4;
  uint4 k[2][kPlane], kt[2][kPlane], qt[2][kPlane], l[2][3 * 128];
  uint4 py[2][4][2 * 64], gy[2][4][3 * 64], x[2][4][2 * 64];   // for 16 columns each: P^T dY, three parts of scale gamma dY, X
  float gains[4][96];
};

// The same for bfloat16 by two kinds of waves, as the forward's: the first carries the state's gradient, the second brings
// the chunks' rows to LDS, makes what dY alone decides, and writes X and dV of the chunk before.
template <int DKP, bool WIDE>
__global__ __launch_bounds__(512, 1) void delta_back_pairs(DeltaRule a) {
  using T = Bf16;
  constexpr int PLANE = DKP * 4, KS = DKP / 32, MT = DKP / 16;
  __shared__ BackPairLds<DKP> lds;
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64) % 4, g = lane / 16;
  const bool carries = __builtin_amdgcn_readfirstlane(threadIdx.x / 256) == 0;
  const int tid = threadIdx.x % 256;
  const int x = blockIdx.x / a.Hv, h = blockIdx.x - x * a.Hv, hk = h / (a.Hv / a.Hk);
  const int seq = __builtin_amdgcn_readfirstlane(longest_first(a, x));
  const int b = a.offsets ? 0 : seq;
  const Span sp = span_of(a, seq);
  const int chunks = chunks_of(sp.rows);
  const int col = blockIdx.y * kBackColumns + wave * 16 + lane % 16;
  const bool mine = col < a.dv;
  const size_t state = (size_t(seq) * a.Hv + h) * a.dk * a.dv + col;

  // step n is of chunk chunks - 1 - n
  if (carries) {
    f32x4_t S[MT];   // the state's gradient
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 16 * m + 4 * g + i;
        S[m][i] = a.dh && mine && r < a.dk ? a.dh[state + size_t(r) * a.dv] : 0.0f;
      }
    for (int n = 0; n < chunks; ++n) {
      const int c = chunks - 1 - n, o = n % 2;
      __syncthreads();
      const float* gains = lds.gains[n % 4];
      if ((c % kChunks == kChunks - 1 || n == 0) && mine) {
        float* st = a.dstates + (size_t(sp.segment + c / kChunks) * a.Hv + h) * a.dk * a.dv + col;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (16 * m + 4 * g + i < a.dk) st[size_t(16 * m + 4 * g + i) * a.dv] = S[m][i];
      }
      f32x4_t ks[2] = {};
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const float x[8] = {S[2 * s][0], S[2 * s][1], S[2 * s][2], S[2 * s][3],
                            S[2 * s + 1][0], S[2 * s + 1][1], S[2 * s + 1][2], S[2 * s + 1][3]};
        Unit u[3];
        split<3>(x, u);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          Unit w[1];
          take(lds.k[o] + (s * 2 + t) * 64 + lane, PLANE, w);
          ks[t] = product(w, u, ks[t]);
        }
      }
      float gm[8], dd[8], bt[8], x[8], dU[8];
      take_rows(gains, g, gm), take_rows(gains + 32, g, dd), take_rows(gains + 64, g, bt);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const f32x4_t py = __builtin_bit_cast(f32x4_t, lds.py[o][wave][t * 64 + lane]);
#pragma unroll
        for (int i = 0; i < 4; ++i) dU[4 * t + i] = py[i] + dd[4 * t + i] * ks[t][i], x[4 * t + i] = bt[4 * t + i] * dU[4 * t + i];
      }
      {
        Unit u[3];
        split<3>(x, u);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          Unit w[3];
          take(lds.l[o] + t * 64 + lane, 128, w);
          const f32x4_t le = product(w, u, f32x4_t{});
          f32x4_t X;
#pragma unroll
          for (int i = 0; i < 4; ++i) X[i] = dU[4 * t + i] - le[i], x[4 * t + i] = -gm[4 * t + i] * bt[4 * t + i] * X[i];
          lds.x[o][wave][t * 64 + lane] = __builtin_bit_cast(uint4, X);
        }
      }
      {
        Unit u[3], v[3];
        take(lds.gy[o][wave] + lane, 64, u);
        split<3>(x, v);
        const float all = gains[31];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          Unit w[1];
          S[m] *= all;
          take(lds.qt[o] + m * 64 + lane, PLANE, w);
          S[m] = product(w, u, S[m]);
          take(lds.kt[o] + m * 64 + lane, PLANE, w);
          S[m] = product(w, v, S[m]);
        }
      }
    }
    __syncthreads();
    if (a.dh0 && mine)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 16 * m + 4 * g + i;
          if (r < a.dk) a.dh0[state + size_t(r) * a.dv] = S[m][i];
        }
    return;
  }

  const int p_tok = tid % 8 + tid / (8 * 2 * KS) * 8, p_at = tid / 8 % (2 * KS);
  const bool p_on = KS == 4 || tid < 64 * KS;
  const int p_col = p_at / 2 * 32 + p_at % 2 * 8;
  const int p_unit = ((p_at / 2 * 2 + p_tok / 16) * 4 + p_at % 2 * 2) * 16 + p_tok % 16;
  const int c_g = tid / (DKP / 2), c_col = tid % (DKP / 2) * 2;
  const bool c_on = DKP == 128 || tid < 2 * DKP;
  const int c_unit = (c_col / 16 * 4 + c_g) * 16 + c_col % 16;
  Piece<T, WIDE> pk;
  Columns<T, WIDE> ck, cq;
  u32x4_t l[2], p[6];
  f32x4_t gm[2];
  float gain;
  uint32_t dy[8];
  const auto fetch = [&](int n) {
    const int c = chunks - 1 - n, rows = sp.rows - c * kChunk;
    const long long t = sp.row + (long long)c * kChunk;
    const Rows k(row_at<T>(a.k, b, t) + hk * a.dk, a.k.row, rows, a.dk), q(row_at<T>(a.q, b, t) + hk * a.dk, a.q.row, rows, a.dk);
    const Rows y(row_at<T>(a.dy, b, t) + h * a.dv, a.dy.row, rows, a.dv);
    const size_t head = size_t(sp.slot + c) * a.Hv + h;
    const u32x4_t* units = reinterpret_cast<const u32x4_t*>(a.units) + head * kUnits;
#pragma unroll
    for (int i = 0; i < 8; ++i) dy[i] = load_element<T>(y, y.at<T, WIDE>(unit_row(4 * g, i), col, a.dv));
    if (p_on) pk.load(k, p_tok, p_col, a.dk);
    if (c_on) ck.load(k, 4 * c_g, c_col, a.dk), cq.load(q, 4 * c_g, c_col, a.dk);
    l[0] = units[tid], l[1] = units[256 + tid % 128];
#pragma unroll
    for (int i = 0; i < 6; ++i) p[i] = units[3 * 128 + 64 * i + lane];
    const float* gains = a.gains + head * 96;
    gain = gains[tid % 96];
#pragma unroll
    for (int t2 = 0; t2 < 2; ++t2) gm[t2] = *reinterpret_cast<const f32x4_t*>(gains + 16 * t2 + 4 * g);
  };
  const auto stash = [&](int n) {   // what step n takes
    const int o = n % 2;
    if (p_on) pk.store(lds.k[o] + p_unit, PLANE);
    if (c_on) ck.store(lds.kt[o] + c_unit, PLANE), cq.store(lds.qt[o] + c_unit, PLANE);
    lds.l[o][tid] = __builtin_bit_cast(uint4, l[0]);
    if (tid < 128) lds.l[o][256 + tid] = __builtin_bit_cast(uint4, l[1]);
    if (tid < 96) lds.gains[n % 4][tid] = gain;
    float dY[8], x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) dY[i] = element<T>(dy[i]), x[i] = a.scale * gm[i / 4][i % 4] * dY[i];
    Unit u[1], v[3];
    split<1>(dY, u), split<3>(x, v);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const Unit w[3] = {__builtin_bit_cast(Unit, p[t]), __builtin_bit_cast(Unit, p[2 + t]), __builtin_bit_cast(Unit, p[4 + t])};
      lds.py[o][wave][t * 64 + lane] = __builtin_bit_cast(uint4, product(w, u, f32x4_t{}));
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) lds.gy[o][wave][i * 64 + lane] = __builtin_bit_cast(uint4, v[i]);
  };
  if (chunks) {
    fetch(0);
    stash(0);
    if (chunks > 1) fetch(1);
  }
  // step n: step n + 1's operands come in, X and dV of step n - 1 go out
  for (int n = 0; n <= chunks; ++n) {
    __syncthreads();
    if (n + 1 < chunks) stash(n + 1);
    if (n + 2 < chunks) fetch(n + 2);
    if (n == 0) continue;
    const int c = chunks - n, rows = sp.rows - c * kChunk, o = (n - 1) % 2;
    float bt[8];
    take_rows(lds.gains[(n - 1) % 4] + 64, g, bt);
    const size_t head = ((size_t(b) * a.T + sp.row + (long long)c * kChunk) * a.Hv + h) * a.dv;
    const Rows dv(static_cast<T*>(a.dv_out) + head, a.Hv * a.dv, rows, a.dv), xx(a.duals + head, a.Hv * a.dv, rows, a.dv);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const f32x4_t X = __builtin_bit_cast(f32x4_t, lds.x[o][wave][t * 64 + lane]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        store_element<T>(dv, dv.at<T, true>(16 * t + 4 * g + i, col, a.dv), bt[4 * t + i] * X[i]);
        store_element<float>(xx, xx.at<float, true>(16 * t + 4 * g + i, col, a.dv), X[i]);
      }
    }
  }
}

// the value of element i of a lane's unit, all parts together
template <int N>
__device__ __forceinline__ float value_of(const Unit (&u)[N], int i) {
  float v = 0.0f;
#pragma unroll
  for (int n = N - 1; n >= 0; --n) v += __uint_as_float(i % 2 ? u[n].w[i / 2] & 0xffff0000u : u[n].w[i / 2] << 16);
  return v;
}

// sum over 16 lanes side by side, by rotations within them
template <int BY>
__device__ __forceinline__ float rotated(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x120 + BY, 0xf, 0xf, true));
}
__device__ __forceinline__ float sum16(float x) {
  x += rotated<8>(x), x += rotated<4>(x), x += rotated<2>(x);
  return x + rotated<1>(x);
}

// the value `BY` lanes before or behind within 16, 0 beyond them
template <int BY>
__device__ __forceinline__ float lane_before(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x110 + BY, 0xf, 0xf, true));
}
template <int BY>
__device__ __forceinline__ float lane_behind(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x100 + BY, 0xf, 0xf, true));
}
// the sum of the lanes before, or behind, within 16
__device__ __forceinline__ float sum_before(float x) {
  x = lane_before<1>(x);
  x += lane_before<1>(x), x += lane_before<2>(x), x += lane_before<4>(x);
  return x + lane_before<8>(x);
}
__device__ __forceinline__ float sum_behind(float x) {
  x = lane_behind<1>(x);
  x += lane_behind<1>(x), x += lane_behind<2>(x), x += lane_behind<4>(x);
  return x + lane_behind<8>(x);
}

// P: dk and dv up to it.  One workgroup for 128 rows of one value head, P / 16 waves.  Y, Z and their transposes take the place
// of U's rows in LDS once those are read, and the columns of d U that of X's rows.
// 64 wide two workgroups share a CU, in 256 registers a thread (training 4 x 4096 x 16 heads of 64: bfloat16 452 -> 281 us,
// float32 519 -> 444); 128 wide that leaves 128 registers, which spill (1280 us in place of 575, without ddecay's terms).  As it
// is it spills too: bfloat16 10 and 17 registers (64 and 128 wide), float32 53 and 63, 128 wide off the vector width 144 and 172.
template <int P, typename T, bool WIDE>
__global__ __launch_bounds__(4 * P, P == 64 && WIDE ? 2 : 1) void delta_grads(DeltaRule a) {
  constexpr int N = PartsOf<T>::n, W = P / 16, KS = P / 32, MT = P / 16, PLANE = P * 4, TASKS = (6 + W - 1) / W;
  constexpr int UROOM = 3 * PLANE > 12 * 128 ? 3 * PLANE : 12 * 128;
  __shared__ uint4 s_y[N * PLANE], s_x[3 * PLANE], s_u[UROOM], s_kt[N * PLANE], s_qt[N * PLANE];
  __shared__ __attribute__((aligned(16))) float s_gains[kChunks][96];
  constexpr int PAIRS = W < 6 ? W : 6;   // waves that have tiles of Y and Z
  // ddecay's terms, by waves: W_ij that cross each row, r, c and gamma_31 <S, dS'>
  __shared__ float s_pairs[PAIRS][kSegment], s_read[W][kSegment], s_write[W][kSegment], s_whole[W][kChunks];
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, g = lane / 16, h = blockIdx.y, hk = h / (a.Hv / a.Hk);
  const bool shared = a.Hv != a.Hk;
  int seq, seg, b = 0;
  if (!a.offsets) {
    const int n = segments_of(a.T);
    seq = b = blockIdx.x / n, seg = blockIdx.x - seq * n;
  } else {
    int lo = 0, hi = a.nseq;   // the last sequence whose segments begin at or before this slot
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (span_of(a, mid).segment <= int(blockIdx.x)) lo = mid;
      else hi = mid;
    }
    seq = lo, seg = blockIdx.x - span_of(a, lo).segment;
  }
  const Span sp = span_of(a, seq);
  if (seg < 0 || seg >= segments_of(sp.rows)) return;
  const int row0 = sp.row + seg * kSegment;
  const int left = sp.rows - seg * kSegment, rows_all = left < kSegment ? left : kSegment, chunks = chunks_of(rows_all);
  const size_t slot0 = size_t(sp.slot) + size_t(seg) * kChunks;
  const int col = wave * 16 + lane % 16;   // of the keys
  const int v_row = a.Hv * a.dv;
  for (int i = tid; i < chunks * 96; i += 4 * P) s_gains[i / 96][i % 96] = a.gains[((slot0 + i / 96) * a.Hv + h) * 96 + i % 96];

  // S^T, or its gradient's: rows of dv, a lane one column of dk
  f32x4_t S[MT];
  const auto load_state = [&](const float* from, f32x4_t (&to)[MT]) {
    const Rows p(from + ((size_t(sp.segment + seg) * a.Hv + h) * a.dk + wave * 16) * a.dv, a.dv, a.dk - wave * 16, a.dv);
#pragma unroll
    for (int m = 0; m < MT; ++m)
      if constexpr (WIDE) {
        to[m] = __builtin_bit_cast(f32x4_t, load16(p, p.at<float, true>(lane % 16, 16 * m + 4 * g, a.dv)));
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) to[m][i] = element<float>(load_element<float>(p, p.at<float, false>(lane % 16, 16 * m + 4 * g + i, a.dv)));
      }
  };
  load_state(a.states, S);
  f32x4_t* passed = reinterpret_cast<f32x4_t*>(a.passed) + ((size_t(sp.segment + seg) * a.Hv + h) * 2 * W + wave) * MT * 64 + lane;

  // each half of the threads takes about half of the splitting
  const bool first = tid < 2 * P;
  const int id = first ? tid : tid - 2 * P;
  const int p_tok = id % 8 + id / (8 * 2 * KS) * 8, p_at = id / 8 % (2 * KS), p_col = p_at / 2 * 32 + p_at % 2 * 8;
  const int p_unit = ((p_at / 2 * 2 + p_tok / 16) * 4 + p_at % 2 * 2) * 16 + p_tok % 16;
  const int c_g = id / (P / 2), c_col = id % (P / 2) * 2, c_unit = (c_col / 16 * 4 + c_g) * 16 + c_col % 16;
  const auto head_of = [&](int c) { return ((size_t(b) * a.T + row0 + c * kChunk) * a.Hv + h) * a.dv; };

  {
    Piece<float, WIDE> px, pe;
    Columns<float, WIDE> ce;
    Piece<T, WIDE> py;
    Columns<T, WIDE> ck, cq;
    const auto fetch = [&](int c) {
      const int rows = rows_all - c * kChunk;
      const long long t = row0 + c * kChunk;
      if (first) {
        const Rows x(a.duals + head_of(c), v_row, rows, a.dv), e(a.errors + head_of(c), v_row, rows, a.dv);
        px.load(x, p_tok, p_col, a.dv), pe.load(e, p_tok, p_col, a.dv);
        const Rows q(row_at<T>(a.q, b, t) + hk * a.dk, a.q.row, rows, a.dk);
        cq.load(q, 4 * c_g, c_col, a.dk);
        asm volatile("");   // the halves' ends stay apart: joined, their values lie in scratch
      } else {
        const Rows e(a.errors + head_of(c), v_row, rows, a.dv), y(row_at<T>(a.dy, b, t) + h * a.dv, a.dy.row, rows, a.dv);
        const Rows k(row_at<T>(a.k, b, t) + hk * a.dk, a.k.row, rows, a.dk);
        ce.load(e, 4 * c_g, c_col, a.dv);
        py.load(y, p_tok, p_col, a.dv);
        ck.load(k, 4 * c_g, c_col, a.dk);
      }
    };
    fetch(0);
    for (int c = 0; c < chunks; ++c) {
      const int rows = rows_all - c * kChunk;
      __syncthreads();
      const float* gains = s_gains[c];
      if (first) {
        const float beta = gains[64 + p_tok];
        px.template store_by<3>(beta, s_x + p_unit, PLANE);
        pe.template store_by<3>(beta, s_u + p_unit, PLANE);
        cq.store(s_qt + c_unit, PLANE);
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) dot = fmaf(px.get(i), pe.get(i), dot);
#pragma unroll
        for (int o = 8; o < 16 * KS; o *= 2) dot += __shfl_xor(dot, o);
        if (p_at == 0 && p_tok < rows) a.dbeta[(size_t(b) * a.T + row0 + c * kChunk + p_tok) * a.Hv + h] = dot;
      } else {
        py.store(s_y + p_unit, PLANE);
        ck.store(s_kt + c_unit, PLANE);
      }
      __syncthreads();

      if (a.ddecay && c > 0 && c + 1 < chunks)
#pragma unroll
        for (int m = 0; m < MT; ++m) passed[((c - 1) * W * MT + m) * 64] = S[m];
      // Y and Z, a 16 x 16 tile a wave: (0, 0), (1, 0) and (1, 1) of both
      f32x4_t tile[TASKS];
      float across[2] = {0.0f, 0.0f};   // W's sums for l = lane % 16 and 16 more
#pragma unroll
      for (int n = 0; n < TASKS; ++n) {
        const int task = wave + n * W, z = task / 3, ti = task % 3 > 0, tj = task % 3 == 2;
        tile[n] = f32x4_t{};
        if (task < 6) {
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            Unit u[3];
            take(s_u + (s * 2 + tj) * 64 + lane, PLANE, u);
            if (z) {
              Unit w[3];
              take(s_x + (s * 2 + ti) * 64 + lane, PLANE, w);
              tile[n] = product(w, u, tile[n]);
            } else {
              Unit w[N];
              take(s_y + (s * 2 + ti) * 64 + lane, PLANE, w);
              tile[n] = product(w, u, tile[n]);
            }
          }
          const float* D = a.decays + ((slot0 + c) * a.Hv + h) * kDecays + 16 * tj + lane % 16;
          if (a.ddecay) {
            const float* M = D + (z ? 2 : 1) * kChunk * kChunk;
            const int l = lane % 16;
            float e[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) e[i] = (z ? -tile[n][i] : tile[n][i]) * M[(16 * ti + 4 * g + i) * kChunk];
            if (ti == tj) {   // rows from l on, columns before l
              float sum = 0.0f;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float before = sum_before(e[i]);
                sum += 4 * g + i >= l ? before : 0.0f;
              }
              if (ti) across[1] += sum;
              else across[0] += sum;
            } else {   // all rows and columns before l; rows from l on and all columns
              across[0] += sum_before((e[0] + e[1]) + (e[2] + e[3]));
              float sum = 0.0f;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float row = sum16(e[i]);
                sum += 4 * g + i >= l ? row : 0.0f;
              }
              across[1] += sum;
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = 16 * ti + 4 * g + i;
            tile[n][i] *= z ? (r == 16 * tj + lane % 16 ? 0.0f : D[r * kChunk]) : a.scale * D[r * kChunk];
          }
        }
      }
      if (a.ddecay && wave < PAIRS) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          across[i] += __shfl_xor(across[i], 16), across[i] += __shfl_xor(across[i], 32);
          if (g == i) s_pairs[wave][c * kChunk + lane] = across[i];
        }
      }
      f32x4_t ys[2] = {}, xs[2] = {};
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const float x[8] = {S[2 * s][0], S[2 * s][1], S[2 * s][2], S[2 * s][3],
                            S[2 * s + 1][0], S[2 * s + 1][1], S[2 * s + 1][2], S[2 * s + 1][3]};
        Unit u[3];
        split<3>(x, u);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          Unit w[N], w3[3];
          take(s_y + (s * 2 + t) * 64 + lane, PLANE, w);
          ys[t] = product(w, u, ys[t]);
          take(s_x + (s * 2 + t) * 64 + lane, PLANE, w3);
          xs[t] = product(w3, u, xs[t]);
        }
      }
      __syncthreads();   // U's rows are read: Y, Z, Y^T and Z^T take their place, 3 parts of 128 units each; X's: d U's columns
      if (!first) {
        float by[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) by[j] = gains[64 + unit_row(4 * c_g, j)] * gains[32 + unit_row(4 * c_g, j)];
        ce.template store_by<3>(by, s_x + c_unit, PLANE);
      }
#pragma unroll
      for (int n = 0; n < TASKS; ++n) {
        const int task = wave + n * W, z = task / 3, ti = task % 3 > 0, tj = task % 3 == 2;
        if (task < 6) {
          const float v[8] = {tile[n][0], tile[n][1], tile[n][2], tile[n][3], 0.0f, 0.0f, 0.0f, 0.0f};
          Unit u[3];
          split<3>(v, u);
          uint16_t* rows16 = reinterpret_cast<uint16_t*>(s_u + z * 3 * 128);
          uint2* turned = reinterpret_cast<uint2*>(s_u + (2 + z) * 3 * 128);
          const int j = lane % 16;
#pragma unroll
          for (int p = 0; p < 3; ++p) {
            // row 16 ti + 4 g + i, column 16 tj + j: unit (ti, j / 4, row), place 4 tj + j % 4
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint16_t* at = rows16 + (p * 128 + ti * 64 + j / 4 * 16 + 4 * g + i) * 8 + j % 4;
              at[4 * tj] = uint16_t(u[p].w[i / 2] >> (i % 2 * 16));
              if (ti == 0) at[4] = 0;                            // tile (0, 1)
            }
            // turned: row 16 tj + j, columns 16 ti + 4 g + 0 .. 3: unit (tj, g, j), places 4 ti ..
            uint2* at = turned + (p * 128 + tj * 64 + g * 16 + j) * 2;
            at[ti] = make_uint2(u[p].w[0], u[p].w[1]);
            if (tj == 1) at[0] = make_uint2(0u, 0u);
          }
        }
      }
      __syncthreads();
      if (c + 1 < chunks) fetch(c + 1);
      Unit kb[N], qb[N];
      take(s_kt + wave * 64 + lane, PLANE, kb);
      take(s_qt + wave * 64 + lane, PLANE, qb);
      float gm[8], dq[8], rd[8], wr[8];
      take_rows(gains, g, gm);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        Unit w[3];
#pragma unroll
        for (int i = 0; i < 4; ++i) ys[t][i] *= a.scale * gm[4 * t + i], xs[t][i] *= gm[4 * t + i];
        if (a.ddecay) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float read = sum16(fmaf(value_of(qb, 4 * t + i), ys[t][i], -value_of(kb, 4 * t + i) * xs[t][i]));
            if (lane % 16 == 0) s_read[wave][c * kChunk + 16 * t + 4 * g + i] = read;
          }
        }
        f32x4_t yq = {}, zk = {};
        take(s_u + t * 64 + lane, 128, w);
        ys[t] = product(w, kb, ys[t]);
        take(s_u + 384 + t * 64 + lane, 128, w);
        xs[t] = product(w, kb, xs[t]);
        take(s_u + 768 + t * 64 + lane, 128, w);
        yq = product(w, qb, yq);
        take(s_u + 1152 + t * 64 + lane, 128, w);
        zk = product(w, kb, zk);
#pragma unroll
        for (int i = 0; i < 4; ++i) dq[4 * t + i] = ys[t][i], rd[4 * t + i] = -xs[t][i], wr[4 * t + i] = yq[i] - zk[i];
      }
      const float all = gains[31];
      if (c + 1 < chunks) {   // the state before the last chunk stays
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          Unit w[3];
          take(s_x + m * 64 + lane, PLANE, w);
          S[m] = product(w, kb, S[m] * all);
        }
      }
      const size_t at_row = size_t(b) * a.T + row0 + c * kChunk;
      const Rows dkh(a.dk_heads + (at_row * a.Hv + h) * a.dk, a.Hv * a.dk, rows, a.dk);
      const Rows dqh(shared ? a.dq_heads + (at_row * a.Hv + h) * a.dk : nullptr, a.Hv * a.dk, shared ? rows : 0, a.dk);
      const Rows dqo(static_cast<T*>(a.dq) + (at_row * a.Hk + hk) * a.dk, a.Hk * a.dk, shared ? 0 : rows, a.dk);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = unit_row(4 * g, i);
        store_element<float>(dkh, dkh.at<float, true>(r, col, a.dk), rd[i] + wr[i]);
        if (shared) store_element<float>(dqh, dqh.at<float, true>(r, col, a.dk), dq[i]);
        else store_element<T>(dqo, dqo.at<T, true>(r, col, a.dk), dq[i]);
      }
    }
  }

  {
    Piece<float, WIDE> pe;
    Columns<float, WIDE> cx;
    Columns<T, WIDE> cy, ck, cq;
    float part[8];
    const auto fetch = [&](int c) {
      const int rows = rows_all - c * kChunk;
      const long long t = row0 + c * kChunk;
      const size_t at_row = size_t(b) * a.T + t;
      const Rows dkh(a.dk_heads + (at_row * a.Hv + h) * a.dk, a.Hv * a.dk, rows, a.dk);
#pragma unroll
      for (int i = 0; i < 8; ++i) part[i] = element<float>(load_element<float>(dkh, dkh.at<float, true>(unit_row(4 * g, i), col, a.dk)));
      if (first) {
        const Rows e(a.errors + head_of(c), v_row, rows, a.dv);
        const Rows k(row_at<T>(a.k, b, t) + hk * a.dk, a.k.row, rows, a.dk), q(row_at<T>(a.q, b, t) + hk * a.dk, a.q.row, rows, a.dk);
        pe.load(e, p_tok, p_col, a.dv);
        ck.load(k, 4 * c_g, c_col, a.dk), cq.load(q, 4 * c_g, c_col, a.dk);
        asm volatile("");
      } else {
        const Rows x(a.duals + head_of(c), v_row, rows, a.dv), y(row_at<T>(a.dy, b, t) + h * a.dv, a.dy.row, rows, a.dv);
        cx.load(x, 4 * c_g, c_col, a.dv);
        cy.load(y, 4 * c_g, c_col, a.dv);
      }
    };
    fetch(chunks - 1);
    const auto whole = [&](int c, const f32x4_t (&x)[MT], const f32x4_t (&y)[MT]) {   // gamma_31 <x, y>
      float with = 0.0f;
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) with = fmaf(x[m][i], y[m][i], with);
#pragma unroll
      for (int o = 1; o < 64; o *= 2) with += __shfl_xor(with, o);
      if (lane == 0) s_whole[wave][c] = s_gains[c][31] * with;
    };
    {
      f32x4_t end[MT];
      load_state(a.dstates, end);
      if (a.ddecay) whole(chunks - 1, S, end);
#pragma unroll
      for (int m = 0; m < MT; ++m) S[m] = end[m];
    }
    for (int c = chunks - 1; c >= 0; --c) {
      const int rows = rows_all - c * kChunk;
      __syncthreads();
      const float* gains = s_gains[c];
      if (first) {
        pe.template store_by<3>(gains[64 + p_tok], s_u + p_unit, PLANE);
        ck.store(s_kt + c_unit, PLANE), cq.store(s_qt + c_unit, PLANE);
      } else {
        float by[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) by[j] = -gains[64 + unit_row(4 * c_g, j)] * gains[unit_row(4 * c_g, j)];
        cx.template store_by<3>(by, s_x + c_unit, PLANE);
        cy.store(s_y + c_unit, PLANE);
      }
      float before[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) before[i] = part[i];
      __syncthreads();
      if (c > 0) fetch(c - 1);
      if (a.ddecay && c + 1 < chunks) {   // with the state before this chunk
        f32x4_t start[MT];
        if (c == 0) {
          load_state(a.states, start);
        } else {
#pragma unroll
          for (int m = 0; m < MT; ++m) start[m] = passed[((c - 1) * W * MT + m) * 64];
        }
        whole(c, start, S);
      }
      f32x4_t us[2] = {};
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const float x[8] = {S[2 * s][0], S[2 * s][1], S[2 * s][2], S[2 * s][3],
                            S[2 * s + 1][0], S[2 * s + 1][1], S[2 * s + 1][2], S[2 * s + 1][3]};
        Unit u[3];
        split<3>(x, u);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          Unit w[3];
          take(s_u + (s * 2 + t) * 64 + lane, PLANE, w);
          us[t] = product(w, u, us[t]);
        }
      }
      Unit kb[N], qb[N];
      take(s_kt + wave * 64 + lane, PLANE, kb);
      take(s_qt + wave * 64 + lane, PLANE, qb);
      float gm[8];
      take_rows(gains, g, gm);
#pragma unroll
      for (int i = 0; i < 8; ++i) gm[i] *= a.scale * value_of(qb, i);
      Unit qg[3];   // scale gamma q: a wave's 16 columns of q to split, not all columns of dy
      split<3>(gm, qg);
      const float all = gains[31];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        Unit w[3], y[N];
        S[m] *= all;
        take(s_y + m * 64 + lane, PLANE, y);
        S[m] = product(y, qg, S[m]);
        take(s_x + m * 64 + lane, PLANE, w);
        S[m] = product(w, kb, S[m]);
      }
      float dd[8];
      take_rows(gains + 32, g, dd);
      const size_t at_row = size_t(b) * a.T + row0 + c * kChunk;
      const Rows dkh(a.dk_heads + (at_row * a.Hv + h) * a.dk, a.Hv * a.dk, rows, a.dk);
      const Rows dko(static_cast<T*>(a.dkey) + (at_row * a.Hk + hk) * a.dk, a.Hk * a.dk, shared ? 0 : rows, a.dk);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = unit_row(4 * g, i);
        const float w = dd[i] * us[i / 4][i % 4];
        if (shared) store_element<float>(dkh, dkh.at<float, true>(r, col, a.dk), before[i] + w);
        else store_element<T>(dko, dko.at<T, true>(r, col, a.dk), before[i] + w);
        if (a.ddecay) {
          const float write = sum16(value_of(kb, i) * w);
          if (lane % 16 == 0) s_write[wave][c * kChunk + r] = write;
        }
      }
    }
  }
  __syncthreads();
  if (a.ddecay && wave == 0) {
    float pairs[2], read[2], write[2], over = 0.0f;   // of rows 2 l and 2 l + 1, 16 lanes a chunk
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = 2 * lane + i;
      pairs[i] = read[i] = write[i] = 0.0f;
      if (r < rows_all) {
#pragma unroll
        for (int w = 0; w < PAIRS; ++w) pairs[i] += s_pairs[w][r];
#pragma unroll
        for (int w = 0; w < W; ++w) read[i] += s_read[w][r], write[i] += s_write[w][r];
      }
    }
    if (lane / 16 < chunks)
#pragma unroll
      for (int w = 0; w < W; ++w) over += s_whole[w][lane / 16];
    const float behind = sum_behind(read[0] + read[1]) + over, before = sum_before(write[0] + write[1]);
    float* out = a.ddecay + (size_t(b) * a.T + row0) * a.Hv + h;
    if (2 * lane < rows_all) out[size_t(2 * lane) * a.Hv] = pairs[0] + (behind + read[0] + read[1]) + before;
    if (2 * lane + 1 < rows_all) out[size_t(2 * lane + 1) * a.Hv] = pairs[1] + (behind + read[1]) + (before + write[0]);
  }
}

// the value heads' shares of dq and dk added up
template <typename T>
__global__ __launch_bounds__(256) void delta_share(const float* q, const float* k, size_t rows, int Hk, int G, int dk, T* dq, T* dkey) {
  const size_t n = rows * Hk * dk;
  for (size_t at = size_t(blockIdx.x) * 256 + threadIdx.x; at < n; at += size_t(gridDim.x) * 256) {
    const size_t head = at / dk, from = head * G * dk + (at - head * dk);
    float x = 0.0f, y = 0.0f;
    for (int i = 0; i < G; ++i) x += q[from + size_t(i) * dk], y += k[from + size_t(i) * dk];
    put(dq + at, x), put(dkey + at, y);
  }
}

// zero behind the last sequence
template <typename T>
__global__ __launch_bounds__(256) void delta_tail(DeltaRule a) {
  const Span sp = span_of(a, a.nseq - 1);
  const int nk = a.Hk * a.dk, nv = a.Hv * a.dv;
  for (int t = sp.row + sp.rows + blockIdx.x; t < a.T; t += gridDim.x) {
    for (int i = threadIdx.x; i < nk; i += 256) {
      put(static_cast<T*>(a.dq) + size_t(t) * nk + i, 0.0f);
      put(static_cast<T*>(a.dkey) + size_t(t) * nk + i, 0.0f);
    }
    for (int i = threadIdx.x; i < nv; i += 256) put(static_cast<T*>(a.dv_out) + size_t(t) * nv + i, 0.0f);
    for (int i = threadIdx.x; i < a.Hv; i += 256) {
      a.dbeta[size_t(t) * a.Hv + i] = 0.0f;
      if (a.ddecay) a.ddecay[size_t(t) * a.Hv + i] = 0.0f;
    }
  }
}

template <typename T, bool WIDE>
void run_as(const DeltaRule& a, hipStream_t s) {
  const int n = a.offsets ? a.nseq : a.B, segments = int(delta_rule_segments(a.B, a.T, a.nseq, a.offsets != nullptr));
  launch_delta_prepare<T, true>(a, WIDE, s);
  const dim3 grid(n * a.Hv, (a.dv + kBackColumns - 1) / kBackColumns);
  if constexpr (sizeof(T) == 2) {
    if (a.dk <= 64) delta_back_pairs<64, WIDE><<<grid, 512, 0, s>>>(a);
    else delta_back_pairs<128, WIDE><<<grid, 512, 0, s>>>(a);
  } else {
    if (a.dk <= 64) delta_walk_back<64, WIDE><<<grid, 256, 0, s>>>(a);
    else delta_walk_back<128, WIDE><<<grid, 256, 0, s>>>(a);
  }
  if (!a.T) return;
  if (a.dk <= 64 && a.dv <= 64) delta_grads<64, T, WIDE><<<dim3(segments, a.Hv), 256, 0, s>>>(a);
  else delta_grads<128, T, WIDE><<<dim3(segments, a.Hv), 512, 0, s>>>(a);
  const size_t rows = size_t(a.B) * a.T, groups = (rows * a.Hk * a.dk + 255) / 256;
  if (a.Hv != a.Hk)
    delta_share<T><<<unsigned(groups < 1 << 16 ? groups : 1 << 16), 256, 0, s>>>(a.dq_heads, a.dk_heads, rows, a.Hk, a.Hv / a.Hk,
                                                                              a.dk, static_cast<T*>(a.dq), static_cast<T*>(a.dkey));
  if (a.offsets) delta_tail<T><<<a.T < 1024 ? a.T : 1024, 256, 0, s>>>(a);
}

template <typename T>
void run(const DeltaRule& a, hipStream_t s) {
  const bool wide = wide_rows<T>(a.q, a.Hk, a.dk) && wide_rows<T>(a.k, a.Hk, a.dk) && wide_rows<T>(a.dy, a.Hv, a.dv) &&
                    reinterpret_cast<uintptr_t>(a.errors) % 16 == 0;
  if (wide) run_as<T, true>(a, s);
  else run_as<T, false>(a, s);
}

size_t up16(size_t n) { return (n + 15) / 16 * 16; }

}  // namespace

size_t delta_rule_bwd_workspace(int B, int T, int Hk, int Hv, int dk, int dv, int nseq, bool packed) {
  const size_t heads = size_t(delta_rule_slots(B, T, nseq, packed)) * Hv, rows = size_t(B) * T * Hv;
  const size_t segments = size_t(delta_rule_segments(B, T, nseq, packed)) * Hv, wide = dk <= 64 && dv <= 64 ? 64 : 128;
  return heads * (kUnits * sizeof(uint4) + (96 + kDecays) * sizeof(float)) + 256 * sizeof(float) +
         up16(rows * dv * sizeof(float)) + up16(segments * dk * dv * sizeof(float)) + segments * 2 * wide * wide * sizeof(float) +
         up16(rows * dk * sizeof(float)) * (Hv != Hk ? 2 : 1);
}

hipError_t launch_delta_rule_bwd(DeltaRule a, int dtype, void* workspace, hipStream_t s) {
  const bool packed = a.offsets != nullptr;
  const size_t heads = size_t(delta_rule_slots(a.B, a.T, a.nseq, packed)) * a.Hv, rows = size_t(a.B) * a.T * a.Hv;
  char* at = static_cast<char*>(workspace);
  const auto room = [&](size_t bytes) {
    char* p = at;
    at += up16(bytes);
    return p;
  };
  a.units = reinterpret_cast<uint4*>(room(heads * kUnits * sizeof(uint4)));
  a.gains = reinterpret_cast<float*>(room((heads * 96 + 256) * sizeof(float)));   // 160 more behind the last are read
  a.decays = reinterpret_cast<float*>(room(heads * kDecays * sizeof(float)));
  a.duals = reinterpret_cast<float*>(room(rows * a.dv * sizeof(float)));
  const size_t segments = size_t(delta_rule_segments(a.B, a.T, a.nseq, packed)) * a.Hv, wide = a.dk <= 64 && a.dv <= 64 ? 64 : 128;
  a.dstates = reinterpret_cast<float*>(room(segments * a.dk * a.dv * sizeof(float)));
  a.passed = reinterpret_cast<float*>(room(segments * 2 * wide * wide * sizeof(float)));
  a.dk_heads = reinterpret_cast<float*>(room(rows * a.dk * sizeof(float)));
  a.dq_heads = a.Hv != a.Hk ? reinterpret_cast<float*>(room(rows * a.dk * sizeof(float))) : nullptr;
  if (dtype == 0) run<float>(a, s);
  else run<Bf16>(a, s);
  return hipGetLastError();
}

}  // namespace cssm
