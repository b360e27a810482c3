// The gated delta rule over token sequences (gfx950).  For each value head, S (dk, dv) the state, a = exp(decay):
//   e_t = v_t - a_t S_{t-1}^T k_t,  S_t = a_t S_{t-1} + k_t (beta_t e_t)^T,  y_t = scale S_t^T q_t
// G value heads next to each other share one query and key head.
//
// In chunks of 32 rows, with D_ij = a_{j+1} .. a_i (i >= j), gamma_i = a_0 .. a_i and d_j = D_31,j, all as products, so
// that no difference of large sums enters and a = 0 is just that:
//   A_ij = D_ij k_i.k_j (i > j),  P_ij = scale D_ij q_i.k_j (i >= j),  L = (1 + A beta)^-1 A   (from the rows above, in order)
//   R = V - gamma K S,  E = R - L beta R,  Y = scale gamma Q S + P beta E,  S <- gamma_31 S + K^T (d beta E)
// delta_prepare computes L and P of all chunks at once; delta_walk then carries S from chunk to chunk, a wave 16 of
// the state's columns, which lie in its registers as the result of one product and the operand of the next.
// The state is float32 and enters its products in three bfloat16 parts (csrc/delta_rule.h), as do L, P, R and U: y is rounded
// once, where it is stored.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "delta_rule.h"
#include "launch.h"
#include "token_util.h"

namespace cssm {

namespace {

typedef float f32x16_t __attribute__((ext_vector_type(16)));

constexpr int kPad = kChunk + 4;

// two results above each other as the parts of the next product's second operand
__device__ __forceinline__ void split_pair(f32x4_t above, f32x4_t below, Unit (&u)[3]) {
  const float x[8] = {above[0], above[1], above[2], above[3], below[0], below[1], below[2], below[3]};
  split<3>(x, u);
}

// the 8 values of a row from `at` on, in their parts
template <typename T, bool WIDE>
__device__ __forceinline__ void load_unit(const Rows& m, int row, int at, int n, Unit (&u)[PartsOf<T>::n]) {
  float v[8];
  if constexpr (WIDE) {
    const uint32_t o = m.at<T, true>(row, at, n);
    const uint4 q = load16(m, o);
    if constexpr (sizeof(T) == 2) {
      u[0] = __builtin_bit_cast(Unit, q);
    } else {
      const uint4 r = load16(m, o + 16);
      v[0] = __uint_as_float(q.x), v[1] = __uint_as_float(q.y), v[2] = __uint_as_float(q.z), v[3] = __uint_as_float(q.w);
      v[4] = __uint_as_float(r.x), v[5] = __uint_as_float(r.y), v[6] = __uint_as_float(r.z), v[7] = __uint_as_float(r.w);
      split<3>(v, u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = element<T>(load_element<T>(m, m.at<T, false>(row, at + i, n)));
    split<PartsOf<T>::n>(v, u);
  }
}

template <int N>
__device__ __forceinline__ f32x16_t product32(const Unit (&a)[N], const Unit (&b)[N], f32x16_t c) {
#pragma unroll
  for (int s = N - 1; s >= 0; --s)
#pragma unroll
    for (int i = 0; i <= s; ++i)
      c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a[i]), __builtin_bit_cast(bf16x8_t, b[s - i]), c, 0, 0, 0);
  return c;
}

// The chunk that a slot of the workspace stands for; false for a slot that no chunk takes
__device__ __forceinline__ bool chunk_at(const DeltaRule& a, int slot, int& b, int& row, int& rows) {
  b = 0;
  if (!a.offsets) {
    const int n = chunks_of(a.T);
    b = slot / n;
    row = (slot - b * n) * kChunk, rows = a.T - row;
  } else {
    int lo = 0, hi = a.nseq;   // the last sequence whose chunks begin at or before this slot
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (span_of(a, mid).slot <= slot) lo = mid;
      else hi = mid;
    }
    const Span sp = span_of(a, lo);
    const int c = slot - sp.slot;
    if (c < 0 || c >= chunks_of(sp.rows)) return false;
    row = sp.row + c * kChunk, rows = sp.rows - c * kChunk;
  }
  if (rows > kChunk) rows = kChunk;
  return true;
}

// One wave for a chunk of two value heads: K K^T and Q K^T of their key heads (one, or two), then one value head in each
// half of the wave, a column of its 32 x 32 a lane: decays, L row by row, and both written as first operands (TURNED: their
// transposes, which the adjoint takes).  What bounds it is the 500 multiplications in a row behind L and the traffic through
// LDS between the layouts; four waves a SIMD hide most of their latencies.
template <int DKP, typename T, bool WIDE, bool TURNED>
__global__ __launch_bounds__(64, sizeof(T) == 2 ? 4 : 2) void delta_prepare(DeltaRule a) {
  __shared__ __attribute__((aligned(16))) float s_m[2][kChunk * kPad];
  __shared__ float s_alpha[2][kChunk];
  const int lane = threadIdx.x, j = lane % 32, half = lane / 32, G = a.Hv / a.Hk, h0 = 2 * blockIdx.y, h = h0 + half;
  const int slot = blockIdx.x;
  int b, row, rows;
  if (!chunk_at(a, slot, b, row, rows)) return;
  const bool two = h0 + 1 < a.Hv, on = half == 0 || two;
  const int hk[2] = {h0 / G, (two ? h0 + 1 : h0) / G};
  float beta = 0.0f, alpha = 1.0f;
  if (on && j < rows) {
    beta = row_at<float>(a.beta, b, row + j)[h];
    if (a.decay.p) alpha = expf(row_at<float>(a.decay, b, row + j)[h]);
  }
  s_alpha[half][j] = alpha;
  float A[kChunk], P[kChunk];
  const Rows k[2] = {Rows(row_at<T>(a.k, b, row) + hk[0] * a.dk, a.k.row, rows, a.dk), Rows(row_at<T>(a.k, b, row) + hk[1] * a.dk, a.k.row, rows, a.dk)};
  const Rows q[2] = {Rows(row_at<T>(a.q, b, row) + hk[0] * a.dk, a.q.row, rows, a.dk), Rows(row_at<T>(a.q, b, row) + hk[1] * a.dk, a.q.row, rows, a.dk)};
  {
    f32x16_t qk[2];
#pragma unroll
    for (int o = 0; o < 2; ++o) {
      f32x16_t kk = {}, x = {};
      if (o == 0 || hk[1] != hk[0]) {
        // all of a head's loads at once: one after the other they would take longer than everything else
        Unit uk[DKP / 16][PartsOf<T>::n], uq[DKP / 16][PartsOf<T>::n];
#pragma unroll
        for (int i = 0; i < DKP / 16; ++i) load_unit<T, WIDE>(k[o], j, 16 * i + 8 * half, a.dk, uk[i]), load_unit<T, WIDE>(q[o], j, 16 * i + 8 * half, a.dk, uq[i]);
#pragma unroll
        for (int i = 0; i < DKP / 16; ++i) kk = product32(uk[i], uk[i], kk), x = product32(uq[i], uk[i], x);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int at = (8 * (i / 4) + 4 * half + i % 4) * kPad + j;
          s_m[o][at] = kk[i];
          if (o == 0) s_m[1][at] = kk[i];   // of the second head too, unless it is of another key
        }
        qk[o] = x;
      } else {
        qk[1] = qk[0];
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kChunk; ++i) A[i] = s_m[half][i * kPad + j];
    __syncthreads();
#pragma unroll
    for (int o = 0; o < 2; ++o)
#pragma unroll
      for (int i = 0; i < 16; ++i) s_m[o][(8 * (i / 4) + 4 * half + i % 4) * kPad + j] = qk[o][i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kChunk; ++i) P[i] = s_m[half][i * kPad + j];
    __syncthreads();
  }
  float d = 0.0f;
#pragma unroll
  for (int i = 0; i < kChunk; ++i) {
    const bool at = i == j;
    d = at ? 1.0f : d * s_alpha[half][i];   // 0 above the diagonal
    A[i] = at ? 0.0f : d * A[i];
    P[i] *= d * a.scale;
    if (TURNED && on) {
      float* to = a.decays + (size_t(slot) * a.Hv + h) * kDecays + i * kChunk + j;
      to[0] = d;
      if (a.decay.p) to[kChunk * kChunk] = P[i], to[2 * kChunk * kChunk] = A[i];
    }
    s_m[half][i * kPad + j] = A[i] * beta;
  }
  float gamma = alpha;   // of this row and those before it in the chunk
#pragma unroll
  for (int o = 1; o < kChunk; o *= 2) {
    const float before = __shfl_up(gamma, o, kChunk);
    if (j >= o) gamma *= before;
  }
  if (on) {
    float* g = a.gains + (size_t(slot) * a.Hv + h) * 96;
    g[j] = gamma, g[32 + j] = d, g[64 + j] = beta;
  }
  __syncthreads();
#pragma unroll
  for (int i = 2; i < kChunk; ++i) {
    float sum = A[i];
#pragma unroll
    for (int l = 0; l < i; l += 4) {
      const float4 m = *reinterpret_cast<const float4*>(&s_m[half][i * kPad + l]);
      sum -= m.x * A[l];
      if (l + 1 < i) sum -= m.y * A[l + 1];
      if (l + 2 < i) sum -= m.z * A[l + 2];
      if (l + 3 < i) sum -= m.w * A[l + 3];
    }
    A[i] = sum;
  }
#pragma unroll
  for (int what = 0; what < 2; ++what) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kChunk; ++i) s_m[half][i * kPad + j] = what ? P[i] : A[i];
    __syncthreads();
#pragma unroll
    for (int o = 0; o < 2; ++o) {
      if (o == 1 && !two) break;
      uint4* u = a.units + (size_t(slot) * a.Hv + h0 + o) * kUnits + (what ? 3 * 128 : 0);
#pragma unroll
      for (int tile = 0; tile < 2; ++tile) {
        const int r = 16 * tile + lane % 16, c = lane / 16 * 4;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int cc = unit_row(c, i);
          v[i] = TURNED ? s_m[o][cc * kPad + r] : s_m[o][r * kPad + cc];
        }
        Unit w[3];
        split<3>(v, w);
#pragma unroll
        for (int n = 0; n < 3; ++n) u[(n * 2 + tile) * 64 + lane] = __builtin_bit_cast(uint4, w[n]);
      }
    }
  }
}

// A sequence, or a part of one that is walked by itself
struct Part {
  int seq, row, rows, slot, segment;   // as a Span, of the part
  bool first, last;                    // of its sequence
};

// part x of the launch; false for a number that no part takes
__device__ __forceinline__ bool part_of(const DeltaRule& a, int x, Part& p) {
  if (!a.fold) {
    const int seq = __builtin_amdgcn_readfirstlane(longest_first(a, x));
    const Span sp = span_of(a, seq);
    p = {seq, sp.row, sp.rows, sp.slot, sp.segment, true, true};
    return true;
  }
  int seq, i;
  if (!a.offsets) {
    const int n = a.T / a.fold + (a.T % a.fold != 0);
    seq = x / n, i = x - seq * n;
  } else {   // sequence s begins at its first row's part and s more, so that an empty one has a number too
    const auto begin = [&](int s) {
      const int lo = a.offsets[s];
      return (lo < 0 ? 0 : lo > a.T ? a.T : lo) / a.fold + s;
    };
    int lo = 0, hi = a.nseq;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (begin(mid) <= x) lo = mid;
      else hi = mid;
    }
    seq = lo, i = x - begin(lo);
  }
  const Span sp = span_of(a, seq);
  const int parts = sp.rows <= a.fold ? 1 : (sp.rows - 1) / a.fold + 1;
  if (i < 0 || i >= parts) return false;
  const int skip = i * a.fold, left = sp.rows - skip;
  p = {seq, sp.row + skip, left < a.fold ? left : a.fold, sp.slot + skip / kChunk, sp.segment + skip / kSegment, i == 0, i == parts - 1};
  return true;
}

// What a walk does with a column: its first state and where its last one goes.  MAP: the part's own effect, for all parts but
// a sequence's last - on the columns of no state (of the first part, of the state before it), and on those of a unit matrix
struct Column {
  int width, col;        // of the states' rows
  bool mine, unit;       // unit: of the unit matrix, which no value enters
  const float* from;     // or null: zeros, or the unit matrix
  float* to;             // or null
};

template <int DKP, bool MAP>
__device__ __forceinline__ bool column_of(const DeltaRule& a, const Part& p, int part, int h, int block, int lane_col, int columns, Column& c) {
  const int values = (a.dv + columns - 1) / columns;
  c.unit = MAP && block >= values;
  if (MAP && (p.last || (c.unit && p.first))) return false;
  c.width = c.unit ? DKP : a.dv;
  c.col = (c.unit ? block - values : block) * columns + lane_col;
  c.mine = c.col < c.width;
  const size_t state = size_t(a.dk) * a.dv, at = size_t(part) * a.Hv + h, seq = size_t(p.seq) * a.Hv + h;
  c.from = c.unit ? nullptr : p.first ? (a.h0 ? a.h0 + seq * state : nullptr) : MAP ? nullptr : a.ends + (at - a.Hv) * state;
  c.to = c.unit ? a.maps + at * DKP * DKP : MAP ? a.ends + at * state : p.last && a.h_out ? a.h_out + seq * state : nullptr;
  return true;
}

template <int DKP>
__device__ __forceinline__ void first_state(const DeltaRule& a, const Column& c, int g, f32x4_t (&S)[DKP / 16]) {
#pragma unroll
  for (int m = 0; m < DKP / 16; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 16 * m + 4 * g + i;
      S[m][i] = c.unit ? (r == c.col ? 1.0f : 0.0f) : c.from && c.mine && r < a.dk ? c.from[size_t(r) * c.width + c.col] : 0.0f;
    }
}

template <int DKP>
__device__ __forceinline__ void last_state(const DeltaRule& a, const Column& c, int g, const f32x4_t (&S)[DKP / 16]) {
  if (!c.to || !c.mine) return;
#pragma unroll
  for (int m = 0; m < DKP / 16; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 16 * m + 4 * g + i;
      if (r < (c.unit ? DKP : a.dk)) c.to[size_t(r) * c.width + c.col] = S[m][i];
    }
}

constexpr int kWalkColumns = 64;   // of a workgroup: 16 for each of its four waves

template <int DKP>
struct WalkLds {
  uint4 k[3 * DKP * 4], q[3 * DKP * 4], kt[3 * DKP * 4], lp[kUnits];
  float gains[256];   // gamma, d, beta; the rest takes what threads without a value write
};

// float32: one workgroup carries 64 columns of one sequence's and head's state through the chunks, one kind of wave for all of
// it.  While a chunk is computed from LDS, the next one's rows are on their way into registers; they take its place between
// two barriers (two buffers would fit 64 wide, 100 KB, and save one of them; 128 wide, 87 KB each, they do not).
// 3 x 197 x 3 heads of 40 and 50: 25 us, 3.5 a chunk.
template <int DKP, bool WIDE, bool KEEP, bool MAP>
__global__ __launch_bounds__(256, 1) void delta_walk(DeltaRule a) {
  using T = float;
  constexpr int N = 3, PLANE = DKP * 4, KS = DKP / 32, MT = DKP / 16, LP = kUnits / 256;
  __shared__ WalkLds<DKP> lds;
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, g = lane / 16;
  const int part = blockIdx.x / a.Hv, h = blockIdx.x - part * a.Hv, hk = h / (a.Hv / a.Hk);
  Part sp;
  Column column;
  if (!part_of(a, part, sp) || !column_of<DKP, MAP>(a, sp, part, h, blockIdx.y, wave * 16 + lane % 16, kWalkColumns, column)) return;
  const int b = a.offsets ? 0 : sp.seq, chunks = chunks_of(sp.rows), col = column.col;
  const bool mine = column.mine;
  const int y_row = a.Hv * a.dv;

  f32x4_t S[MT];
  first_state<DKP>(a, column, g, S);

  // a thread's share of a chunk's rows
  const int p_tok = tid % 8 + tid / (8 * 2 * KS) * 8, p_at = tid / 8 % (2 * KS);   // row, 32 (p_at / 2) + 8 (p_at % 2)
  const bool p_on = KS == 4 || tid < 64 * KS;
  const int p_col = p_at / 2 * 32 + p_at % 2 * 8;
  const int p_unit = ((p_at / 2 * 2 + p_tok / 16) * 4 + p_at % 2 * 2) * 16 + p_tok % 16;
  const int c_g = tid / (DKP / 2), c_col = tid % (DKP / 2) * 2;
  const bool c_on = DKP == 128 || tid < 2 * DKP;
  const int c_unit = (c_col / 16 * 4 + c_g) * 16 + c_col % 16;
  Piece<T, WIDE> pk, pq;
  Columns<T, WIDE> ck;
  u32x4_t lp[LP];
  float gain;
  uint32_t v[8];
  const auto fetch = [&](int c) {
    const long long t = sp.row + (long long)c * kChunk;
    const int rows = sp.rows - c * kChunk;
    const Rows k(row_at<T>(a.k, b, t) + hk * a.dk, a.k.row, rows, a.dk), q(row_at<T>(a.q, b, t) + hk * a.dk, a.q.row, rows, a.dk);
    const Rows vv(row_at<T>(a.v, b, t) + h * a.dv, a.v.row, MAP && column.unit ? 0 : rows, a.dv);
    const size_t head = size_t(sp.slot + c) * a.Hv + h;
    const u32x4_t* units = reinterpret_cast<const u32x4_t*>(a.units) + head * kUnits + tid;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = load_element<T>(vv, vv.at<T, WIDE>(unit_row(4 * g, i), col, a.dv));
    if (p_on) pk.load(k, p_tok, p_col, a.dk);
    if (p_on && !MAP) pq.load(q, p_tok, p_col, a.dk);
    if (c_on) ck.load(k, 4 * c_g, c_col, a.dk);
#pragma unroll
    for (int i = 0; i < LP; ++i) lp[i] = units[256 * i];
    gain = a.gains[head * 96 + tid];   // past the 96: the next ones, or the room behind the last
  };
  const auto stash = [&] {
    if (p_on) pk.store(lds.k + p_unit, PLANE);
    if (p_on && !MAP) pq.store(lds.q + p_unit, PLANE);
    if (c_on) ck.store(lds.kt + c_unit, PLANE);
#pragma unroll
    for (int i = 0; i < LP; ++i) lds.lp[tid + 256 * i] = __builtin_bit_cast(uint4, lp[i]);
    lds.gains[tid] = gain;
  };

  if (chunks) {
    fetch(0);
    stash();
  }
  for (int c = 0; c < chunks; ++c) {
    __syncthreads();
    float V[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) V[i] = element<T>(v[i]);
    if (c + 1 < chunks) fetch(c + 1);

    if (KEEP && c % (kSegment / kChunk) == 0 && mine) {
      float* st = a.states + (size_t(sp.segment + c / (kSegment / kChunk)) * a.Hv + h) * a.dk * a.dv + col;
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (16 * m + 4 * g + i < a.dk) st[size_t(16 * m + 4 * g + i) * a.dv] = S[m][i];
    }
    f32x4_t ks[2] = {}, qs[2] = {};
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
        if constexpr (MAP) continue;
        take(lds.q + (s * 2 + t) * 64 + lane, PLANE, w);
        qs[t] = product(w, u, qs[t]);
      }
    }
    float R[8], E[8], x[8], gm[8], dd[8], bt[8];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const float4 g4 = *reinterpret_cast<const float4*>(&lds.gains[16 * t + 4 * g]);
      const float4 d4 = *reinterpret_cast<const float4*>(&lds.gains[32 + 16 * t + 4 * g]);
      const float4 b4 = *reinterpret_cast<const float4*>(&lds.gains[64 + 16 * t + 4 * g]);
      gm[4 * t] = g4.x, gm[4 * t + 1] = g4.y, gm[4 * t + 2] = g4.z, gm[4 * t + 3] = g4.w;
      dd[4 * t] = d4.x, dd[4 * t + 1] = d4.y, dd[4 * t + 2] = d4.z, dd[4 * t + 3] = d4.w;
      bt[4 * t] = b4.x, bt[4 * t + 1] = b4.y, bt[4 * t + 2] = b4.z, bt[4 * t + 3] = b4.w;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      R[i] = V[i] - gm[i] * ks[i / 4][i % 4];
      x[i] = bt[i] * R[i];
      qs[i / 4][i % 4] *= a.scale * gm[i];
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
        for (int i = 0; i < 4; ++i) E[4 * t + i] = R[4 * t + i] - le[i];
      }
    }
    {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = bt[i] * E[i];
    }
    if constexpr (!MAP) {
      Unit u[3];
      split<3>(x, u);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        Unit w[3];
        take(lds.lp + 3 * 128 + t * 64 + lane, 128, w);
        qs[t] = product(w, u, qs[t]);
      }
      const long long t0 = sp.row + (long long)c * kChunk;
      const int rows = sp.rows - c * kChunk;
      const size_t head = ((size_t(b) * a.T + t0) * a.Hv + h) * a.dv;
      const Rows yy(static_cast<T*>(a.y) + head, y_row, rows, a.dv);
#pragma unroll
      for (int i = 0; i < 8; ++i) store_element<T>(yy, yy.at<T, true>(unit_row(4 * g, i), col, a.dv), qs[i / 4][i % 4]);
      if constexpr (KEEP) {
        const Rows ee(a.errors + head, y_row, rows, a.dv);
#pragma unroll
        for (int i = 0; i < 8; ++i) store_element<float>(ee, ee.at<float, true>(unit_row(4 * g, i), col, a.dv), E[i]);
      }
    }
    {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= dd[i];
      Unit u[3];
      split<3>(x, u);
      const float all = lds.gains[31];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        Unit w[N];
        take(lds.kt + m * 64 + lane, PLANE, w);
        S[m] = product(w, u, S[m] * all);
      }
    }
    if (c + 1 < chunks) {
      __syncthreads();
      stash();
    }
  }
  last_state<DKP>(a, column, g, S);
  // rows behind the last sequence
  if (!MAP && a.offsets && a.zero_tail && sp.seq == a.nseq - 1 && sp.last && mine)
    for (int t = sp.row + sp.rows + g; t < a.T; t += 4) put(static_cast<T*>(a.y) + (size_t(t) * a.Hv + h) * a.dv + col, 0.0f);
}

template <int DKP>
struct PairLds {
  static constexpr int kPlane = DKP * 4;
  uint4 k[2][kPlane], kt[2][kPlane], l[2][3 * 128], q[2][kPlane], p[2][3 * 128];
  f32x4_t qs[2][4][2 * 64], u[2][4][2 * 64];   // Q S and U, a wave's columns each
  float gains[4][96];
};

// The same for bfloat16 by two kinds of waves, a pair for 16 columns on each SIMD: the first carries the state and takes Q S from
// its parts while it has them, the second brings the chunks' rows to LDS and makes y of the chunk before, from Q S and U that the
// first leaves in LDS: 2.4 us a chunk on a full chip (8 x 2048 x 16 heads of 128: 154 us) and 1.9 with few workgroups.  One kind
// of wave for all of it took 3.4 and 2.6; Q S by the second wave, which splits the state once more, 3.1.  What bounds it: the 600
// instructions that the first wave issues a step, 84 products and those that split and combine, one behind the other.
template <int DKP, bool WIDE, bool KEEP, bool MAP>
__global__ __launch_bounds__(512, 1) void delta_walk_pairs(DeltaRule a) {
  using T = Bf16;
  using Lds = PairLds<DKP>;
  constexpr int PLANE = Lds::kPlane, KS = DKP / 32, MT = DKP / 16;
  __shared__ Lds lds;
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64) % 4, g = lane / 16;
  const bool carries = __builtin_amdgcn_readfirstlane(threadIdx.x / 256) == 0;
  const int tid = threadIdx.x % 256;
  const int part = blockIdx.x / a.Hv, h = blockIdx.x - part * a.Hv, hk = h / (a.Hv / a.Hk);
  Part sp;
  Column column;
  if (!part_of(a, part, sp) || !column_of<DKP, MAP>(a, sp, part, h, blockIdx.y, wave * 16 + lane % 16, kWalkColumns, column)) return;
  const int b = a.offsets ? 0 : sp.seq, chunks = chunks_of(sp.rows), col = column.col;
  const bool mine = column.mine;
  const int y_row = a.Hv * a.dv;

  if (carries) {
    f32x4_t S[MT];
    first_state<DKP>(a, column, g, S);
    uint32_t v[8];
    const auto fetch = [&](int c) {
      const Rows vv(row_at<T>(a.v, b, sp.row + (long long)c * kChunk) + h * a.dv, a.v.row, MAP && column.unit ? 0 : sp.rows - c * kChunk, a.dv);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = load_element<T>(vv, vv.at<T, WIDE>(unit_row(4 * g, i), col, a.dv));
    };
    if (chunks) fetch(0);
    for (int c = 0; c < chunks; ++c) {
      __syncthreads();
      const int o = c % 2;
      const float* gains = lds.gains[c % 4];
      float V[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) V[i] = element<T>(v[i]);
      if (c + 1 < chunks) fetch(c + 1);
      if (KEEP && c % (kSegment / kChunk) == 0 && mine) {
        float* st = a.states + (size_t(sp.segment + c / (kSegment / kChunk)) * a.Hv + h) * a.dk * a.dv + col;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (16 * m + 4 * g + i < a.dk) st[size_t(16 * m + 4 * g + i) * a.dv] = S[m][i];
      }
      f32x4_t ks[2] = {}, qs[2] = {};
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        Unit u[3];
        split_pair(S[2 * s], S[2 * s + 1], u);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          Unit w[1];
          take(lds.k[o] + (s * 2 + t) * 64 + lane, PLANE, w);
          ks[t] = product(w, u, ks[t]);
          if constexpr (MAP) continue;
          take(lds.q[o] + (s * 2 + t) * 64 + lane, PLANE, w);
          qs[t] = product(w, u, qs[t]);
        }
      }
      if constexpr (!MAP) lds.qs[o][wave][lane] = qs[0], lds.qs[o][wave][64 + lane] = qs[1];
      float R[8], E[8], x[8], gm[8], dd[8], bt[8];
      take_rows(gains, g, gm), take_rows(gains + 32, g, dd), take_rows(gains + 64, g, bt);
#pragma unroll
      for (int i = 0; i < 8; ++i) R[i] = V[i] - gm[i] * ks[i / 4][i % 4], x[i] = bt[i] * R[i];
      {
        Unit u[3];
        split<3>(x, u);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          Unit w[3];
          take(lds.l[o] + t * 64 + lane, 128, w);
          const f32x4_t le = product(w, u, f32x4_t{});
#pragma unroll
          for (int i = 0; i < 4; ++i) E[4 * t + i] = R[4 * t + i] - le[i];
        }
      }
      {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = bt[i] * E[i];
        if constexpr (!MAP) lds.u[o][wave][lane] = f32x4_t{x[0], x[1], x[2], x[3]}, lds.u[o][wave][64 + lane] = f32x4_t{x[4], x[5], x[6], x[7]};
      }
      if constexpr (KEEP) {
        const Rows ee(a.errors + ((size_t(b) * a.T + sp.row + (long long)c * kChunk) * a.Hv + h) * a.dv, y_row, sp.rows - c * kChunk, a.dv);
#pragma unroll
        for (int i = 0; i < 8; ++i) store_element<float>(ee, ee.at<float, true>(unit_row(4 * g, i), col, a.dv), E[i]);
      }
      {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] *= dd[i];
        Unit u[3];
        split<3>(x, u);
        const float all = gains[31];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          Unit w[1];
          take(lds.kt[o] + m * 64 + lane, PLANE, w);
          S[m] = product(w, u, S[m] * all);
        }
      }
    }
    __syncthreads();
    last_state<DKP>(a, column, g, S);
    // rows behind the last sequence
    if (!MAP && a.offsets && a.zero_tail && sp.seq == a.nseq - 1 && sp.last && mine)
      for (int t = sp.row + sp.rows + g; t < a.T; t += 4) put(static_cast<T*>(a.y) + (size_t(t) * a.Hv + h) * a.dv + col, 0.0f);
    return;
  }

  // a thread's share of a chunk's rows
  const int p_tok = tid % 8 + tid / (8 * 2 * KS) * 8, p_at = tid / 8 % (2 * KS);   // row, 32 (p_at / 2) + 8 (p_at % 2)
  const bool p_on = KS == 4 || tid < 64 * KS;
  const int p_col = p_at / 2 * 32 + p_at % 2 * 8;
  const int p_unit = ((p_at / 2 * 2 + p_tok / 16) * 4 + p_at % 2 * 2) * 16 + p_tok % 16;
  const int c_g = tid / (DKP / 2), c_col = tid % (DKP / 2) * 2;
  const bool c_on = DKP == 128 || tid < 2 * DKP;
  const int c_unit = (c_col / 16 * 4 + c_g) * 16 + c_col % 16;
  Piece<T, WIDE> pk, pq;
  Columns<T, WIDE> ck;
  u32x4_t l[2], p[2];
  float gain;
  const auto units_of = [&](int c) {
    return reinterpret_cast<const u32x4_t*>(a.units) + (size_t(sp.slot + c) * a.Hv + h) * kUnits;
  };
  const auto fetch_rows = [&](int c) {   // what the state takes
    const Rows k(row_at<T>(a.k, b, sp.row + (long long)c * kChunk) + hk * a.dk, a.k.row, sp.rows - c * kChunk, a.dk);
    if (p_on) pk.load(k, p_tok, p_col, a.dk);
    if (c_on) ck.load(k, 4 * c_g, c_col, a.dk);
    if (!MAP) {
      const Rows q(row_at<T>(a.q, b, sp.row + (long long)c * kChunk) + hk * a.dk, a.q.row, sp.rows - c * kChunk, a.dk);
      if (p_on) pq.load(q, p_tok, p_col, a.dk);
    }
    l[0] = units_of(c)[tid], l[1] = units_of(c)[256 + tid % 128];
    gain = a.gains[(size_t(sp.slot + c) * a.Hv + h) * 96 + tid % 96];
  };
  const auto stash_rows = [&](int c) {
    if (p_on) pk.store(lds.k[c % 2] + p_unit, PLANE);
    if (c_on) ck.store(lds.kt[c % 2] + c_unit, PLANE);
    if (p_on && !MAP) pq.store(lds.q[c % 2] + p_unit, PLANE);
    lds.l[c % 2][tid] = __builtin_bit_cast(uint4, l[0]);
    if (tid < 128) lds.l[c % 2][256 + tid] = __builtin_bit_cast(uint4, l[1]);
    if (tid < 96) lds.gains[c % 4][tid] = gain;
  };
  const auto fetch_pairs = [&](int c) {   // what y takes
    p[0] = units_of(c)[3 * 128 + tid], p[1] = units_of(c)[3 * 128 + 256 + tid % 128];
  };
  const auto stash_pairs = [&](int c) {
    lds.p[c % 2][tid] = __builtin_bit_cast(uint4, p[0]);
    if (tid < 128) lds.p[c % 2][256 + tid] = __builtin_bit_cast(uint4, p[1]);
  };
  // step c: chunk c + 1's rows and chunk c's P come in, chunk c - 1's y goes out
  if (chunks) {
    fetch_rows(0);
    stash_rows(0);
    if (chunks > 1) fetch_rows(1);
    if (!MAP) fetch_pairs(0);
  }
  for (int c = 0; c <= chunks; ++c) {
    __syncthreads();
    if (c + 1 < chunks) stash_rows(c + 1);
    if (!MAP && c < chunks) stash_pairs(c);
    if (c + 2 < chunks) fetch_rows(c + 2);
    if (!MAP && c + 1 < chunks) fetch_pairs(c + 1);
    if (MAP || c == 0) continue;
    const int o = (c - 1) % 2;
    const float* gains = lds.gains[(c - 1) % 4];
    f32x4_t qs[2] = {lds.qs[o][wave][lane], lds.qs[o][wave][64 + lane]};
    float gm[8];
    take_rows(gains, g, gm);
    Unit u[3];
    split_pair(lds.u[o][wave][lane], lds.u[o][wave][64 + lane], u);
    const Rows yy(static_cast<T*>(a.y) + ((size_t(b) * a.T + sp.row + (long long)(c - 1) * kChunk) * a.Hv + h) * a.dv, y_row,
                  sp.rows - (c - 1) * kChunk, a.dv);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      Unit w[3];
      take(lds.p[o] + t * 64 + lane, 128, w);
#pragma unroll
      for (int i = 0; i < 4; ++i) qs[t][i] *= a.scale * gm[4 * t + i];
      qs[t] = product(w, u, qs[t]);
#pragma unroll
      for (int i = 0; i < 4; ++i) store_element<T>(yy, yy.at<T, true>(16 * t + 4 * g + i, col, a.dv), qs[t][i]);
    }
  }
}

// The state behind each part of a sequence but its last, from the one before: ends[i] <- maps[i] ends[i - 1] + ends[i], the
// first being right already.  A wave 16 columns; a part's map, 64 KB, goes to LDS in three bfloat16 parts while the next is
// on its way to registers: 7.5 us a part.
template <int DKP>
__global__ __launch_bounds__(256, 1) void delta_join(DeltaRule a) {
  constexpr int KS = DKP / 32, MT = DKP / 16, PLANE = MT * KS * 64, PIECES = DKP / 32;
  __shared__ uint4 s_map[3 * PLANE];
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, g = lane / 16;
  const int seq = blockIdx.x / a.Hv, h = blockIdx.x - seq * a.Hv, col = blockIdx.y * kWalkColumns + wave * 16 + lane % 16;
  const bool mine = col < a.dv;
  const Span sp = span_of(a, seq);
  const int parts = sp.rows <= a.fold ? 1 : (sp.rows - 1) / a.fold + 1;
  const int part0 = a.offsets ? sp.row / a.fold + seq : seq * (a.T / a.fold + (a.T % a.fold != 0));
  if (parts <= 2) return;
  const auto end_of = [&](int i) { return a.ends + ((size_t(part0) + i) * a.Hv + h) * a.dk * a.dv + col; };
  const auto load = [&](int i, f32x4_t (&S)[MT]) {
    const float* p = end_of(i);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 16 * m + 4 * g + e;
        S[m][e] = mine && r < a.dk ? p[size_t(r) * a.dv] : 0.0f;
      }
  };
  // a thread's pieces of a map: rows p_row + 32 n
  const int p_row = tid % 8 + tid / (8 * 2 * KS) * 8, p_at = tid / 8 % (2 * KS);
  const bool p_on = KS == 4 || tid < 64 * KS;
  const int p_col = p_at / 2 * 32 + p_at % 2 * 8;
  Piece<float, true> piece[PIECES];
  const auto fetch = [&](int i) {
#pragma unroll
    for (int n = 0; n < PIECES; ++n)
      if (p_on) {
        const Rows mm(a.maps + ((size_t(part0) + i) * a.Hv + h) * DKP * DKP + n * 32 * DKP, DKP, kChunk, DKP);
        piece[n].load(mm, p_row, p_col, DKP);
      }
  };
  f32x4_t S[MT], next[MT];
  load(0, S);
  fetch(1);
  for (int i = 1; i < parts - 1; ++i) {
    __syncthreads();
#pragma unroll
    for (int n = 0; n < PIECES; ++n)
      if (p_on) piece[n].store(s_map + ((p_at / 2 * MT + 2 * n + p_row / 16) * 4 + p_at % 2 * 2) * 16 + p_row % 16, PLANE);
    __syncthreads();
    if (i + 1 < parts - 1) fetch(i + 1);
    load(i, next);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const float x[8] = {S[2 * s][0], S[2 * s][1], S[2 * s][2], S[2 * s][3],
                          S[2 * s + 1][0], S[2 * s + 1][1], S[2 * s + 1][2], S[2 * s + 1][3]};
      Unit u[3];
      split<3>(x, u);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        Unit w[3];
        take(s_map + (s * MT + m) * 64 + lane, PLANE, w);
        next[m] = product(w, u, next[m]);
      }
    }
    float* p = end_of(i);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      S[m] = next[m];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 16 * m + 4 * g + e;
        if (mine && r < a.dk) p[size_t(r) * a.dv] = S[m][e];
      }
    }
  }
}

// One token: 32 columns of a head's state to a workgroup, 8 threads of 4 columns side by side and 32 rows, or with
// element loads 32 threads of one column and 8 rows, at a time.  The state is read once, kept in registers between
// the two sums over its rows, and written once: HBM bounds it.  128 x 16 heads of 128 x 128: 268 MB in 49 to 62 us, 4.3 to
// 5.5 TB/s.
template <typename T, int V>
__global__ __launch_bounds__(256) void delta_step(DeltaRule a) {
  constexpr int X = 32 / V, RG = 256 / X, R = 128 / RG, W = RG * X / 64;   // rows side by side, rows a thread, waves
  __shared__ float s_k[128], s_q[128], s_sum[W][32];
  const int tid = threadIdx.x, tx = tid % X, ty = tid / X, seq = blockIdx.x / a.Hv, h = blockIdx.x - seq * a.Hv;
  const int hk = h / (a.Hv / a.Hk), col = blockIdx.y * 32 + tx * V;
  if (tid < 128) {
    const bool in = tid < a.dk;
    s_k[tid] = in ? to_f32(row_at<T>(a.k, seq, 0)[hk * a.dk + tid]) : 0.0f;
    s_q[tid] = in ? to_f32(row_at<T>(a.q, seq, 0)[hk * a.dk + tid]) : 0.0f;
  }
  const bool mine = col < a.dv;
  const float beta = row_at<float>(a.beta, seq, 0)[h];
  const float alpha = a.decay.p ? expf(row_at<float>(a.decay, seq, 0)[h]) : 1.0f;
  const size_t at = (size_t(seq) * a.Hv + h) * a.dk * a.dv + col;
  float S[R][V], e[V];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = ty + i * RG;
    if (mine && r < a.dk) {
      const auto raw = load_raw<float, V>(a.h0 + at + size_t(r) * a.dv);
#pragma unroll
      for (int x = 0; x < V; ++x) S[i][x] = raw.get(x);
    } else {
#pragma unroll
      for (int x = 0; x < V; ++x) S[i][x] = 0.0f;
    }
  }
#pragma unroll
  for (int x = 0; x < V; ++x) e[x] = mine ? to_f32(row_at<T>(a.v, seq, 0)[h * a.dv + col + x]) : 0.0f;
  __syncthreads();
  // the workgroup's sum over rows of w_r S_r, for the thread's columns
  const auto over_rows = [&](const float* w, float (&sum)[V]) {
#pragma unroll
    for (int x = 0; x < V; ++x) sum[x] = 0.0f;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const float f = w[ty + i * RG];
#pragma unroll
      for (int x = 0; x < V; ++x) sum[x] = fmaf(f, S[i][x], sum[x]);
    }
#pragma unroll
    for (int o = X; o < 64; o *= 2)
#pragma unroll
      for (int x = 0; x < V; ++x) sum[x] += __shfl_xor(sum[x], o);
    if (tid % 64 < X)
#pragma unroll
      for (int x = 0; x < V; ++x) s_sum[tid / 64][tx * V + x] = sum[x];
    __syncthreads();
#pragma unroll
    for (int x = 0; x < V; ++x) {
      sum[x] = 0.0f;
#pragma unroll
      for (int w2 = 0; w2 < W; ++w2) sum[x] += s_sum[w2][tx * V + x];
    }
    __syncthreads();
  };
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int x = 0; x < V; ++x) S[i][x] *= alpha;
  float sum[V];
  over_rows(s_k, sum);
#pragma unroll
  for (int x = 0; x < V; ++x) e[x] = beta * (e[x] - sum[x]);
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = ty + i * RG;
    const float f = s_k[r];
#pragma unroll
    for (int x = 0; x < V; ++x) S[i][x] = fmaf(f, e[x], S[i][x]);
    if (mine && r < a.dk) store_row<V>(a.h_out + at + size_t(r) * a.dv, S[i]);
  }
  over_rows(s_q, sum);
  if (mine && ty == 0) {
    T* y = static_cast<T*>(a.y) + (size_t(seq) * a.Hv + h) * a.dv + col;
#pragma unroll
    for (int x = 0; x < V; ++x) put(y + x, a.scale * sum[x]);
  }
}

long long delta_rule_parts(int fold, int B, int T, int nseq, bool packed) {
  return packed ? T / fold + (long long)nseq : (long long)B * (T / fold + (T % fold != 0));
}

// Rows of the parts that sequences are walked in, or 0.  Few heads of long sequences leave most CUs without work: P parts are
// walked once for what they do to the state (0.75 of a walk's time, for their values' and their keys' columns) and once with
// the state before them, with a product for each between (128 rows' time); a CU walks one workgroup's 64 columns at a time.
// More than 128 workgroups: two parts of each would not run at once any more.
// 1 x 65536 x 8 heads: whole 3810 us, in 16 parts of 4224 rows 435 + 107 + 310.
int delta_rule_fold(int B, int T, int Hv, int dk, int dv, int nseq, bool packed) {
  const long long n = packed ? nseq : B, blocks = (dv + kWalkColumns - 1) / kWalkColumns, units = dk <= 64 ? 1 : 2;
  if (n < 1 || n * Hv * blocks > 128) return 0;
  const int rows = int(T / n);
  const auto rounds = [](long long groups) { return (groups + 255) / 256; };
  int best = 0;
  long long least = 4LL * rows;
  for (int parts = 2; parts <= 32; parts *= 2) {
    const int fold = (rows / parts + kSegment) / kSegment * kSegment;
    if (fold < 2 * kSegment || fold >= rows) continue;
    const long long walks = n * Hv * parts;
    const long long cost = fold * (4 * rounds(walks * blocks) + 3 * rounds(walks * (blocks + units))) + 4 * 128LL * (parts - 2);
    if (cost < least) least = cost, best = fold;
  }
  return best;
}

template <int DKP, typename T, bool WIDE, bool KEEP, bool MAP>
void walk(const DeltaRule& a, int blocks, int columns, hipStream_t s) {
  const dim3 grid(blocks, columns);
  if constexpr (sizeof(T) == 2) delta_walk_pairs<DKP, WIDE, KEEP, MAP><<<grid, 512, 0, s>>>(a);
  else delta_walk<DKP, WIDE, KEEP, MAP><<<grid, 256, 0, s>>>(a);
}

template <int DKP, typename T, bool WIDE>
void walk_all(const DeltaRule& a, hipStream_t s) {
  const int n = a.offsets ? a.nseq : a.B, columns = (a.dv + kWalkColumns - 1) / kWalkColumns;
  const int parts = a.fold ? int(delta_rule_parts(a.fold, a.B, a.T, a.nseq, a.offsets != nullptr)) : n;
  if (a.fold) {
    walk<DKP, T, WIDE, false, true>(a, parts * a.Hv, columns + DKP / kWalkColumns, s);
    delta_join<DKP><<<dim3(n * a.Hv, columns), 256, 0, s>>>(a);
  }
  if (a.errors) walk<DKP, T, WIDE, true, false>(a, parts * a.Hv, columns, s);
  else walk<DKP, T, WIDE, false, false>(a, parts * a.Hv, columns, s);
}

template <typename T, bool WIDE>
void run_as(const DeltaRule& a, hipStream_t s) {
  launch_delta_prepare<T, false>(a, WIDE, s);
  if (a.dk <= 64) walk_all<64, T, WIDE>(a, s);
  else walk_all<128, T, WIDE>(a, s);
}

template <typename T>
void run(const DeltaRule& a, hipStream_t s) {
  if (wide_rows<T>(a.q, a.Hk, a.dk) && wide_rows<T>(a.k, a.Hk, a.dk) && a.v.row >= (long long)a.Hv * a.dv)
    run_as<T, true>(a, s);
  else run_as<T, false>(a, s);
}

template <typename T>
void step(DeltaRule& a, hipStream_t s) {
  const dim3 grid(a.B * a.Hv, (a.dv + 31) / 32);
  const bool vec = a.dv % 4 == 0 && reinterpret_cast<uintptr_t>(a.h0) % 16 == 0 && reinterpret_cast<uintptr_t>(a.h_out) % 16 == 0;
  if (vec) delta_step<T, 4><<<grid, 256, 0, s>>>(a);
  else delta_step<T, 1><<<grid, 256, 0, s>>>(a);
}

}  // namespace

template <typename T, bool TURNED>
void launch_delta_prepare(const DeltaRule& a, bool wide, hipStream_t s) {
  const int slots = int(delta_rule_slots(a.B, a.T, a.nseq, a.offsets != nullptr));   // times Hv below 2^23
  if (!slots) return;
  const dim3 grid(slots, (a.Hv + 1) / 2);
  if (wide && a.dk <= 64) delta_prepare<64, T, true, TURNED><<<grid, 64, 0, s>>>(a);
  else if (wide) delta_prepare<128, T, true, TURNED><<<grid, 64, 0, s>>>(a);
  else if (a.dk <= 64) delta_prepare<64, T, false, TURNED><<<grid, 64, 0, s>>>(a);
  else delta_prepare<128, T, false, TURNED><<<grid, 64, 0, s>>>(a);
}
template void launch_delta_prepare<float, true>(const DeltaRule&, bool, hipStream_t);
template void launch_delta_prepare<Bf16, true>(const DeltaRule&, bool, hipStream_t);

long long delta_rule_slots(int B, int T, int nseq, bool packed) {
  return packed ? T / kChunk + (long long)nseq : (long long)B * chunks_of(T);
}

long long delta_rule_segments(int B, int T, int nseq, bool packed) {
  return packed ? T / kSegment + (long long)nseq : (long long)B * segments_of(T);
}

size_t delta_rule_workspace(int B, int T, int Hv, int dk, int dv, int nseq, bool packed) {
  const int fold = delta_rule_fold(B, T, Hv, dk, dv, nseq, packed), wide = dk <= 64 ? 64 : 128;
  const size_t parts = fold ? size_t(delta_rule_parts(fold, B, T, nseq, packed)) * Hv : 0;
  return size_t(delta_rule_slots(B, T, nseq, packed)) * Hv * (kUnits * sizeof(uint4) + 96 * sizeof(float)) +
         256 * sizeof(float) + parts * (size_t(wide) * wide + size_t(dk) * dv) * sizeof(float);
}

hipError_t launch_delta_rule(DeltaRule a, int dtype, void* workspace, hipStream_t s) {
  const bool packed = a.offsets != nullptr;
  const size_t heads = size_t(delta_rule_slots(a.B, a.T, a.nseq, packed)) * a.Hv, wide = a.dk <= 64 ? 64 : 128;
  a.units = static_cast<uint4*>(workspace);
  a.gains = reinterpret_cast<float*>(a.units + heads * kUnits);
  float* at = a.gains + heads * 96 + 256;   // 160 more behind the last are read
  a.fold = delta_rule_fold(a.B, a.T, a.Hv, a.dk, a.dv, a.nseq, packed);
  if (a.fold) {
    a.maps = at;
    a.ends = at + size_t(delta_rule_parts(a.fold, a.B, a.T, a.nseq, packed)) * a.Hv * wide * wide;
  }
  if (dtype == 0) run<float>(a, s);
  else run<Bf16>(a, s);
  return hipGetLastError();
}

hipError_t launch_delta_rule_step(DeltaRule a, int dtype, hipStream_t s) {
  if (dtype == 0) step<float>(a, s);
  else step<Bf16>(a, s);
  return hipGetLastError();
}

}  // namespace cssm
