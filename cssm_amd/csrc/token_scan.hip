// The gated recurrence over token sequences (gfx950), for each channel in real arithmetic:
//   u = delta + bias,  D = softplus(u),  a = kappa exp(-D) = kappa sigmoid(-u)
//   h_t = a_t h_{t-1} + D_t x_t,  y_t = h_t SiLU(z_t)
// and its adjoint, with p_t = dy_t SiLU(z_t) and G_t = a_t (p_t + G_{t+1}) the gradient handed to h_{t-1}:
//   g_t = p_t + G_{t+1},  dx = D g,  ddelta = sigmoid(u) g (x - a h_{t-1}),  dz = dy h SiLU'(z)
//   dkappa = sum g sigmoid(-u) h_{t-1},  dbias = sum ddelta
// Every step is h -> A h + S, and such maps compose: (A1, S1) then (A2, S2) is (A2 A1, A2 S1 + S2).  So time is cut
// into tiles of 128 rows, and one pass over the data does all: a workgroup loads its tile, publishes the tile's map,
// gathers the state before the tile from the maps of the tiles before it, and only then walks its rows from
// registers and writes the outputs.  The adjoint does the same from the end, with the states the forward kept.
// One tile is 128 rows x 16 V channels on 256 threads: 16 lanes side by side over channels, 16 groups of 8
// consecutive rows, so a thread's rows stay in registers from load to store.
// All sums and states are float32; y and the gradients are rounded once, to their type.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "launch.h"
#include "token_util.h"

namespace cssm {

namespace {

constexpr int kTile = kTokenTile, kRows = 8, kSubs = kTile / kRows, kLanes = 16;

// the A of a tile's map in which a sequence starts: nothing from before comes through (not 0 times it, which
// would let an infinite state of the sequence before leak).  A NaN that no arithmetic makes.
constexpr uint32_t kCut = 0x7fc0c0deu;
__device__ __forceinline__ bool is_cut(float a) { return __float_as_uint(a) == kCut; }
__device__ __forceinline__ float cut() { return __uint_as_float(kCut); }

struct Map { float A, S; };
// first, then `next`
__device__ __forceinline__ Map then(Map first, Map next) {
  if (is_cut(next.A)) return next;
  return {is_cut(first.A) ? cut() : next.A * first.A, fmaf(next.A, first.S, next.S)};
}
__device__ __forceinline__ float apply(Map m, float h) { return is_cut(m.A) ? m.S : fmaf(m.A, h, m.S); }

// D = softplus(u), keep = sigmoid(-u) = exp(-D), gate = sigmoid(u), each to a few ulp: with e = exp(-|u|) and
// w = 1 + e rounded, ln(1 + e) = ln(w) + (e - (w - 1)) / w holds its relative accuracy down to e alone
struct Gains { float D, keep, gate; };
__device__ __forceinline__ Gains gains(float u) {
  const float e = fast_exp(-fabsf(u)), w = 1.0f + e, r = __builtin_amdgcn_rcpf(w);
  const float l = fmaf(e - (w - 1.0f), r, 0.69314718055994531f * __builtin_amdgcn_logf(w));
  const float s = e * r;
  return {fmaxf(u, 0.0f) + l, u > 0.0f ? s : r, u > 0.0f ? r : s};
}

// Which sequence starts / ends at each row of a tile, -1 where none does (packed sequences).
struct Marks {
  int start[kTile], end[kTile];
};
// Offsets are compared, never used as an index, so a bad one cannot leave the tensors.  Ends in a barrier.
__device__ __forceinline__ void find_marks(Marks& m, const int* __restrict__ off, int nseq, int r0, int limit) {
  for (int i = threadIdx.x; i < kTile; i += 256) m.start[i] = m.end[i] = -1;
  __syncthreads();
  for (int s = threadIdx.x; s < nseq; s += 256) {
    const int b = off[s], e = off[s + 1];
    if (e <= b || e > limit || b < 0) continue;
    if (b >= r0 && b - r0 < kTile) m.start[b - r0] = s;
    if (e > r0 && e - 1 - r0 < kTile) m.end[e - 1 - r0] = s;
  }
  __syncthreads();
}
__device__ __forceinline__ int packed_limit(const int* off, int nseq, int T) {
  const int e = off[nseq];
  return e < 0 ? 0 : e > T ? T : e;
}

struct Where {
  int ct, chunk, b, sub, c, r;   // channel tile, row tile, batch; row group, first channel, first row
  int place;                     // of the row tile on the way: chunk, or from the end
};
// Tiles are handed out by a counter in the order of their place on the way, so that every tile waits only for tiles
// whose workgroups run already; with one tile a sequence nothing waits and the block index does.
template <int V, bool REV>
__device__ __forceinline__ Where where(const TokenScan& a, int nchunks) {
  __shared__ unsigned ticket;
  unsigned blk = blockIdx.x;
  if (nchunks > 1) {
    if (threadIdx.x == 0) ticket = atomicAdd(a.ticket, 1u) + 1u;   // starts at all ones
    __syncthreads();
    blk = ticket;
  }
  const unsigned nct = unsigned(a.C + kLanes * V - 1) / (kLanes * V);
  Where w;
  w.ct = int(blk % nct);
  w.b = int(blk / nct % unsigned(a.B));
  w.place = int(blk / nct / unsigned(a.B));
  w.chunk = REV ? nchunks - 1 - w.place : w.place;
  w.sub = threadIdx.x / kLanes;
  w.c = (w.ct * kLanes + int(threadIdx.x % kLanes)) * V;
  w.r = w.chunk * kTile + w.sub * kRows;
  return w;
}

// A map (or with A = 0 a state) as one 64-bit word, which other workgroups see whole or not at all: all ones until it is
// published, so it is its own flag and needs no fence.
constexpr uint64_t kNotYet = ~uint64_t(0);
__device__ __forceinline__ void publish(uint64_t* at, Map m) {
  uint32_t a = __float_as_uint(m.A);
  if (a == 0xffffffffu) a = 0x7fc00000u;   // a NaN is a NaN
  __hip_atomic_store(at, uint64_t(a) << 32 | __float_as_uint(m.S), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t peek(const uint64_t* at) {
  return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// The word's publisher has a lower ticket, so it runs and waits only for lower ones: the wait ends.  (The count only
// keeps a defect from hanging the device; it would end in NaN.)
__device__ __forceinline__ Map await(const uint64_t* at, uint64_t v) {
  for (int i = 0; v == kNotYet && i < (1 << 22); ++i) {
    __builtin_amdgcn_s_sleep(1);
    v = peek(at);
  }
  return {__uint_as_float(uint32_t(v >> 32)), __uint_as_float(uint32_t(v))};
}

// The value entering the tile at this place for one channel, by its own map `own` and those before it.  Places
// come in spans of kSpan: a tile joins the maps of its span's earlier places (at most kSpan - 1, published without
// waiting) and applies them to the value entering the span, which the last tile of the span before published.  So
// the chain of waits has a link for each kSpan tiles, and the sums come in the same order every time.
constexpr int kSpan = 16;
__device__ __forceinline__ float entering(const TokenScan& a, const Where& w, int nchunks, int c, Map own, float first) {
  if (nchunks == 1) return first;
  const int spans = (nchunks + kSpan - 1) / kSpan, span = w.place / kSpan, p0 = span * kSpan;
  uint64_t* maps = a.maps + size_t(w.b) * nchunks * a.C + c;
  uint64_t* heads = a.heads + size_t(w.b) * spans * a.C + c;
  if (w.place + 1 < nchunks) publish(maps + size_t(w.place) * a.C, own);
  Map m = {1.0f, 0.0f};
  uint64_t v[kSpan];   // the last: the span's head
  const uint64_t* head = heads + size_t(span) * a.C;
  if (span > 0) v[kSpan - 1] = peek(head);
#pragma unroll
  for (int i = 0; i < kSpan - 1; ++i)
    if (p0 + i < w.place) v[i] = peek(maps + size_t(p0 + i) * a.C);
#pragma unroll
  for (int i = 0; i < kSpan - 1; ++i)
    if (p0 + i < w.place) m = then(m, await(maps + size_t(p0 + i) * a.C, v[i]));
  if (span > 0) first = await(head, v[kSpan - 1]).S;
  const float in = apply(m, first);
  if (w.place % kSpan == kSpan - 1 && w.place + 1 < nchunks) publish(heads + size_t(span + 1) * a.C, {0.0f, apply(own, in)});
  return in;
}

template <typename T, int V>
__device__ __forceinline__ void load_rows(Raw<T, V> (&q)[kRows], const TokenRows& t, const Where& w, int limit) {
  const T* p = static_cast<const T*>(t.p) + (long long)w.b * t.batch + (long long)w.r * t.row + w.c;
#pragma unroll
  for (int i = 0; i < kRows; ++i)
    if (w.r + i < limit) q[i] = load_raw<T, V>(p + (long long)i * t.row);
}

// Rows kept in 8 bits: plane k of (planes, B, T, C) e4m3 and (planes, B, ceil(T / 8), ceil(C / 16)) exponents.  A
// thread's 8 rows x V channels lie in one block, so it has one scale.
template <int V>
struct Kept {
  uint32_t q[kRows];
  float s;
  __device__ __forceinline__ void load(const TokenScan& a, int plane, const Where& w, int limit) {
    const size_t pb = size_t(plane) * a.B + w.b;
    const uint8_t* p = a.kept + (pb * a.T + w.r) * a.C + w.c;
    if (w.r < limit) s = pow2_of(a.kept_scales[(pb * ((a.T + 7) / 8) + w.r / 8) * ((a.C + 15) / 16) + w.c / 16]);
#pragma unroll
    for (int i = 0; i < kRows; ++i)
      if (w.r + i < limit) {
        const uint8_t* at = p + size_t(i) * a.C;
        q[i] = V == 4 ? *reinterpret_cast<const uint32_t*>(at) : V == 2 ? *reinterpret_cast<const uint16_t*>(at) : *at;
      }
  }
  __device__ __forceinline__ float get(int i, int v) const {
    return s * (v == 0   ? __builtin_amdgcn_cvt_f32_fp8(int(q[i]), 0)
                : v == 1 ? __builtin_amdgcn_cvt_f32_fp8(int(q[i]), 1)
                : v == 2 ? __builtin_amdgcn_cvt_f32_fp8(int(q[i]), 2)
                         : __builtin_amdgcn_cvt_f32_fp8(int(q[i]), 3));
  }
};
template <typename T, int V>
struct Plain {
  Raw<T, V> q[kRows];
  __device__ __forceinline__ float get(int i, int v) const { return q[i].get(v); }
};
template <typename T, int V, bool KEPT>
struct Source : Plain<T, V> {
  __device__ __forceinline__ void load(const TokenScan& a, const TokenRows& t, int, const Where& w, int limit) {
    load_rows<T, V>(this->q, t, w, limit);
  }
};
template <typename T, int V>
struct Source<T, V, true> : Kept<V> {
  __device__ __forceinline__ void load(const TokenScan& a, const TokenRows&, int plane, const Where& w, int limit) {
    Kept<V>::load(a, plane, w, limit);
  }
};

// Keeps 8 rows x V channels in e4m3: the block's largest finite magnitude sets the power of two (16 / V lanes share a
// block of 16 channels); a NaN or an infinite value is kept as NaN.
template <typename T, int V>
__device__ __forceinline__ void keep_rows(const TokenScan& a, int plane, const Raw<T, V> (&q)[kRows], const Where& w,
                                          int limit) {
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < kRows; ++i)
    if (w.c < a.C && w.r + i < limit)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float m = fabsf(q[i].get(v));
        top = fmaxf(top, m < INFINITY ? m : 0.0f);
      }
#pragma unroll
  for (int l = 1; l < 16 / V; l *= 2) top = fmaxf(top, __shfl_xor(top, l));
  if (w.c >= a.C || w.r >= limit) return;
  const int byte = e4m3_scale_byte(top);
  const float inv = pow2_inv(byte);
  const size_t pb = size_t(plane) * a.B + w.b;
  if (w.c % 16 == 0)
    a.kept_scales[(pb * ((a.T + 7) / 8) + w.r / 8) * ((a.C + 15) / 16) + w.c / 16] = uint8_t(byte);
  uint8_t* p = a.kept + (pb * a.T + w.r) * a.C + w.c;
#pragma unroll
  for (int i = 0; i < kRows; ++i)
    if (w.r + i < limit) {
      uint8_t* at = p + size_t(i) * a.C;
      if constexpr (V == 4)
        *reinterpret_cast<uint32_t*>(at) = pack_e4m3x4(q[i].get(0) * inv, q[i].get(1) * inv, q[i].get(2) * inv, q[i].get(3) * inv);
      else if constexpr (V == 2) *reinterpret_cast<uint16_t*>(at) = uint16_t(pack_e4m3x2(q[i].get(0) * inv, q[i].get(1) * inv));
      else *at = uint8_t(pack_e4m3x2(q[i].get(0) * inv, 0.0f));
    }
}

template <int V>
struct Carry {
  Map m[kSubs][kLanes * V];
  float in[kSubs][kLanes * V];
};

// The 16 row groups' maps of each channel, joined in order (REV: from the last): the whole tile's map, and with WRITE
// the value entering each group.  The threads tid < 16 V take a channel each.
template <int V, bool REV, bool WRITE>
__device__ __forceinline__ Map fold(Carry<V>& k, int ch, float in) {
  Map all = {1.0f, 0.0f};
  Map m[kSubs];
#pragma unroll
  for (int i = 0; i < kSubs; ++i) m[i] = k.m[REV ? kSubs - 1 - i : i][ch];
#pragma unroll
  for (int i = 0; i < kSubs; ++i) {
    if (WRITE) {
      k.in[REV ? kSubs - 1 - i : i][ch] = in;
      in = apply(m[i], in);
    } else {
      all = then(all, m[i]);
    }
  }
  return all;
}

// ---- forward

template <typename T, int V, bool PACKED, bool KEEP>
__global__ void __launch_bounds__(256) token_scan_fwd(TokenScan a, int nchunks) {
  __shared__ Carry<V> k;
  __shared__ Marks marks;
  const Where w = where<V, false>(a, nchunks);
  const int limit = PACKED ? packed_limit(a.offsets, a.nseq, a.T) : a.T;
  const bool on = w.c < a.C;
  const int lim = on ? limit : 0;
  Raw<T, V> d[kRows], x[kRows], z[kRows];
  load_rows<T, V>(d, a.delta, w, lim);
  load_rows<T, V>(x, a.x, w, lim);
  if (a.gated) load_rows<T, V>(z, a.z, w, lim);
  float kap[V], bia[V];
#pragma unroll
  for (int v = 0; v < V; ++v) kap[v] = on ? a.kappa[w.c + v] : 0.0f, bia[v] = on ? a.bias[w.c + v] : 0.0f;
  if (PACKED) find_marks(marks, a.offsets, a.nseq, w.chunk * kTile, limit);
  float A[kRows][V], S[kRows][V];
  Map m[V];
#pragma unroll
  for (int v = 0; v < V; ++v) m[v] = {1.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const bool row = w.r + i < lim;
    const int mark = PACKED ? marks.start[w.sub * kRows + i] : -1;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      A[i][v] = 1.0f, S[i][v] = 0.0f;
      if (!row) continue;
      const Gains g = gains(d[i].get(v) + bia[v]);
      A[i][v] = kap[v] * g.keep, S[i][v] = g.D * x[i].get(v);
      if (PACKED && mark >= 0) {
        S[i][v] = fmaf(A[i][v], a.h0 ? a.h0[size_t(mark) * a.C + w.c + v] : 0.0f, S[i][v]);
        A[i][v] = cut();
      }
      m[v] = PACKED ? then(m[v], {A[i][v], S[i][v]}) : Map{m[v].A * A[i][v], fmaf(A[i][v], m[v].S, S[i][v])};
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) k.m[w.sub][int(threadIdx.x % kLanes) * V + v] = m[v];
  __syncthreads();
  const int ch = threadIdx.x, c = w.ct * kLanes * V + ch;
  if (ch < kLanes * V && c < a.C) {
    const float h0 = !PACKED && a.h0 ? a.h0[size_t(w.b) * a.C + c] : 0.0f;   // packed: the starts carry theirs
    const float in = entering(a, w, nchunks, c, fold<V, false, false>(k, ch, 0.0f), h0);
    if (a.states) a.states[(size_t(w.b) * nchunks + w.chunk) * a.C + c] = in;
    fold<V, false, true>(k, ch, in);
    if (w.chunk == 0 && a.h_out) {   // sequences without a row end where they start
      if (PACKED) {
        for (int s = 0; s < a.nseq; ++s)
          if (a.offsets[s + 1] <= a.offsets[s]) a.h_out[size_t(s) * a.C + c] = a.h0 ? a.h0[size_t(s) * a.C + c] : 0.0f;
      } else if (a.T == 0) {
        a.h_out[size_t(w.b) * a.C + c] = in;
      }
    }
  }
  float sz[kRows][V];   // SiLU(z), by the waves that wait for the states
#pragma unroll
  for (int i = 0; i < kRows; ++i)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      sz[i][v] = 1.0f;
      if (a.gated && w.r + i < lim) {
        const float zz = z[i].get(v);
        sz[i][v] = zz * sigmoidf(zz);
      }
    }
  if (KEEP) {
    keep_rows<T, V>(a, 0, x, w, limit);
    keep_rows<T, V>(a, 1, d, w, limit);
    if (a.gated) keep_rows<T, V>(a, 2, z, w, limit);
  }
  __syncthreads();
  if (!on) return;
  float h[V];
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = k.in[w.sub][int(threadIdx.x % kLanes) * V + v];
  T* y = static_cast<T*>(a.y) + (size_t(w.b) * a.T + w.r) * a.C + w.c;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    float out[V];
    if (w.r + i >= limit) {
      if (PACKED && a.zero_tail && w.r + i < a.T) {
#pragma unroll
        for (int v = 0; v < V; ++v) out[v] = 0.0f;
        store_row<V>(y + size_t(i) * a.C, out);
      }
      continue;
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      h[v] = PACKED ? apply({A[i][v], S[i][v]}, h[v]) : fmaf(A[i][v], h[v], S[i][v]);
      out[v] = a.gated ? h[v] * sz[i][v] : h[v];
    }
    store_row<V>(y + size_t(i) * a.C, out);
    const int end = PACKED ? marks.end[w.sub * kRows + i] : w.r + i == a.T - 1 ? w.b : -1;
    if (end >= 0 && a.h_out)
#pragma unroll
      for (int v = 0; v < V; ++v) a.h_out[size_t(end) * a.C + w.c + v] = h[v];
  }
}

// ---- adjoint: the tile's states again from the one before it, the gradients backwards

template <typename T, int V, bool PACKED, bool KEPT>
__global__ void __launch_bounds__(256) token_scan_bwd(TokenScan a, int nchunks) {
  __shared__ Carry<V> k, kr;
  __shared__ Marks marks;
  const Where w = where<V, true>(a, nchunks);
  const int limit = PACKED ? packed_limit(a.offsets, a.nseq, a.T) : a.T;
  const bool on = w.c < a.C;
  const int lim = on ? limit : 0;
  Source<T, V, KEPT> d, x, z;
  Raw<T, V> dy[kRows];
  d.load(a, a.delta, 1, w, lim);
  x.load(a, a.x, 0, w, lim);
  load_rows<T, V>(dy, a.dy, w, lim);
  if (a.gated) z.load(a, a.z, 2, w, lim);
  float kap[V], bia[V];
#pragma unroll
  for (int v = 0; v < V; ++v) kap[v] = on ? a.kappa[w.c + v] : 0.0f, bia[v] = on ? a.bias[w.c + v] : 0.0f;
  if (PACKED) find_marks(marks, a.offsets, a.nseq, w.chunk * kTile, limit);
  // maps of the group's 8 rows, both ways
  float D[kRows][V], keep[kRows][V], P[kRows][V];
  Map m[V], mr[V];
#pragma unroll
  for (int v = 0; v < V; ++v) m[v] = mr[v] = {1.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    if (w.r + i >= lim) continue;
    const int mark = PACKED ? marks.start[w.sub * kRows + i] : -1;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const Gains g = gains(d.get(i, v) + bia[v]);
      D[i][v] = g.D, keep[i][v] = g.keep;
      const float A = kap[v] * g.keep;
      if (mark >= 0) m[v] = {cut(), a.h0 ? a.h0[size_t(mark) * a.C + w.c + v] : 0.0f};
      m[v] = {PACKED && is_cut(m[v].A) ? cut() : m[v].A * A, fmaf(A, m[v].S, g.D * x.get(i, v))};
      P[i][v] = dy[i].get(v);
      if (a.gated) {
        const float zz = z.get(i, v);
        P[i][v] *= zz * sigmoidf(zz);
      }
    }
  }
#pragma unroll
  for (int i = kRows - 1; i >= 0; --i) {
    if (w.r + i >= lim) continue;
    const int mark = PACKED ? marks.end[w.sub * kRows + i] : -1;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float A = kap[v] * keep[i][v];
      if (mark >= 0) mr[v] = {cut(), a.dh ? a.dh[size_t(mark) * a.C + w.c + v] : 0.0f};
      mr[v] = {PACKED && is_cut(mr[v].A) ? cut() : mr[v].A * A, A * (P[i][v] + mr[v].S)};
    }
  }
  const int lc = int(threadIdx.x % kLanes) * V;
#pragma unroll
  for (int v = 0; v < V; ++v) k.m[w.sub][lc + v] = m[v], kr.m[w.sub][lc + v] = mr[v];
  __syncthreads();
  {
    const int half = threadIdx.x / 128, ch = threadIdx.x % 128, c = w.ct * kLanes * V + ch;
    if (ch < kLanes * V && c < a.C) {
      const size_t at = (size_t(w.b) * nchunks + w.chunk) * a.C + c;
      if (half == 0) {
        fold<V, false, true>(k, ch, a.states[at]);
      } else {
        const float dh = !PACKED && a.dh ? a.dh[size_t(w.b) * a.C + c] : 0.0f;
        fold<V, true, true>(kr, ch, entering(a, w, nchunks, c, fold<V, true, false>(kr, ch, 0.0f), dh));
      }
      if (half == 0 && w.chunk == 0 && a.dh0) {
        if (PACKED) {
          for (int s = 0; s < a.nseq; ++s)
            if (a.offsets[s + 1] <= a.offsets[s]) a.dh0[size_t(s) * a.C + c] = a.dh ? a.dh[size_t(s) * a.C + c] : 0.0f;
        } else if (a.T == 0) {
          a.dh0[size_t(w.b) * a.C + c] = a.dh ? a.dh[size_t(w.b) * a.C + c] : 0.0f;
        }
      }
    }
  }
  __syncthreads();
  float h[V], G[V], dk[V], db[V], before[kRows][V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    h[v] = k.in[w.sub][lc + v], G[v] = kr.in[w.sub][lc + v];
    dk[v] = db[v] = 0.0f;
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    if (w.r + i >= lim) continue;
    const int mark = PACKED ? marks.start[w.sub * kRows + i] : -1;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (mark >= 0) h[v] = a.h0 ? a.h0[size_t(mark) * a.C + w.c + v] : 0.0f;
      before[i][v] = h[v];
      h[v] = fmaf(kap[v] * keep[i][v], h[v], D[i][v] * x.get(i, v));
    }
  }
  const size_t row0 = (size_t(w.b) * a.T + w.r) * a.C + w.c;
#pragma unroll
  for (int i = kRows - 1; i >= 0; --i) {
    if (!on) continue;
    const size_t at = row0 + size_t(i) * a.C;
    float ox[V], od[V], oz[V];
    if (w.r + i >= limit) {
      if (PACKED && w.r + i < a.T) {   // rows behind the last sequence have no gradient
#pragma unroll
        for (int v = 0; v < V; ++v) ox[v] = 0.0f;
        store_row<V>(static_cast<T*>(a.dx) + at, ox);
        store_row<V>(static_cast<T*>(a.ddelta) + at, ox);
        if (a.gated) store_row<V>(static_cast<T*>(a.dz) + at, ox);
      }
      continue;
    }
    const int end = PACKED ? marks.end[w.sub * kRows + i] : -1;
    const int start = PACKED ? marks.start[w.sub * kRows + i] : w.r + i == 0 ? w.b : -1;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (end >= 0) G[v] = a.dh ? a.dh[size_t(end) * a.C + w.c + v] : 0.0f;
      const float A = kap[v] * keep[i][v], g = P[i][v] + G[v], xx = x.get(i, v);
      ox[v] = D[i][v] * g;
      const float u = d.get(i, v) + bia[v];
      const float gate = sigmoidf(u);
      od[v] = gate * (g * (xx - A * before[i][v]));
      dk[v] = fmaf(g * keep[i][v], before[i][v], dk[v]);
      db[v] += od[v];
      if (a.gated) {
        const float zz = z.get(i, v), s = sigmoidf(zz);
        const float hh = fmaf(A, before[i][v], D[i][v] * xx);
        oz[v] = dy[i].get(v) * hh * (s * fmaf(zz, 1.0f - s, 1.0f));
      }
      G[v] = A * g;
      if (start >= 0 && a.dh0) a.dh0[size_t(start) * a.C + w.c + v] = G[v];
    }
    store_row<V>(static_cast<T*>(a.dx) + at, ox);
    store_row<V>(static_cast<T*>(a.ddelta) + at, od);
    if (a.gated) store_row<V>(static_cast<T*>(a.dz) + at, oz);
  }
  __syncthreads();
#pragma unroll
  for (int v = 0; v < V; ++v) k.m[w.sub][lc + v] = {dk[v], db[v]};
  __syncthreads();
  const int ch = threadIdx.x, c = w.ct * kLanes * V + ch;
  if (ch < kLanes * V && c < a.C) {
    Map sum = k.m[0][ch];
#pragma unroll
    for (int s = 1; s < kSubs; ++s) sum.A += k.m[s][ch].A, sum.S += k.m[s][ch].S;
    reinterpret_cast<Map*>(a.parts)[(size_t(w.b) * nchunks + w.chunk) * a.C + c] = sum;
  }
}

// dkappa and dbias: the tiles' sums in a fixed order, in float64
// all ones: nothing published, the counter before 0
__global__ void __launch_bounds__(256) token_scan_clear(uint64_t* __restrict__ p, size_t n) {
  for (size_t i = size_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += size_t(gridDim.x) * 256) p[i] = kNotYet;
}

__global__ void __launch_bounds__(1024) token_scan_sums(const float2* __restrict__ parts, int n, int C,
                                                        float* __restrict__ dkappa, float* __restrict__ dbias) {
  __shared__ double sk[64][16], sb[64][16];
  const int l = threadIdx.x % 16, grp = threadIdx.x / 16, c = int(blockIdx.x) * 16 + l;
  double k = 0.0, b = 0.0;
  if (c < C)
#pragma unroll 4
    for (int i = grp; i < n; i += 64) {
      const float2 p = parts[size_t(i) * C + c];
      k += double(p.x), b += double(p.y);
    }
  sk[grp][l] = k, sb[grp][l] = b;
  for (int m = 32; m > 0; m /= 2) {
    __syncthreads();
    if (grp < m) sk[grp][l] += sk[grp + m][l], sb[grp][l] += sb[grp + m][l];
  }
  if (grp == 0 && c < C) dkappa[c] = float(sk[0][l]), dbias[c] = float(sb[0][l]);
}

// ---- one token for each sequence: h = a state + D x, elementwise over (B, C)

template <typename T, int V>
__global__ void __launch_bounds__(256) token_scan_one(TokenScan a) {
  const int per = a.C / V;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long long)a.B * per) return;
  const int b = int(i / per), c = int(i % per) * V;
  const Raw<T, V> d = load_raw<T, V>(static_cast<const T*>(a.delta.p) + b * a.delta.batch + c);
  const Raw<T, V> x = load_raw<T, V>(static_cast<const T*>(a.x.p) + b * a.x.batch + c);
  Raw<T, V> z;
  if (a.gated) z = load_raw<T, V>(static_cast<const T*>(a.z.p) + b * a.z.batch + c);
  const Raw<float, V> h0 = load_raw<float, V>(a.h0 + size_t(b) * a.C + c), kap = load_raw<float, V>(a.kappa + c),
                      bia = load_raw<float, V>(a.bias + c);
  float h[V], y[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const Gains g = gains(d.get(v) + bia.get(v));
    h[v] = fmaf(kap.get(v) * g.keep, h0.get(v), g.D * x.get(v));
    y[v] = h[v];
    if (a.gated) {
      const float zz = z.get(v);
      y[v] *= zz * sigmoidf(zz);
    }
  }
  store_row<V>(static_cast<T*>(a.y) + size_t(b) * a.C + c, y);
  store_row<V>(a.h_out + size_t(b) * a.C + c, h);
}

bool fits(const void* p, long long batch, long long row, int V, size_t size) {
  return reinterpret_cast<uintptr_t>(p) % (V * size) == 0 && batch % V == 0 && row % V == 0;
}
bool fits(const TokenRows& t, int V, size_t size) { return !t.p || fits(t.p, t.batch, t.row, V, size); }

// channels a thread takes: 4 (bf16) or 2 (float32) where every row is aligned for it, else 1
int width(const TokenScan& a, int dtype) {
  const int V = dtype == 0 ? 2 : 4;
  const size_t size = dtype == 0 ? 4 : 2;
  const bool ok = a.C % V == 0 && fits(a.x, V, size) && fits(a.delta, V, size) && fits(a.z, V, size) &&
                  fits(a.dy, V, size) && fits(a.y, 0, 0, V, size) && fits(a.dx, 0, 0, V, size) &&
                  fits(a.ddelta, 0, 0, V, size) && fits(a.dz, 0, 0, V, size) && fits(a.kept, 0, 0, V, 1);
  return ok ? V : 1;
}

template <typename F>
hipError_t by_type(const TokenScan& a, int dtype, F&& f) {
  const int V = width(a, dtype);
  if (dtype == 0) return V == 2 ? f(float(), std::integral_constant<int, 2>()) : f(float(), std::integral_constant<int, 1>());
  return V == 4 ? f(Bf16(), std::integral_constant<int, 4>()) : f(Bf16(), std::integral_constant<int, 1>());
}

}  // namespace

int token_scan_chunks(int T) { return T <= kTile ? 1 : (T + kTile - 1) / kTile; }

// words of the maps, the spans' heads and the counter
size_t token_scan_words(int B, int T, int C) {
  const size_t n = size_t(token_scan_chunks(T));
  return n == 1 ? 0 : 1 + size_t(B) * size_t(C) * (n + (n + kSpan - 1) / kSpan);
}

static void clear(TokenScan& a, uint64_t* words, hipStream_t s) {
  const size_t n = token_scan_words(a.B, a.T, a.C);
  if (!n) return;
  const size_t maps = size_t(a.B) * size_t(a.C) * size_t(token_scan_chunks(a.T));
  a.ticket = reinterpret_cast<unsigned*>(words);
  a.maps = words + 1;
  a.heads = a.maps + maps;
  const size_t g = (n + 1023) / 1024;
  token_scan_clear<<<unsigned(g < 2048 ? g : 2048), 256, 0, s>>>(words, n);
}

hipError_t launch_token_scan(const TokenScan& args, int dtype, uint64_t* words, hipStream_t s) {
  TokenScan a = args;
  clear(a, words, s);
  const int n = token_scan_chunks(a.T);
  return by_type(a, dtype, [&](auto t, auto vw) {
    using T = decltype(t);
    constexpr int V = decltype(vw)::value;
    const unsigned nct = unsigned((a.C + kLanes * V - 1) / (kLanes * V)) * unsigned(a.B);
    if (a.offsets) {
      if (a.kept) token_scan_fwd<T, V, true, true><<<nct * unsigned(n), 256, 0, s>>>(a, n);
      else token_scan_fwd<T, V, true, false><<<nct * unsigned(n), 256, 0, s>>>(a, n);
    } else {
      if (a.kept) token_scan_fwd<T, V, false, true><<<nct * unsigned(n), 256, 0, s>>>(a, n);
      else token_scan_fwd<T, V, false, false><<<nct * unsigned(n), 256, 0, s>>>(a, n);
    }
    return hipGetLastError();
  });
}

hipError_t launch_token_scan_bwd(const TokenScan& args, int dtype, uint64_t* words, hipStream_t s) {
  TokenScan a = args;
  clear(a, words, s);
  const int n = token_scan_chunks(a.T);
  return by_type(a, dtype, [&](auto t, auto vw) {
    using T = decltype(t);
    constexpr int V = decltype(vw)::value;
    const unsigned nct = unsigned((a.C + kLanes * V - 1) / (kLanes * V)) * unsigned(a.B);
    auto run = [&](auto packed, auto kept) {
      constexpr bool P = decltype(packed)::value, K = decltype(kept)::value;
      token_scan_bwd<T, V, P, K><<<nct * unsigned(n), 256, 0, s>>>(a, n);
    };
    const std::true_type yes;
    const std::false_type no;
    if (a.offsets) a.kept ? run(yes, yes) : run(yes, no);
    else a.kept ? run(no, yes) : run(no, no);
    token_scan_sums<<<unsigned((a.C + 15) / 16), 1024, 0, s>>>(reinterpret_cast<const float2*>(a.parts), n * a.B, a.C,
                                                               a.dkappa, a.dbias);
    return hipGetLastError();
  });
}

hipError_t launch_token_scan_step(const TokenScan& a, int dtype, hipStream_t s) {
  const size_t fa = 16;
  auto al = [&](const void* p) { return reinterpret_cast<uintptr_t>(p) % fa == 0; };
  const bool wide = a.C % 4 == 0 && al(a.h0) && al(a.h_out) && al(a.kappa) && al(a.bias);
  auto run = [&](auto t, auto vw) {
    using T = decltype(t);
    constexpr int V = decltype(vw)::value;
    const long long n = (long long)a.B * (a.C / V);
    token_scan_one<T, V><<<unsigned((n + 255) / 256), 256, 0, s>>>(a);
    return hipGetLastError();
  };
  const size_t size = dtype == 0 ? 4 : 2;
  const bool v4 = wide && fits(a.x, 4, size) && fits(a.delta, 4, size) && fits(a.z, 4, size) && fits(a.y, 0, 0, 4, size);
  if (dtype == 0)
    return v4 ? run(float(), std::integral_constant<int, 4>()) : run(float(), std::integral_constant<int, 1>());
  return v4 ? run(Bf16(), std::integral_constant<int, 4>()) : run(Bf16(), std::integral_constant<int, 1>());
}

}  // namespace cssm
