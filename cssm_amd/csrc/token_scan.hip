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
// One tile is 128 rows of 16 V or 32 V channels: LX = 16 or 32 threads side by side over channels, 16 groups of 8
// consecutive rows, so a thread's rows stay in registers from load to store.
// All sums and states are float32; y and the gradients are rounded once, to their type.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "launch.h"
#include "token_rows.h"
#include "token_util.h"

namespace cssm {

namespace {

constexpr int kTile = kTokenTile, kRows = kTokenRows, kSubs = kTile / kRows;

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

// D = softplus(u), keep = exp(-D) = sigmoid(-u) and gate = sigmoid(u), from v = u log2(e), each to a few ulp and |u| half
// steps of float32 (v's rounding moves the logarithm of exp(-|u|) by that much): with
// e = exp(-|u|) and w = 1 + e rounded, ln(w) + (e - (w - 1)) is ln(1 + e) with its relative accuracy down to e alone (what
// w lost is at most 2^-25, next to ln(1 + e) where that is large).
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.69314718055994531f;
struct Gains { float D, keep, gate; };
__device__ __forceinline__ Gains gains(float v) {
  const float e = __builtin_amdgcn_exp2f(-fabsf(v)), w = 1.0f + e, r = __builtin_amdgcn_rcpf(w), s = e * r;
  const float D = fmaf(kLn2, fmaxf(v, 0.0f) + __builtin_amdgcn_logf(w), e - (w - 1.0f));
  const bool up = v > 0.0f;
  const float t = 1.0f - s;   // nearer to 1 / w than r where that is near 1: half a step, not w's and r's roundings
  return {D, up ? s : t, up ? t : s};
}

// Hides from the compiler that a register holds what it held before, and fixes the point by which it is computed.  A tile's
// phases unpack and combine the same packed rows; seen as the same values, the unpacked ones would stay in registers
// from phase to phase, and a row's results be put off until the last row's: twice the registers, which costs more than
// unpacking again.
__device__ __forceinline__ void renew(uint32_t& v) { asm volatile("" : "+v"(v)); }
__device__ __forceinline__ void renew(float& v) { asm volatile("" : "+v"(v)); }
__device__ __forceinline__ void renew(uint2& v) { renew(v.x), renew(v.y); }
__device__ __forceinline__ void renew(float2& v) { renew(v.x), renew(v.y); }
__device__ __forceinline__ void renew(uint16_t& v) {
  uint32_t w = v;
  renew(w);
  v = uint16_t(w);
}
template <typename T, int V>
__device__ __forceinline__ void renew(Raw<T, V> (&q)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) renew(q[i].q);
}

// Which sequence starts / ends at each row of a tile, -1 where none does (packed sequences).
struct Marks {
  int start[kTile], end[kTile];
};
// Offsets are compared, never used as an index, so a bad one cannot leave the tensors.  Ends in a barrier.
__device__ __forceinline__ void find_marks(Marks& m, const int* __restrict__ off, int nseq, int r0, int limit) {
  for (int i = threadIdx.x; i < kTile; i += blockDim.x) m.start[i] = m.end[i] = -1;
  __syncthreads();
  for (int s = threadIdx.x; s < nseq; s += blockDim.x) {
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
template <int LX, int V, bool REV>
__device__ __forceinline__ Where where(const TokenScan& a, int nchunks, unsigned tile) {
  tile = __builtin_amdgcn_readfirstlane(tile);   // it came by shared memory: the same for all
  const unsigned nct = unsigned(a.C + LX * V - 1) / (LX * V);
  Where w;
  w.ct = int(tile % nct);
  w.b = int(tile / nct % unsigned(a.B));
  w.place = int(tile / nct / unsigned(a.B));
  w.chunk = REV ? nchunks - 1 - w.place : w.place;
  w.sub = threadIdx.x / LX;
  w.c = (w.ct * LX + int(threadIdx.x % LX)) * V;
  w.r = w.chunk * kTile + w.sub * kRows;
  return w;
}
// Tiles are handed out by a counter in the order of their place on the way, so that every tile waits only for tiles
// that workgroups already have; with one tile a sequence nothing waits.
__device__ __forceinline__ unsigned my_tile(const TokenScan& a, int nchunks) {
  __shared__ unsigned tile;
  if (nchunks == 1) return blockIdx.x;
  if (threadIdx.x == 0) tile = atomicAdd(a.ticket, 1u) + 1u;   // from all ones
  __syncthreads();
  return tile;
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
// The word's publisher has a lower number than the tile that waits, so its workgroup runs already, and waits only for
// lower ones itself: the wait ends.  (The count only keeps a defect from hanging the device; it would end in NaN.)
__device__ __forceinline__ Map unpack(uint64_t v) {
  return {__uint_as_float(uint32_t(v >> 32)), __uint_as_float(uint32_t(v))};
}
// n <= N words `step` apart, each once it is published; `at` and `step` the same for the wave, `c` its lanes'
template <int N>
__device__ __forceinline__ void await(uint64_t (&v)[N], const uint64_t* at, unsigned c, size_t step, int n) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = i < n ? peek(at + step * i + c) : 0;
  for (int tries = 0; tries < (1 << 22); ++tries) {
    bool all = true;
#pragma unroll
    for (int i = 0; i < N; ++i) all = all && v[i] != kNotYet;
    if (all) break;
    __builtin_amdgcn_s_sleep(1);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (v[i] == kNotYet) v[i] = peek(at + step * i + c);   // only what is missing: each peek goes to memory
  }
}

// The value entering the tile at this place for one channel, by its own map `own` and those before it.  Places
// come in spans of kSpan: a tile joins the maps of its span's earlier places (at most kSpan - 1, published without
// waiting) and applies them to the value entering the span, which the last tile of the span before published.  So
// the chain of waits has a link for each kSpan tiles, and the sums come in the same order every time.
constexpr int kSpan = 8;
__device__ __forceinline__ float entering(const TokenScan& a, const Where& w, int nchunks, int c, Map own, float first) {
  if (nchunks == 1) return first;
  const int spans = (nchunks + kSpan - 1) / kSpan, span = w.place / kSpan, p0 = span * kSpan;
  uint64_t* maps = a.maps + size_t(w.b) * nchunks * a.C;
  uint64_t* heads = a.heads + size_t(w.b) * spans * a.C;
  if (w.place + 1 < nchunks) publish(maps + size_t(w.place) * a.C + c, own);
  Map m = {1.0f, 0.0f};
  const int before = w.place - p0;
  if (before > 0) {
    uint64_t v[kSpan - 1];
    await(v, maps + size_t(p0) * a.C, unsigned(c), size_t(a.C), before);
#pragma unroll
    for (int i = 0; i < kSpan - 1; ++i)
      if (i < before) m = then(m, unpack(v[i]));
  }
  if (span > 0) {
    uint64_t v[1];
    await(v, heads + size_t(span) * a.C, unsigned(c), 0, 1);
    first = unpack(v[0]).S;
  }
  const float in = apply(m, first);
  if (w.place % kSpan == kSpan - 1 && w.place + 1 < nchunks) publish(heads + size_t(span + 1) * a.C + c, {0.0f, apply(own, in)});
  return in;
}

template <int V>
using Off = TileOff<V>;

// The thread's 8 rows, every one of them: rows behind the limit (> 0) give the last one again and channels behind C
// the last ones, which nothing uses.
template <typename T, int V>
__device__ __forceinline__ void load_rows(Raw<T, V> (&q)[kRows], const TokenRows& t, const Where& w, int C, int limit) {
  const int r0 = min(w.chunk * kTile, limit - 1);
  const char* p = static_cast<const char*>(t.p) + ((long long)w.b * t.batch + (long long)r0 * t.row) * (long long)sizeof(T);
  const TileRows<Off<V>> at(Off<V>(t.row) * Off<V>(sizeof(T)), w.sub, Off<V>(min(w.c, C - V)) * Off<V>(sizeof(T)), limit - 1 - r0);
#pragma unroll
  for (int i = 0; i < kRows; ++i) q[i] = load_raw<T, V>(reinterpret_cast<const T*>(p + at(i)));
}

// Rows kept in 8 bits: plane k of (planes, B, T, C) e4m3 and (planes, B, ceil(T / 8), ceil(C / 16)) exponents.  A
// thread's 8 rows x V channels lie in one block, so it has one scale.  Where u = delta + bias <= -104, exp(u) is under
// half of the least float32: D and sigmoid(u) are 0, as for delta = -inf, whatever x is.  That is how such a value is
// kept, as -inf with x = 0, and neither counts for its block's exponent: masked rows, with the type's lowest value in
// delta or anything finite in x, leave the rows beside them their bits.
constexpr float kNoGain = -104.0f;
constexpr int kPlaneX = 0, kPlaneDelta = 1, kPlaneZ = 2;
constexpr uint32_t kNaN8 = 0x7f, kMasked8 = 0xff;   // e4m3 has two NaN; in delta's plane the negative one is -inf
template <int V>
struct Kept {
  uint32_t q[kRows];
  float s;
  __device__ __forceinline__ void again() {
#pragma unroll
    for (int i = 0; i < kRows; ++i) renew(q[i]);
  }
  __device__ __forceinline__ void load(const TokenScan& a, int plane, const Where& w, int limit) {
    const size_t pb = size_t(plane) * a.B + w.b;
    const int c = min(w.c, a.C - V), r0 = min(w.chunk * kTile, limit - 1);
    const uint8_t* p = a.kept + (pb * a.T + r0) * a.C;
    s = pow2_of(a.kept_scales[(pb * ((a.T + 7) / 8) + min(w.r, limit - 1) / 8) * ((a.C + 15) / 16) + c / 16]);
    const TileRows<Off<V>> at(Off<V>(a.C), w.sub, Off<V>(c), limit - 1 - r0);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const uint8_t* x = p + at(i);
      q[i] = V == 4 ? *reinterpret_cast<const uint32_t*>(x) : V == 2 ? *reinterpret_cast<const uint16_t*>(x) : *x;
    }
  }
  __device__ __forceinline__ float get(int i, int v) const {
    const f32x2_t two = v < 2 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(q[i], s, false) : __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(q[i], s, true);
    return two[v & 1];
  }
  // whether a value of the wave's is masked (uniform); a row's masked values as -inf
  __device__ __forceinline__ bool any_masked() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kRows; ++i) m |= (~q[i] - 0x01010101u) & q[i];
    return __any((m & 0x80808080u) != 0);
  }
  __device__ __forceinline__ void mask(int i, float (&f)[V]) const {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if ((q[i] >> (8 * v) & 0xffu) == kMasked8) f[v] = -INFINITY;
      asm volatile("" : "+v"(f[v]));   // kept behind the branch: selects in every row would cost 2 % of the adjoint
    }
  }
};
template <typename T, int V>
struct Plain {
  Raw<T, V> q[kRows];
  __device__ __forceinline__ void again() { renew(q); }
  __device__ __forceinline__ float get(int i, int v) const { return q[i].get(v); }
};
template <typename T, int V, bool KEPT>
struct Source : Plain<T, V> {
  __device__ __forceinline__ void load(const TokenScan& a, const TokenRows& t, int, const Where& w, int limit) {
    load_rows<T, V>(this->q, t, w, a.C, limit);
  }
};
template <typename T, int V>
struct Source<T, V, true> : Kept<V> {
  __device__ __forceinline__ void load(const TokenScan& a, const TokenRows&, int plane, const Where& w, int limit) {
    Kept<V>::load(a, plane, w, limit);
  }
};

// Keeps 8 rows x V channels in e4m3: the block's largest finite magnitude sets the power of two (16 / V lanes share a
// block of 16 channels); a NaN or an infinite value is kept as NaN, but delta's -inf as itself.
template <int V>
__device__ __forceinline__ float largest(const Raw<float, V> (&q)[kRows]) {   // magnitudes order as their bits
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < kRows; ++i)
#pragma unroll
    for (int v = 0; v < V; ++v) m = max(m, __float_as_uint(q[i].get(v)) & 0x7fffffffu);
  return __uint_as_float(m);
}
template <int V>
__device__ __forceinline__ float largest(const Raw<Bf16, V> (&q)[kRows]) {
  if constexpr (V == 4) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t w = (k ? q[i].q.y : q[i].q.x) & 0x7fff7fffu;
        m = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, m), __builtin_bit_cast(u16x2_t, w)));
      }
    return __uint_as_float(max(m << 16, m & 0xffff0000u));
  } else {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kRows; ++i) m = max(m, uint32_t(q[i].q) & 0x7fffu);
    return __uint_as_float(m << 16);
  }
}
// V values over the block's power of two, to nearest even
template <int V>
__device__ __forceinline__ uint32_t keep_row(const Raw<float, V>& q, float scale) {
  s16x2_t r = {};
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, q.get(0), V > 1 ? q.get(V > 1) : 0.0f, scale, false);
  return __builtin_bit_cast(uint32_t, r);
}
template <int V>
__device__ __forceinline__ uint32_t keep_row(const Raw<Bf16, V>& q, float scale) {
  s16x2_t r = {};
  if constexpr (V == 4) {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2_t, q.q.x), scale, false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2_t, q.q.y), scale, true);
  } else {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2_t, uint32_t(q.q)), scale, false);
  }
  return __builtin_bit_cast(uint32_t, r);
}
// value v of a row as T's nearest to f
template <int V>
__device__ __forceinline__ void put(Raw<float, V>& r, int v, float f) {
  if constexpr (V == 2) (v ? r.q.y : r.q.x) = f;
  else r.q = f;
}
template <int V>
__device__ __forceinline__ void put(Raw<Bf16, V>& r, int v, float f) {
  const uint32_t b = __float_as_uint(f) >> 16;
  if constexpr (V == 4) {
    uint32_t& w = v < 2 ? r.q.x : r.q.y;
    w = v & 1 ? (w & 0xffffu) | b << 16 : (w & 0xffff0000u) | b;
  } else {
    r.q = uint16_t(b);
  }
}
// masked values (kNoGain) become delta = -inf and x = 0; an x that is not finite stays, as it made the state not a number
// The largest magnitude of d afterwards.
template <typename T, int V>
__device__ __forceinline__ float hide_masked(Raw<T, V> (&d)[kRows], Raw<T, V> (&x)[kRows], const float* bias) {
  float b[V], most = 0.0f;
#pragma unroll
  for (int v = 0; v < V; ++v) b[v] = bias[v], most = fmaxf(most, fabsf(b[v]));
  const float top = largest<V>(d);
  if (top + most < -kNoGain) return top;
#pragma unroll
  for (int i = 0; i < kRows; ++i)
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (d[i].get(v) + b[v] <= kNoGain) {
        put(d[i], v, -INFINITY);
        if (fabsf(x[i].get(v)) < INFINITY) put(x[i], v, 0.0f);
      }
  return largest<V>(d);
}
template <typename T, int V>
__device__ __forceinline__ void keep_rows(const TokenScan& a, int plane, const Raw<T, V> (&q)[kRows], float top,
                                          const Where& w, int limit) {   // top: the largest of q
  const bool odd = !(top < INFINITY);
  if (odd) {                   // something is not finite: the largest of what is
    top = 0.0f;
    for (int i = 0; i < kRows; ++i)
      for (int v = 0; v < V; ++v) {
        const float m = fabsf(q[i].get(v));
        top = fmaxf(top, m < INFINITY ? m : 0.0f);
      }
  }
#pragma unroll
  for (int l = 1; l < 16 / V; l *= 2) top = fmaxf(top, __shfl_xor(top, l));
  if (w.c >= a.C || w.r >= limit) return;
  const int byte = e4m3_scale_byte(top);
  const float scale = pow2_of(byte);
  const size_t pb = size_t(plane) * a.B + w.b;
  if (w.c % 16 == 0)
    a.kept_scales[(pb * ((a.T + 7) / 8) + w.r / 8) * ((a.C + 15) / 16) + w.c / 16] = uint8_t(byte);
  uint8_t* p = a.kept + (pb * a.T + w.chunk * kTile) * a.C;
  const Off<V> off = Off<V>(w.sub * kRows) * Off<V>(a.C) + Off<V>(w.c);
#pragma unroll
  for (int i = 0; i < kRows; ++i)
    if (w.r + i < limit) {
      uint8_t* at = p + size_t(i) * a.C + off;
      uint32_t k = keep_row<V>(q[i], scale);
      if (plane == kPlaneDelta && odd)
        for (int v = 0; v < V; ++v) {
          const float f = q[i].get(v);
          if (!(fabsf(f) < INFINITY)) k = (k & ~(0xffu << (8 * v))) | (f == -INFINITY ? kMasked8 : kNaN8) << (8 * v);
        }
      if constexpr (V == 4) *reinterpret_cast<uint32_t*>(at) = k;
      else if constexpr (V == 2) *reinterpret_cast<uint16_t*>(at) = uint16_t(k);
      else *at = uint8_t(k);
    }
}

template <int CW>
struct Carry {
  Map m[kSubs][CW];
  float in[kSubs][CW];
};

// The 16 row groups' maps of each channel, joined in order (REV: from the last): the whole tile's map, and with WRITE
// the value entering each group.  A thread takes a channel.
template <int CW, bool REV, bool WRITE>
__device__ __forceinline__ Map fold(Carry<CW>& k, int ch, float in) {
  Map all = {1.0f, 0.0f};
#pragma unroll
  for (int j = 0; j < kSubs; j += 8) {
    asm volatile("" ::: "memory");   // a second call reads again: 32 registers less than holding all maps between the two
    Map m[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) m[i] = k.m[REV ? kSubs - 1 - i - j : i + j][ch];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (WRITE) {
        k.in[REV ? kSubs - 1 - i - j : i + j][ch] = in;
        in = apply(m[i], in);
      } else {
        all = then(all, m[i]);
      }
    }
  }
  return all;
}

// ---- forward
// Bound by HBM, then by the arithmetic between a tile's loads and its stores (about 10 of 72 us: the loads and stores alone
// took 54) and the wait for the tiles before (8).  bf16 with a gate 8 x 4096 x 1024 76 us, 3.5 TB/s (float32 122, 4.4), 1 x
// 65536 x 1024 137 us; with the 8-bit checkpoint 106 us.  8 rows a thread keep the tile in registers between the map and the
// walk, so every value is read once.  Packed rows pay in every tile for its marks, each a look at all offsets, and the first
// tile for empty sequences one by one: 16001 x 2048 in 23 sequences 83 us, in 4096 of them 710.

template <typename T, int V, int LX, bool PACKED, bool KEEP>
__global__ void __launch_bounds__(LX * kSubs, KEEP ? 3 : 4) token_scan_fwd(TokenScan a, int nchunks) {
  __shared__ Carry<LX * V> k;
  __shared__ Marks marks;
  const Where w = where<LX, V, false>(a, nchunks, my_tile(a, nchunks));
  const int limit = PACKED ? packed_limit(a.offsets, a.nseq, a.T) : a.T;
  const bool on = w.c < a.C;
  Raw<T, V> d[kRows], x[kRows], z[kRows];
  if (limit > 0) {
    load_rows<T, V>(d, a.delta, w, a.C, limit);
    load_rows<T, V>(x, a.x, w, a.C, limit);
    if (a.gated) load_rows<T, V>(z, a.z, w, a.C, limit);
  }
  float kap[V], bia[V];
#pragma unroll
  for (int v = 0; v < V; ++v) kap[v] = a.kappa[min(w.c, a.C - V) + v], bia[v] = a.bias[min(w.c, a.C - V) + v];
  if (PACKED) find_marks(marks, a.offsets, a.nseq, w.chunk * kTile, limit);
  float A[kRows][V], S[kRows][V];
  Map m[V];
#pragma unroll
  for (int v = 0; v < V; ++v) m[v] = {1.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    // (rows behind the limit come behind all that counts)
    const int mark = PACKED && on ? marks.start[w.sub * kRows + i] : -1;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const Gains g = gains((d[i].get(v) + bia[v]) * kLog2e);
      A[i][v] = kap[v] * g.keep, S[i][v] = g.D * x[i].get(v);
      if (PACKED && mark >= 0) {
        S[i][v] = fmaf(A[i][v], a.h0 ? a.h0[size_t(mark) * a.C + w.c + v] : 0.0f, S[i][v]);
        A[i][v] = cut();
      }
      m[v] = PACKED ? then(m[v], {A[i][v], S[i][v]}) : Map{m[v].A * A[i][v], fmaf(A[i][v], m[v].S, S[i][v])};
      renew(m[v].S), renew(A[i][v]);
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) k.m[w.sub][int(threadIdx.x % LX) * V + v] = m[v];
  __syncthreads();
  const int ch = threadIdx.x, c = w.ct * LX * V + ch;
  if (ch < LX * V && c < a.C) {
    const float h0 = !PACKED && a.h0 ? a.h0[size_t(w.b) * a.C + c] : 0.0f;   // packed: the starts carry theirs
    const float in = entering(a, w, nchunks, c, fold<LX * V, false, false>(k, ch, 0.0f), h0);
    if (a.states) a.states[(size_t(w.b) * nchunks + w.chunk) * a.C + c] = in;
    fold<LX * V, false, true>(k, ch, in);
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
  for (int i = 0; i < kRows; ++i) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      sz[i][v] = 1.0f;
      if (a.gated) {
        const float zz = z[i].get(v);
        sz[i][v] = zz * sigmoidf(zz);
        renew(sz[i][v]);
      }
    }
  }
  if (KEEP) {
    renew(x), renew(d), renew(z);
    // (a row or channels twice, see load_rows, are of the same block)
    const float top = hide_masked<T, V>(d, x, a.bias + min(w.c, a.C - V));
    keep_rows<T, V>(a, kPlaneX, x, largest<V>(x), w, limit);
    keep_rows<T, V>(a, kPlaneDelta, d, top, w, limit);
    if (a.gated) keep_rows<T, V>(a, kPlaneZ, z, largest<V>(z), w, limit);
  }
  __syncthreads();
  float h[V];
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = k.in[w.sub][int(threadIdx.x % LX) * V + v];
  T* y = static_cast<T*>(a.y) + (size_t(w.b) * a.T + w.chunk * kTile) * a.C;
  const Off<V> off = Off<V>(w.sub * kRows) * Off<V>(a.C) + Off<V>(w.c);
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    float out[V];
    if (!on) continue;
    if (w.r + i >= limit) {
      if (PACKED && a.zero_tail && w.r + i < a.T) {
#pragma unroll
        for (int v = 0; v < V; ++v) out[v] = 0.0f;
        store_row<V>(y + size_t(i) * a.C + off, out);
      }
      continue;
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      h[v] = PACKED ? apply({A[i][v], S[i][v]}, h[v]) : fmaf(A[i][v], h[v], S[i][v]);
      out[v] = a.gated ? h[v] * sz[i][v] : h[v];
    }
    store_row<V>(y + size_t(i) * a.C + off, out);
    const int end = PACKED ? marks.end[w.sub * kRows + i] : w.r + i == a.T - 1 ? w.b : -1;
    if (end >= 0 && a.h_out)
#pragma unroll
      for (int v = 0; v < V; ++v) a.h_out[size_t(end) * a.C + w.c + v] = h[v];
  }
}

// ---- adjoint: the tile's states again from the one before it, the gradients backwards
// 8 x 4096 x 1024 bf16 141 us (3.3 TB/s); from the 8-bit checkpoint, which is 3 bytes a value less to read, 140 all the same.
// The loads and stores alone take 95 to 104.  Its 253 registers (243 from the checkpoint) leave two workgroups a CU, whose
// loads, arithmetic and stores overlap only with each other's.

template <typename T, int V, int LX, bool PACKED, bool KEPT>
__global__ void __launch_bounds__(LX * kSubs, 2) token_scan_bwd(TokenScan a, int nchunks) {
  __shared__ Carry<LX * V> k, kr;
  __shared__ Marks marks;
  const Where w = where<LX, V, true>(a, nchunks, my_tile(a, nchunks));
  const int limit = PACKED ? packed_limit(a.offsets, a.nseq, a.T) : a.T;
  const bool on = w.c < a.C;
  Source<T, V, KEPT> d, x, z;
  Raw<T, V> dy[kRows];
  if (limit > 0) {
    d.load(a, a.delta, kPlaneDelta, w, limit);
    x.load(a, a.x, kPlaneX, w, limit);
    load_rows<T, V>(dy, a.dy, w, a.C, limit);
    if (a.gated) z.load(a, a.z, kPlaneZ, w, limit);
  }
  float kap[V], bia[V];
#pragma unroll
  for (int v = 0; v < V; ++v) kap[v] = a.kappa[min(w.c, a.C - V) + v], bia[v] = a.bias[min(w.c, a.C - V) + v];
  if (PACKED) find_marks(marks, a.offsets, a.nseq, w.chunk * kTile, limit);
  auto again = [&] {
    x.again(), renew(dy);
    if (a.gated) z.again();
  };
  // Rows behind the limit come first on the way back: the end of the last sequence starts afresh.
  auto ends_at = [&](int i) { return !on ? -1 : PACKED ? marks.end[w.sub * kRows + i] : w.r + i == a.T - 1 ? w.b : -1; };
  // Maps of the group's 8 rows both ways, from the last row up, where a row enters the forward map by the product of the
  // A behind it: that product is the A of both.
  float D[kRows][V], kp[kRows][V], gt[kRows][V], sz[kRows][V];   // softplus, sigmoid(-u), sigmoid(u), sigmoid(z)
  Map m[V], mr[V];
  bool cut_fwd = false, cut_rev = false;   // packed: a sequence starts / ends in the group
  bool masks = false;
  if constexpr (KEPT) masks = limit > 0 && d.any_masked();
#pragma unroll
  for (int v = 0; v < V; ++v) m[v] = mr[v] = {1.0f, 0.0f};
#pragma unroll
  for (int i = kRows - 1; i >= 0; --i) {
    const int end = ends_at(i), start = PACKED && on ? marks.start[w.sub * kRows + i] : -1;
    if (end >= 0) {
      cut_rev = true;
#pragma unroll
      for (int v = 0; v < V; ++v) mr[v] = {0.0f, a.dh ? a.dh[size_t(end) * a.C + w.c + v] : 0.0f};
    }
    float dl[V];
#pragma unroll
    for (int v = 0; v < V; ++v) dl[v] = d.get(i, v);
    if constexpr (KEPT)
      if (masks) d.mask(i, dl);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const Gains g = gains((dl[v] + bia[v]) * kLog2e);
      D[i][v] = g.D, kp[i][v] = g.keep, gt[i][v] = g.gate;
      const float A = kap[v] * g.keep;
      if (!PACKED || !cut_fwd) {
        m[v].S = fmaf(m[v].A, g.D * x.get(i, v), m[v].S);
        m[v].A *= A;
      }
      if (PACKED) mr[v].A *= A;
      float p = dy[i].get(v);
      if (a.gated) {
        const float zz = z.get(i, v);
        sz[i][v] = sigmoidf(zz);
        p *= zz * sz[i][v];
        renew(sz[i][v]);
      }
      mr[v].S = A * (p + mr[v].S);
      renew(m[v].A), renew(m[v].S), renew(mr[v].S), renew(D[i][v]), renew(kp[i][v]), renew(gt[i][v]);
    }
    if (PACKED && start >= 0 && !cut_fwd) {
      cut_fwd = true;
#pragma unroll
      for (int v = 0; v < V; ++v) m[v].S = fmaf(m[v].A, a.h0 ? a.h0[size_t(start) * a.C + w.c + v] : 0.0f, m[v].S);
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if (!PACKED) mr[v].A = cut_rev ? 0.0f : m[v].A;
    if (PACKED && cut_rev) mr[v].A = cut();
    if (PACKED && cut_fwd) m[v].A = cut();
  }
  again();
  if (w.r >= limit)
#pragma unroll
    for (int v = 0; v < V; ++v) mr[v] = {1.0f, 0.0f};
  const int lc = int(threadIdx.x % LX) * V;
#pragma unroll
  for (int v = 0; v < V; ++v) k.m[w.sub][lc + v] = m[v], kr.m[w.sub][lc + v] = mr[v];
  __syncthreads();
  {
    const int half = threadIdx.x / (LX * 8), ch = threadIdx.x % (LX * 8), c = w.ct * LX * V + ch;
    if (ch < LX * V && c < a.C) {
      const size_t at = (size_t(w.b) * nchunks + w.chunk) * a.C + c;
      if (half == 0) {
        fold<LX * V, false, true>(k, ch, a.states[at]);
      } else {
        fold<LX * V, true, true>(kr, ch, entering(a, w, nchunks, c, fold<LX * V, true, false>(kr, ch, 0.0f), 0.0f));
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
    const int mark = PACKED && on ? marks.start[w.sub * kRows + i] : -1;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (PACKED && mark >= 0) h[v] = a.h0 ? a.h0[size_t(mark) * a.C + w.c + v] : 0.0f;
      before[i][v] = h[v];
      h[v] = fmaf(kap[v] * kp[i][v], h[v], D[i][v] * x.get(i, v));
      renew(h[v]), renew(kp[i][v]), renew(D[i][v]);
    }
  }
  again();
  const size_t row0 = (size_t(w.b) * a.T + w.chunk * kTile) * a.C;
  const Off<V> off = Off<V>(w.sub * kRows) * Off<V>(a.C) + Off<V>(w.c);
#pragma unroll
  for (int i = kRows - 1; i >= 0; --i) {
    if (!on) continue;
    const size_t at = row0 + size_t(i) * a.C;   // + off
    float ox[V], od[V], oz[V];
    if (w.r + i >= limit) {
      if (PACKED && w.r + i < a.T) {   // rows behind the last sequence have no gradient
#pragma unroll
        for (int v = 0; v < V; ++v) ox[v] = 0.0f;
        store_row<V>(static_cast<T*>(a.dx) + at + off, ox);
        store_row<V>(static_cast<T*>(a.ddelta) + at + off, ox);
        if (a.gated) store_row<V>(static_cast<T*>(a.dz) + at + off, ox);
      }
      continue;
    }
    const int end = ends_at(i);
    const int start = PACKED ? marks.start[w.sub * kRows + i] : w.r + i == 0 ? w.b : -1;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (end >= 0) G[v] = a.dh ? a.dh[size_t(end) * a.C + w.c + v] : 0.0f;
      const float A = kap[v] * kp[i][v], xx = x.get(i, v), dyv = dy[i].get(v), zz = a.gated ? z.get(i, v) : 0.0f;
      const float s = a.gated ? sz[i][v] : 0.0f, w1 = zz * s;
      const float g = (a.gated ? dyv * w1 : dyv) + G[v];
      ox[v] = D[i][v] * g;
      od[v] = gt[i][v] * g * fmaf(-A, before[i][v], xx);   // (in this order a masked x, gt = 0, cannot overflow with g)
      dk[v] = fmaf(g * kp[i][v], before[i][v], dk[v]);
      db[v] += od[v];
      if (a.gated) {   // SiLU'(z) = s (1 + z (1 - s)) = s + w1 (1 - s)
        const float hh = !PACKED ? (i + 1 < kRows ? before[i + 1 < kRows ? i + 1 : i][v] : h[v])
                                 : fmaf(A, before[i][v], D[i][v] * xx);
        oz[v] = dyv * hh * fmaf(w1, 1.0f - s, s);
      }
      G[v] = A * g;
      renew(G[v]), renew(dk[v]), renew(db[v]);
      if (start >= 0 && a.dh0) a.dh0[size_t(start) * a.C + w.c + v] = G[v];
    }
    store_row<V>(static_cast<T*>(a.dx) + at + off, ox);
    store_row<V>(static_cast<T*>(a.ddelta) + at + off, od);
    if (a.gated) store_row<V>(static_cast<T*>(a.dz) + at + off, oz);
  }
  __syncthreads();
#pragma unroll
  for (int v = 0; v < V; ++v) k.m[w.sub][lc + v] = {dk[v], db[v]};
  __syncthreads();
  const int ch = threadIdx.x, c = w.ct * LX * V + ch;
  if (ch < LX * V && c < a.C) {
    Map sum = k.m[0][ch];
#pragma unroll
    for (int s = 1; s < kSubs; ++s) sum.A += k.m[s][ch].A, sum.S += k.m[s][ch].S;
    reinterpret_cast<Map*>(a.parts)[(size_t(w.b) * nchunks + w.chunk) * a.C + c] = sum;
  }
}

// all ones: nothing published, the counter before 0
__global__ void __launch_bounds__(256) token_scan_clear(uint64_t* __restrict__ p, size_t n) {
  for (size_t i = size_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += size_t(gridDim.x) * 256) p[i] = kNotYet;
}

// dkappa and dbias: the tiles' sums in a fixed order, in float64
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

// ---- one token for each sequence: h = a state + D x, elementwise over (B, C).  16 x 1024 3 us, a launch's least;
// 8192 x 4096 bf16 97 us, 5.5 TB/s

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
    const Gains g = gains((d.get(v) + bia.get(v)) * kLog2e);
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
  return reinterpret_cast<uintptr_t>(p) % (V * size) == 0 && batch % V == 0 && row % V == 0 && row >= 0 && row <= 1 << 22;
}
bool fits(const TokenRows& t, int V, size_t size) { return !t.p || fits(t.p, t.batch, t.row, V, size); }

// channels a thread takes: 4 (bf16) or 2 (float32) where every row is aligned for it and a tile's 128 rows lie within
// 2^31 bytes, else 1
int width(const TokenScan& a, int dtype) {
  const int V = dtype == 0 ? 2 : 4;
  const size_t size = dtype == 0 ? 4 : 2;
  const bool ok = a.C % V == 0 && a.C <= 1 << 22 && fits(a.x, V, size) && fits(a.delta, V, size) && fits(a.z, V, size) &&
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

int token_scan_chunks(int T) { return T <= kTile ? 1 : (T - 1) / kTile + 1; }

// words of the maps, the spans' heads and the counter
size_t token_scan_words(int B, int T, int C) {
  const size_t n = size_t(token_scan_chunks(T));
  return n == 1 ? 0 : 1 + size_t(B) * size_t(C) * (n + (n + kSpan - 1) / kSpan);
}

// Threads side by side in a tile.  32 of them read 256 bytes of a row in one piece instead of 128, which the memory serves
// faster once there is a tile for every CU: bf16, 1 x 4096 x 1024 (256 wide tiles) 22.5 -> 18.7 us, 8 x 4096 x 1024
// (2048) 79 -> 72, 1 x 65536 x 1024 141 -> 133; with 8 x 256 x 1024 (128) it costs, 18.4 -> 19.3.  The forward that keeps
// checkpoints (162 registers, so one workgroup of 512 threads a CU; 105 -> 111 us, 188 -> 214) and the adjoint (143 ->
// 152, 272 -> 290) are slower with it.
constexpr int kNarrow = 16, kWide = 32;
constexpr unsigned kWideFrom = 256;
static unsigned tiles(const TokenScan& a, int channels) {
  return unsigned((a.C + channels - 1) / channels) * unsigned(a.B) * unsigned(token_scan_chunks(a.T));
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
    const unsigned grid = tiles(a, kNarrow * V);
    if (a.kept) {
      if (a.offsets) token_scan_fwd<T, V, kNarrow, true, true><<<grid, kNarrow * kSubs, 0, s>>>(a, n);
      else token_scan_fwd<T, V, kNarrow, false, true><<<grid, kNarrow * kSubs, 0, s>>>(a, n);
      return hipGetLastError();
    }
    if constexpr (V > 1) {
      const unsigned wide = tiles(a, kWide * V);
      if (wide >= kWideFrom) {
        if (a.offsets) token_scan_fwd<T, V, kWide, true, false><<<wide, kWide * kSubs, 0, s>>>(a, n);
        else token_scan_fwd<T, V, kWide, false, false><<<wide, kWide * kSubs, 0, s>>>(a, n);
        return hipGetLastError();
      }
    }
    if (a.offsets) token_scan_fwd<T, V, kNarrow, true, false><<<grid, kNarrow * kSubs, 0, s>>>(a, n);
    else token_scan_fwd<T, V, kNarrow, false, false><<<grid, kNarrow * kSubs, 0, s>>>(a, n);
    return hipGetLastError();
  });
}

hipError_t launch_token_scan_bwd(const TokenScan& args, int dtype, uint64_t* words, hipStream_t s) {
  TokenScan a = args;
  clear(a, words, s);
  const int n = token_scan_chunks(a.T);
  return by_type(a, dtype, [&](auto t, auto vw) {
    using T = decltype(t);
    constexpr int V = decltype(vw)::value, LX = kNarrow;
    const unsigned grid = tiles(a, LX * V);
    if (a.offsets) {
      if (a.kept) token_scan_bwd<T, V, LX, true, true><<<grid, LX * kSubs, 0, s>>>(a, n);
      else token_scan_bwd<T, V, LX, true, false><<<grid, LX * kSubs, 0, s>>>(a, n);
    } else {
      if (a.kept) token_scan_bwd<T, V, LX, false, true><<<grid, LX * kSubs, 0, s>>>(a, n);
      else token_scan_bwd<T, V, LX, false, false><<<grid, LX * kSubs, 0, s>>>(a, n);
    }
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
