// What the kernels of the delta rule over token sequences share: chunks of sequences, values split into bfloat16 parts,
// and rows laid out as the operands of v_mfma_f32_16x16x32_bf16.
//
// Operands.  Lane l of that instruction holds, of its first operand, 8 values of row l % 16, of its second 8 values of
// column l % 16, and of its result rows 4 (l / 16) .. + 3 of column l % 16.  A sum does not care for the order of its
// terms, so the 32 terms are dealt to the lanes as the result of an earlier product holds its rows: lane l takes
// 4 g .. 4 g + 3 and 16 + 4 g .. + 3, g = l / 16.  Then two results above each other are the next product's second
// operand without leaving their registers.  A "unit" is those 8 values in bfloat16, 16 bytes; the units of one
// instruction lie in the order of the lanes.
//
// Parts.  float32 values enter as sums of bfloat16 parts, each the rounded rest of those before: 3 parts hold all
// 24 bits, and of the products of parts those are taken that lie within 2^-24 of the whole (6 of 9).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "launch.h"
#include "token_util.h"

namespace cssm {

constexpr int kChunk = 32;     // rows of a chunk
constexpr int kSegment = 128;  // rows between the states that a training pass keeps (CSSM_DELTA_SEGMENT)

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

struct Unit { uint32_t w[4]; };

__device__ __forceinline__ f32x4_t mfma16(const Unit& a, const Unit& b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// N parts of 8 values
template <int N>
__device__ __forceinline__ void split(const float (&v)[8], Unit (&u)[N]) {
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = v[i];
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = pack_bf16(x[2 * i], x[2 * i + 1]);
      u[n].w[i] = w;
      if (n + 1 < N) x[2 * i] -= __uint_as_float(w << 16), x[2 * i + 1] -= __uint_as_float(w & 0xffff0000u);
    }
}

// c += a b, small terms first
template <int NA, int NB>
__device__ __forceinline__ f32x4_t product(const Unit (&a)[NA], const Unit (&b)[NB], f32x4_t c) {
  constexpr int most = (NA > NB ? NA : NB) - 1;
#pragma unroll
  for (int s = most; s >= 0; --s)
#pragma unroll
    for (int i = 0; i < NA; ++i)
      if (s - i >= 0 && s - i < NB) c = mfma16(a[i], b[s - i], c);
  return c;
}

// the n units of a lane's operand, `stride` apart
template <int N>
__device__ __forceinline__ void take(const uint4* p, int stride, Unit (&u)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) u[n] = __builtin_bit_cast(Unit, p[n * stride]);
}

// parts of a tensor's own values: bfloat16 is one
template <typename T>
struct PartsOf { static constexpr int n = 3; };
template <>
struct PartsOf<Bf16> { static constexpr int n = 1; };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(Bf16 v) { return __uint_as_float(uint32_t(v.u) << 16); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(Bf16* p, float v) { p->u = uint16_t(pack_bf16(v, 0.0f) & 0xffffu); }

// ---- rows as first operands (16 rows a tile, the terms along the row)

// 8 values from each of two places 16 apart
template <typename T>
struct Piece;
template <>
struct Piece<Bf16> {
  uint4 q[2];
  __device__ __forceinline__ float get(int i) const { return Raw<Bf16, 8>{q[i / 8]}.get(i % 8); }
};
template <>
struct Piece<float> {
  float4 q[4];
  __device__ __forceinline__ float get(int i) const { return Raw<float, 4>{q[i / 4]}.get(i % 4); }
};

// values at .. at + 7 and at + 16 .. at + 23 of a row of n; zero behind its end, or without a row
__device__ __forceinline__ void load_piece(const Bf16* row, bool live, int at, int n, bool vec, Piece<Bf16>& p) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int c = at + 16 * h;
    p.q[h] = make_uint4(0, 0, 0, 0);
    if (vec) {
      if (live && c < n) p.q[h] = *reinterpret_cast<const uint4*>(row + c);
    } else {
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = live && c + i < n ? row[c + i].u : 0u;
      p.q[h] = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
    }
  }
}
__device__ __forceinline__ void load_piece(const float* row, bool live, int at, int n, bool vec, Piece<float>& p) {
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    const int c = at + 16 * (h / 2) + 4 * (h % 2);
    p.q[h] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (vec) {
      if (live && c < n) p.q[h] = *reinterpret_cast<const float4*>(row + c);
    } else {
      if (live && c < n) p.q[h].x = row[c];
      if (live && c + 1 < n) p.q[h].y = row[c + 1];
      if (live && c + 2 < n) p.q[h].z = row[c + 2];
      if (live && c + 3 < n) p.q[h].w = row[c + 3];
    }
  }
}

// the piece as two units (g = 2 p and 2 p + 1), each in N parts `plane` apart, times `by`
template <int N, typename T>
__device__ __forceinline__ void store_piece(const Piece<T>& p, float by, uint4* at, int plane) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    Unit u[N];
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = p.get(4 * h + i) * by, v[4 + i] = p.get(8 + 4 * h + i) * by;
    split<N>(v, u);
#pragma unroll
    for (int n = 0; n < N; ++n) at[n * plane + h * 16] = __builtin_bit_cast(uint4, u[n]);
  }
}
// as it is
__device__ __forceinline__ void store_piece(const Piece<Bf16>& p, uint4* at, int) {
  at[0] = make_uint4(p.q[0].x, p.q[0].y, p.q[1].x, p.q[1].y);
  at[16] = make_uint4(p.q[0].z, p.q[0].w, p.q[1].z, p.q[1].w);
}
__device__ __forceinline__ void store_piece(const Piece<float>& p, uint4* at, int plane) { store_piece<3>(p, 1.0f, at, plane); }

// ---- columns as first operands, or rows as second ones (16 columns a tile, the terms down the chunk's rows)

// two columns of the 8 rows first .. first + 3 and first + 16 .. first + 19
template <typename T>
struct Columns;
template <>
struct Columns<Bf16> {
  uint32_t w[8];
  __device__ __forceinline__ float get(int j, int h) const { return __uint_as_float(h ? w[j] & 0xffff0000u : w[j] << 16); }
};
template <>
struct Columns<float> {
  float2 w[8];
  __device__ __forceinline__ float get(int j, int h) const { return h ? w[j].y : w[j].x; }
};

template <typename T>
__device__ __forceinline__ void load_columns(const T* base, long long stride, int first, int rows, int at, int n, bool vec,
                                             Columns<T>& c) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int r = first + (j < 4 ? j : 12 + j);
    const T* p = base + (long long)r * stride + at;
    const bool one = r < rows && at < n, two = r < rows && at + 1 < n;
    if constexpr (sizeof(T) == 2) {
      c.w[j] = 0;
      if (vec) {
        if (one) c.w[j] = *reinterpret_cast<const uint32_t*>(p);
      } else {
        if (one) c.w[j] = p[0].u;
        if (two) c.w[j] |= uint32_t(p[1].u) << 16;
      }
    } else {
      c.w[j] = make_float2(0.0f, 0.0f);
      if (vec) {
        if (one) c.w[j] = *reinterpret_cast<const float2*>(p);
      } else {
        if (one) c.w[j].x = p[0];
        if (two) c.w[j].y = p[1];
      }
    }
  }
}

// the two units, each in N parts, row j times by[j]
template <int N, typename T>
__device__ __forceinline__ void store_columns(const Columns<T>& c, const float (&by)[8], uint4* at, int plane) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    Unit u[N];
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c.get(j, h) * by[j];
    split<N>(v, u);
#pragma unroll
    for (int n = 0; n < N; ++n) at[n * plane + h] = __builtin_bit_cast(uint4, u[n]);
  }
}
// as they are
__device__ __forceinline__ void store_columns(const Columns<Bf16>& c, uint4* at, int) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    Unit u;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      u.w[i] = h ? c.w[2 * i] >> 16 | (c.w[2 * i + 1] & 0xffff0000u) : (c.w[2 * i] & 0xffffu) | c.w[2 * i + 1] << 16;
    at[h] = __builtin_bit_cast(uint4, u);
  }
}
__device__ __forceinline__ void store_columns(const Columns<float>& c, uint4* at, int plane) {
  const float one[8] = {1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f};
  store_columns<3>(c, one, at, plane);
}

// ---- sequences and their chunks

struct Span { int row, rows, slot, segment; };   // first row, number of rows, first chunk's and first segment's slot

__host__ __device__ __forceinline__ int chunks_of(int rows) { return rows / kChunk + (rows % kChunk != 0); }
__host__ __device__ __forceinline__ int segments_of(int rows) { return rows / kSegment + (rows % kSegment != 0); }

// sequence i; offsets outside the rows are taken to the nearest inside
__device__ __forceinline__ Span span_of(const DeltaRule& a, int i) {
  if (!a.offsets) return {0, a.T, i * chunks_of(a.T), i * segments_of(a.T)};
  int lo = a.offsets[i], hi = a.offsets[i + 1];
  lo = lo < 0 ? 0 : lo > a.T ? a.T : lo;
  hi = hi < lo ? lo : hi > a.T ? a.T : hi;
  return {lo, hi - lo, lo / kChunk + i, lo / kSegment + i};
}

// batch b's row t of a tensor of rows
template <typename T>
__device__ __forceinline__ const T* row_at(const TokenRows& r, int b, long long t) {
  return static_cast<const T*>(r.p) + (long long)b * r.batch + t * r.row;
}

}  // namespace cssm
