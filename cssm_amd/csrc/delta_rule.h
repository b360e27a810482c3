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
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

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

// ---- a chunk's rows in memory.  They are read through buffer descriptors, which give 0 beyond their end: loads need no
// branches, so that all of a chunk's are on their way at once.  WIDE: aligned 16-byte vectors, and rows that do not
// overlap, so that a row behind the last lies beyond the descriptor's end; else single elements with every row's number
// looked at.

constexpr uint32_t kNowhere = 0x80000000u;   // beyond the end of every descriptor
constexpr int kMostStride = 1 << 24;         // elements from row to row: 31 rows within 2^31 bytes

struct Rows {
  __amdgpu_buffer_rsrc_t r;
  uint32_t stride;   // elements
  int rows;
  // `rows` rows of `width` elements (more than 32: the first 32)
  template <typename T>
  __device__ __forceinline__ Rows(const T* base, long long stride_, int rows_, int width)
      : r(__builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base), 0,
                                            rows_ <= 0 ? 0 : int((uint32_t((rows_ < kChunk ? rows_ : kChunk) - 1) * uint32_t(stride_) + uint32_t(width)) * sizeof(T)),
                                            0x00020000)),
        stride(uint32_t(stride_)), rows(rows_) {}
  // byte offset of an element
  template <typename T, bool WIDE>
  __device__ __forceinline__ uint32_t at(int row, int col, int width) const {
    const bool in = col < width && (WIDE || row < rows);
    return in ? (uint32_t(row) * stride + uint32_t(col)) * uint32_t(sizeof(T)) : kNowhere;
  }
};

template <typename T>
__device__ __forceinline__ uint32_t load_element(const Rows& m, uint32_t off) {
  if constexpr (sizeof(T) == 2) return uint16_t(__builtin_amdgcn_raw_buffer_load_b16(m.r, int(off), 0, 0));
  else return __builtin_amdgcn_raw_buffer_load_b32(m.r, int(off), 0, 0);
}
template <typename T>
__device__ __forceinline__ float element(uint32_t raw) { return __uint_as_float(sizeof(T) == 2 ? raw << 16 : raw); }
template <typename T>
__device__ __forceinline__ void store_element(const Rows& m, uint32_t off, float v) {
  if constexpr (sizeof(T) == 2) __builtin_amdgcn_raw_buffer_store_b16(short(pack_bf16(v, 0.0f) & 0xffffu), m.r, int(off), 0, 0);
  else __builtin_amdgcn_raw_buffer_store_b32(int(__float_as_uint(v)), m.r, int(off), 0, 0);
}
__device__ __forceinline__ uint4 load16(const Rows& m, uint32_t off) {
  return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(m.r, int(off), 0, 0));
}

// ---- rows as first operands (16 rows a tile, the terms along the row)

// 8 values from each of two places of a row 16 apart
template <typename T, bool WIDE>
struct Piece {
  static constexpr int kWords = WIDE ? 4 * sizeof(T) : 16;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const Rows& m, int row, int col, int n) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if constexpr (WIDE) {
        const uint32_t o = m.at<T, true>(row, col + 16 * h, n);
#pragma unroll
        for (int i = 0; i < int(sizeof(T)) / 2; ++i) {
          const uint4 q = load16(m, o + 16 * i);
          uint32_t* d = w + 2 * h * sizeof(T) + 4 * i;
          d[0] = q.x, d[1] = q.y, d[2] = q.z, d[3] = q.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[8 * h + i] = load_element<T>(m, m.at<T, false>(row, col + 16 * h + i, n));
      }
    }
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (WIDE && sizeof(T) == 2) return __uint_as_float(i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    else return element<T>(w[i]);
  }
  // values 2 i and 2 i + 1 of bfloat16
  __device__ __forceinline__ uint32_t pair(int i) const {
    if constexpr (WIDE) return w[i];
    else return w[2 * i] | w[2 * i + 1] << 16;
  }
  // as two units (g = 2 p and 2 p + 1), each in N parts `plane` apart, times `by`
  template <int N>
  __device__ __forceinline__ void store_by(float by, uint4* at, int plane) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      Unit u[N];
      float v[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = get(4 * h + i) * by, v[4 + i] = get(8 + 4 * h + i) * by;
      split<N>(v, u);
#pragma unroll
      for (int n = 0; n < N; ++n) at[n * plane + h * 16] = __builtin_bit_cast(uint4, u[n]);
    }
  }
  // as they are
  __device__ __forceinline__ void store(uint4* at, int plane) const {
    if constexpr (sizeof(T) == 2) {
      at[0] = make_uint4(pair(0), pair(1), pair(4), pair(5));
      at[16] = make_uint4(pair(2), pair(3), pair(6), pair(7));
    } else {
      store_by<3>(1.0f, at, plane);
    }
  }
};

// ---- columns as first operands, or rows as second ones (16 columns a tile, the terms down the chunk's rows)

// row j of a unit of column operands whose first is `first`
__device__ __forceinline__ int unit_row(int first, int j) { return first + (j < 4 ? j : 12 + j); }

// two columns of 8 rows
template <typename T, bool WIDE>
struct Columns {
  static constexpr int kWords = WIDE ? sizeof(T) / 2 : 2;
  uint32_t w[8][kWords];
  __device__ __forceinline__ void load(const Rows& m, int first, int col, int n) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int r = unit_row(first, j);
      if constexpr (WIDE && sizeof(T) == 2) {
        w[j][0] = __builtin_amdgcn_raw_buffer_load_b32(m.r, int(m.at<T, true>(r, col, n)), 0, 0);
      } else if constexpr (WIDE) {
        const uint2 q = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(m.r, int(m.at<T, true>(r, col, n)), 0, 0));
        w[j][0] = q.x, w[j][1] = q.y;
      } else {
        w[j][0] = load_element<T>(m, m.at<T, false>(r, col, n));
        w[j][1] = load_element<T>(m, m.at<T, false>(r, col + 1, n));
      }
    }
  }
  __device__ __forceinline__ float get(int j, int h) const {
    if constexpr (WIDE && sizeof(T) == 2) return __uint_as_float(h ? w[j][0] & 0xffff0000u : w[j][0] << 16);
    else return element<T>(w[j][h]);
  }
  // the two units, each in N parts, row j times by[j]
  template <int N>
  __device__ __forceinline__ void store_by(const float (&by)[8], uint4* at, int plane) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      Unit u[N];
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = get(j, h) * by[j];
      split<N>(v, u);
#pragma unroll
      for (int n = 0; n < N; ++n) at[n * plane + h] = __builtin_bit_cast(uint4, u[n]);
    }
  }
  __device__ __forceinline__ void store(uint4* at, int plane) const {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        Unit u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (WIDE)
            u.w[i] = h ? w[2 * i][0] >> 16 | (w[2 * i + 1][0] & 0xffff0000u) : (w[2 * i][0] & 0xffffu) | w[2 * i + 1][0] << 16;
          else u.w[i] = w[2 * i][h] | w[2 * i + 1][h] << 16;
        }
        at[h] = __builtin_bit_cast(uint4, u);
      }
    } else {
      const float one[8] = {1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f};
      store_by<3>(one, at, plane);
    }
  }
};

// 8 values of a result's rows from LDS: those of the rows that a lane holds
__device__ __forceinline__ void take_rows(const float* s, int g, float (&v)[8]) {
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const float4 q = *reinterpret_cast<const float4*>(s + 16 * t + 4 * g);
    v[4 * t] = q.x, v[4 * t + 1] = q.y, v[4 * t + 2] = q.z, v[4 * t + 3] = q.w;
  }
}

constexpr int kDecays = 3 * kChunk * kChunk;   // D, and with decays P and A, of one chunk and head for the adjoint
constexpr int kUnits = 6 * 128;   // units of L and P of one chunk and head, three parts each

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

// The x-th longest of up to 64 packed sequences (the first of equals first), x itself of more or of a batch: workgroups begin in
// order, and the longest sequence, begun last, would be walked by a chip that has nothing else left (23 sequences in 16001
// rows x 16 heads, twelve draws: 266 us in their order, 241 so).  All lanes take part.
__device__ __forceinline__ int longest_first(const DeltaRule& a, int x) {
  if (!a.offsets || a.nseq > 64) return x;
  const int lane = threadIdx.x % 64, mine = lane < a.nseq ? span_of(a, lane).rows : -1;
  int longer = 0;
  for (int i = 0; i < a.nseq; ++i) {
    const int other = __shfl(mine, i);
    longer += other > mine || (other == mine && i < lane);
  }
  return __ffsll((unsigned long long)__ballot(longer == x && lane < a.nseq)) - 1;
}

// rows that WIDE takes: 16-byte vectors, and none overlapping the next
template <typename T>
inline bool wide_rows(const TokenRows& r, int heads, int n) {
  return n % 8 == 0 && reinterpret_cast<uintptr_t>(r.p) % 16 == 0 && r.batch * (long long)sizeof(T) % 16 == 0 &&
         r.row * (long long)sizeof(T) % 16 == 0 && r.row >= (long long)heads * n;
}

// L and P of all chunks, or their transposes and D, into the workspace
template <typename T, bool TURNED>
void launch_delta_prepare(const DeltaRule& a, bool wide, hipStream_t s);

// batch b's row t of a tensor of rows
template <typename T>
__device__ __forceinline__ const T* row_at(const TokenRows& r, int b, long long t) {
  return static_cast<const T*>(r.p) + (long long)b * r.batch + t * r.row;
}

}  // namespace cssm
